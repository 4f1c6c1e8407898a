"""GPU: the policy with a memory whose constants are replaced."""
import pytest
import torch

from test_gpu_retention import _replay, _same, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_replaced_decays_are_seen(graph):
    """log_decay replaced after a (captured) collection: the next one acts by the new values."""
    env, policy, buf, col = _setup(64, 20)
    col.collect()
    col.collect(graph=graph)
    old = policy.log_decay  # held: its memory is not used again
    policy.log_decay = old * 0.25
    col.collect(graph=graph)
    with torch.no_grad():
        values, log_probs, _ = _replay(policy, buf, col.rollout_memory)
    _same(values, buf.values)
    _same(log_probs, buf.log_probs)
    assert old is not policy.log_decay
    env.close()

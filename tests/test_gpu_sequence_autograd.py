"""GPU: what autograd has to know of the sequence operators: writes in place."""
import pytest
import torch

from test_gpu_sequence import DEV, _case, _dev, _seq

pytestmark = pytest.mark.gpu


def _step(d, state, **kw):
    return _seq().linear_attention_step(d["q"][0], d["k"][0], d["v"][0], d["log_decay"], state, **kw)


@pytest.mark.parametrize("out", [False, True])
def test_a_step_on_a_saved_state_is_seen(out):
    """The backward pass reads the initial state again: after a step has written into it, the pass is refused."""
    d = _dev(_case(6, 2, 2, 16, 16, torch.float32))
    q, state = d["q"].requires_grad_(), d["state"]
    y, _ = _seq().linear_attention(q, d["k"], d["v"], d["log_decay"], state)
    version = state._version
    with torch.no_grad():
        if out:
            _step(d, torch.zeros_like(state), state_out=state)
        else:
            _step(d, state)
    assert state._version > version
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, q, d["dout"])
    # a state that is only read stays as it is
    y, _ = _seq().linear_attention(q, d["k"], d["v"], d["log_decay"], state)
    with torch.no_grad():
        _step(d, state, state_out=torch.empty_like(state))
    torch.autograd.grad(y, q, d["dout"])


def test_steps_in_inference_mode():
    d = _dev(_case(1, 2, 2, 16, 16, torch.float32))
    want = _step(d, d["state"].clone())
    with torch.inference_mode():
        got = _step(d, d["state"].clone())  # a state without a version
        again = _step(d, d["state"])        # one with
    assert torch.equal(got, want) and torch.equal(again, want)


@pytest.mark.parametrize("graph", [False, True])
def test_a_collection_on_a_saved_memory_is_seen(graph):
    from test_gpu_retention import _setup
    env, policy, buf, col = _setup(16, 8)
    col.collect()
    values, log_probs, _ = policy.evaluate_actions(buf.observations.clone(), buf.actions.clone(), buf.dones.clone(), col.memory)
    col.collect(graph=graph)
    with pytest.raises(RuntimeError, match="inplace"):
        (values.sum() + log_probs.sum()).backward()
    env.close()

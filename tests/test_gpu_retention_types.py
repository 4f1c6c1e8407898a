"""GPU: the policy with a memory whose constants are replaced, in 16 bits, and in a collector that starts over.

Tolerance of the 16-bit runs: a chain of about ten roundings to the type, half a step each, on values of size up to about 10,
a norm between them: 30 steps relative to the largest value."""
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


def _same16(a, b, dtype):
    assert bool(b.isfinite().all())
    assert float((a.detach().float() - b).abs().max()) < 30 * torch.finfo(dtype).eps * (1 + float(b.abs().max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_step_captured_under_autocast(dtype):
    """It makes its own casts of the weights: those of the capture's context are gone after it and know no later update.
    Outside of autocast it is captured anew."""
    env, policy, buf, col = _setup(64, 20)
    col.collect()
    with torch.autocast("cuda", dtype=dtype):
        col.collect()
        col.collect(graph=True)
        _same16(_replay(policy, buf, col.rollout_memory)[0], buf.values, dtype)
    old = buf.values.clone()
    with torch.no_grad():
        policy.value_net.weight.mul_(-3.0)
        policy.value_net.bias.add_(1.0)
    with torch.autocast("cuda", dtype=dtype):
        col.collect(graph=True)
        _same16(_replay(policy, buf, col.rollout_memory)[0], buf.values, dtype)
    assert float((old - buf.values).abs().max()) > 0.5
    col.collect(graph=True)
    with torch.no_grad():
        values, log_probs, _ = _replay(policy, buf, col.rollout_memory)
    _same(values, buf.values)
    _same(log_probs, buf.log_probs)
    env.close()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_collection_and_update_in_one_autocast(dtype, graph):
    """The collection's casts of the weights carry no gradient; the update makes its own."""
    env, policy, buf, col = _setup(64, 20)
    with torch.autocast("cuda", dtype=dtype):
        col.collect()
        col.collect(graph=graph)
        values, _, _ = _replay(policy, buf, col.rollout_memory)
    _same16(values, buf.values, dtype)
    values.float().sum().backward()
    for p in (policy.embed.weight, policy.qkv.weight, policy.mix.weight, policy.value_net.weight):
        assert bool(p.grad.any()) and bool(p.grad.isfinite().all())
    env.close()


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_policy_cast_to_16_bits(dtype, graph):
    env, policy, buf, col = _setup(64, 20)
    decay = policy.log_decay.clone()
    assert policy.to(dtype) is policy
    assert torch.equal(policy.log_decay, decay) and policy.embed.weight.dtype == dtype
    assert "log_decay" in policy.state_dict()
    col.collect()
    col.collect(graph=graph)
    assert col.memory.dtype == torch.float32
    values, _, _ = _replay(policy, buf, col.rollout_memory)
    _same16(values, buf.values, dtype)
    values.float().sum().backward()
    for p in (policy.embed.weight, policy.qkv.weight, policy.mix.weight, policy.value_net.weight):
        assert bool(p.grad.any()) and bool(p.grad.isfinite().all())
    env.close()


def test_a_collector_started_over_has_no_memory():
    """last_obs = None resets the environments with the next collection: what they remembered goes with their episodes."""
    env, policy, buf, col = _setup(16, 8)
    col.collect()
    assert bool(col.memory.any())
    at = col.memory.data_ptr()
    col.last_obs = None
    col.collect()
    assert not bool(col.rollout_memory.any()) and col.memory.data_ptr() == at
    with torch.no_grad():
        values, _, _ = _replay(policy, buf, None)
    _same(values, buf.values)
    env.close()

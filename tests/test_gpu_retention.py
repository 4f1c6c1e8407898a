"""GPU: the policy with a memory (rollout.RetentionActorCritic) in the collector: what the single-token form computed
step by step while the rollout was collected, the form over whole columns computes again for the update.

Tolerance: both are float32 chains of a few products of width 64 (2^-24 x 64 each, on values of size up to about 10)
and a group norm, which divides by a spread that is not small here; 2e-4 relative is some 20 times the sum of these.
"""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _setup(n, T, steps_max=12, normalize=True):
    from tum_adlr_deep_reinforcement_learning_amd.rollout import RetentionActorCritic, RolloutBuffer, RolloutCollector
    from tum_adlr_deep_reinforcement_learning_amd.vec_env import FixedWingVecEnv
    from tum_adlr_deep_reinforcement_learning_amd.vec_normalize import VecNormalize
    torch.manual_seed(0)
    env = FixedWingVecEnv(n, config_kw={"steps_max": steps_max}, sim_config_kw={"turbulence": False}, device=DEV, seed=4,
                          return_tensors=True)
    if normalize:
        env = VecNormalize(env)
    policy = RetentionActorCritic(env.observation_space.shape[0], env.action_space.shape[0]).to(DEV)
    with torch.no_grad():  # heads that depend on the memory visibly
        policy.action_net.weight.mul_(30.0)
        policy.value_net.weight.mul_(3.0)
    buf = RolloutBuffer(T, env.observation_space, env.action_space, device=DEV, gae_lambda=0.95, gamma=0.99, n_envs=n)
    return env, policy, buf, RolloutCollector(env, policy, buf)


def _replay(policy, buf, memory):
    return policy.evaluate_actions(buf.observations, buf.actions, buf.dones, memory)


def _same(a, b):
    assert float((a - b).abs().max()) < 2e-4 * (1 + float(b.abs().max()))


@pytest.mark.parametrize("graph", [False, True])
def test_collected_rows_are_what_the_columns_give(graph):
    n, T = 64, 40  # episodes of 12 steps: several starts in every column
    env, policy, buf, col = _setup(n, T)
    col.collect()
    for _ in range(2):  # the second collection begins with a memory, in the middle of episodes
        before = col.memory.clone()
        col.collect(graph=graph)
        assert hasattr(col, "_graphs") == graph
        assert torch.equal(col.rollout_memory, before)
        assert int((buf.dones != 0).sum()) >= 2 * n
        with torch.no_grad():
            values, log_probs, _ = _replay(policy, buf, col.rollout_memory)
        _same(values, buf.values)
        _same(log_probs, buf.log_probs)
        # the memory matters: from an empty one the first rows come out otherwise
        with torch.no_grad():
            other, _, _ = _replay(policy, buf, None)
        assert float((other - buf.values).abs().max()) > 1e-2
    env.close()


def test_two_collectors_share_one_policy():
    env, policy, buf, col = _setup(16, 20)
    from tum_adlr_deep_reinforcement_learning_amd.rollout import RolloutCollector
    env2, _, buf2, _ = _setup(16, 20)
    other = RolloutCollector(env2, policy, buf2)
    for graph in (False, True, True):  # a captured collection follows one eager one
        for c in (col, other):
            c.collect(graph=graph)
    for c, b in ((col, buf), (other, buf2)):
        with torch.no_grad():
            values, log_probs, _ = _replay(policy, b, c.rollout_memory)
        _same(values, b.values)
        _same(log_probs, b.log_probs)
    some = torch.tensor([3, 0, 7], device=DEV)  # a minibatch of columns
    with torch.no_grad():
        values, _, _ = policy.evaluate_actions(buf.observations[:, some], buf.actions[:, some], buf.dones[:, some],
                                               col.rollout_memory[some])
    _same(values, buf.values[:, some])
    env.close()
    env2.close()


def test_the_memory_after_a_collection_is_the_columns_final_state():
    from tum_adlr_deep_reinforcement_learning_amd import sequence
    env, policy, buf, col = _setup(32, 30)
    col.collect()
    col.collect()
    with torch.no_grad():
        _, q, k, v = policy._project(buf.observations)
        _, final = sequence.linear_attention(q, k, v, policy.log_decay, col.rollout_memory, buf.dones)
        before = col.memory.clone()
        policy.predict_values(col.last_obs, col.memory, col.last_dones)
    _same(final, col.memory)
    assert torch.equal(before, col.memory)
    env.close()


def test_update_gradients_against_a_plain_restatement():
    """A PPO-like loss through evaluate_actions: every parameter's gradient against the same policy in float64 with the
    recurrence written out token by token."""
    env, policy, buf, col = _setup(16, 25)
    col.collect()
    col.collect()
    g = torch.randn(25, 16, device=DEV)

    def loss(values, logp, entropy, w):
        return (logp * w).mean() + 0.5 * ((values - w) ** 2).mean() - 0.01 * entropy
    out = loss(*_replay(policy, buf, col.rollout_memory), g)
    grads = torch.autograd.grad(out, list(policy.parameters()))

    ref = copy.deepcopy(policy).double().cpu()
    obs, act, starts, w = (x.detach().cpu() for x in (buf.observations, buf.actions, buf.dones, g))
    x, q, k, v = ref._project(obs.double())
    S, rows = col.rollout_memory.cpu().double(), []
    decay = torch.exp(ref.log_decay.double())[None, :, None, None]
    for t in range(25):
        keep = (starts[t] == 0).double()[:, None, None, None]
        S = keep * decay * S + k[t][..., None] * v[t][..., None, :]
        rows.append((q[t][..., None] * S).sum(-2))
    m = torch.stack(rows)
    y = torch.nn.functional.group_norm(m.reshape(25 * 16, -1), 4, ref.norm_weight, ref.norm_bias, 1e-5)
    f = x + ref.mix(torch.nn.functional.silu(y).view(x.shape))
    ent = (0.5 + 0.5 * torch.log(torch.tensor(2 * torch.pi)) + ref.log_std).sum()
    want = loss(ref.value_net(f).squeeze(-1), ref._log_prob(act.double(), ref.action_net(f)), ent, w.double())
    assert abs(float(want.detach()) - float(out.detach())) < 1e-4 * (1 + abs(float(want.detach())))
    for (name, p), a, b in zip(policy.named_parameters(), grads, torch.autograd.grad(want, list(ref.parameters()))):
        err = float((a.cpu().double() - b).abs().max())
        assert err < 1e-3 * (float(b.abs().max()) + 1e-3), (name, err, float(b.abs().max()))
    env.close()


def test_refusals():
    from tum_adlr_deep_reinforcement_learning_amd.rollout import RetentionActorCritic
    with pytest.raises(ValueError):
        RetentionActorCritic(14, 3, width=64, heads=5)
    p = RetentionActorCritic(14, 3)
    with pytest.raises(ValueError, match="GPU"):
        p(torch.zeros(4, 14), p.new_memory(4))

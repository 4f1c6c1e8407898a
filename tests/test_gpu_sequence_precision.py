"""GPU: the sequence operators where a result hangs on few bits: terms that cancel.  Expected values are exact sums."""
import pytest
import torch

from test_gpu_sequence import DEV, DTYPES, _seq

pytestmark = pytest.mark.gpu
SIZES = [(8, 8), (16, 16), (20, 40), (64, 64), (128, 128), (128, 24)]
BIT = 2.0 ** -17  # 1 + 2^-9 + BIT has three runs of bits, each a bfloat16 of its own
# Two terms of size 1 meet: products and weights of 1 are exact, and the sum is rounded at most four times.
TOL = 4 * 2 * 2.0 ** -24


def _zeros(T, Dk, Dv, dtype):
    z = lambda d: torch.zeros(T, 1, 1, d, dtype=dtype, device=DEV)
    return z(Dk), z(Dk), z(Dv), torch.zeros(1, device=DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", SIZES)
@pytest.mark.parametrize("T", [1, 40])
def test_states_that_cancel(T, Dk, Dv, dtype):
    """q picks the difference of two state rows that agree to 2^-17."""
    q, k, v, ld = _zeros(T, Dk, Dv, dtype)
    q[..., :2] = 1
    state = torch.zeros(1, 1, Dk, Dv, device=DEV)
    state[..., 0, :] = 1 + 2.0 ** -9 + BIT
    state[..., 1, :] = -(1 + 2.0 ** -9)
    out, final = _seq().linear_attention(q, k, v, ld, state)
    assert torch.equal(final, state)
    assert float((out.double() - BIT).abs().max()) <= TOL


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", SIZES)
@pytest.mark.parametrize("at", [(0, 1), (3, 20), (17, 30)])
def test_scores_that_cancel(at, Dk, Dv, dtype):
    """Two tokens' scores agree to 2^-17 and their values are opposite; the gradient of the values likewise."""
    q, k, v, ld = _zeros(40, Dk, Dv, dtype)
    q[..., :3] = 1
    k[at[0], ..., 0] = k[at[1], ..., 0] = 1
    k[at[0], ..., 1] = k[at[1], ..., 1] = 2.0 ** -9
    k[at[0], ..., 2] = BIT
    v[at[0]], v[at[1]] = 1, -1
    out, _ = _seq().linear_attention(q, k, v, ld)
    assert float((out[at[1]:].double() - BIT).abs().max()) <= TOL
    # reversed in time: dv_0 = sum_t (q_t . k_0) dout_t, with the roles of q and k and the order of tokens turned around
    k, q = q.flip(0), k.flip(0)
    v = torch.zeros_like(v).requires_grad_()
    dout = torch.zeros_like(v)
    dout[39 - at[0]], dout[39 - at[1]] = 1, -1
    out, _ = _seq().linear_attention(q, k, v, ld)
    dv, = torch.autograd.grad(out, v, dout)
    assert float((dv[:40 - at[1]].double() - BIT).abs().max()) <= TOL


# ------------------------------------------------------------------ decays
DECAYS = [-1e-4, -0.3, -0.5, -1.1, -2.0, -18.0]


def _decayed(T, ld, state):
    return state.double() * torch.exp(ld.double() * T)[None, :, None, None]


def _near(got, want, rel, ld):
    # what float32 cannot hold any more may be anything up to its smallest normal number
    err, tol = (got.double() - want).abs(), rel * want.abs() + torch.finfo(got.dtype).tiny
    worst = (err / tol).amax((0, 2, 3)) if got.dim() == 4 else (err / tol).max()
    assert bool((err <= tol).all()), "log_decay %s: %s times the tolerance" % (ld.tolist(), worst.tolist())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(16, 16), (33, 20), (64, 64), (128, 128)])
@pytest.mark.parametrize("T,N", [(1, 2), (16, 2), (33, 2), (70, 2), (520, 1)])  # the last in time segments
def test_a_state_that_only_decays(T, N, Dk, Dv, dtype):
    """No keys: the final state, and the gradient of the initial one, are the state given times g^T.  Per block of 16
    tokens (and per segment) the weight may be off by two units of float32's exponential and one rounding, and its product
    with the state by another: 2^-22 together.  The float32 exponent log_decay x c is off by 2^-24 of itself besides."""
    H = len(DECAYS)
    z = lambda d: torch.zeros(T, N, H, d, dtype=dtype, device=DEV)
    ld = torch.tensor(DECAYS, device=DEV)
    state = (torch.rand(N, H, Dk, Dv, device=DEV) + 0.5) * 1e6
    dfinal = torch.rand(N, H, Dk, Dv, device=DEV) + 0.5
    state.requires_grad_()
    _, final = _seq().linear_attention(z(Dk), z(Dk), z(Dv), ld, state)
    dstate, = torch.autograd.grad(final, state, dfinal)
    rel = ((T // 16 + 4) * 2.0 ** -22 + 2.0 ** -23 * T * ld.double().abs())[None, :, None, None]
    _near(final.detach(), _decayed(T, ld, state.detach()), rel, ld)
    _near(dstate, _decayed(T, ld, dfinal), rel, ld)


@pytest.mark.parametrize("N,Dk,Dv", [(3, 16, 16), (3, 128, 128), (700, 64, 64), (3, 20, 3), (5, 9, 33)])
def test_a_step_that_only_decays(N, Dk, Dv):
    H = len(DECAYS)
    z = lambda d: torch.zeros(N, H, d, device=DEV)
    ld = torch.tensor(DECAYS, device=DEV)
    state = (torch.rand(N, H, Dk, Dv, device=DEV) + 0.5) * 1e6
    want = _decayed(1, ld, state)
    q = z(Dk)
    q[..., 0] = 1
    out = _seq().linear_attention_step(q, z(Dk), z(Dv), ld, state)
    _near(state, want, 2.0 ** -22, ld)
    _near(out, want[:, :, 0], 2.0 ** -22, ld)


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (64, 64), (128, 128), (20, 40)])
def test_weights_of_a_block(Dk, Dv):
    """One key and one query at a time: out_t = g^(t+1) S + g^t v, relative to 2^-21 at every distance: the weight's
    exponent is carried beyond float32 (its rounding alone would be 2^-24 of an exponent of up to 30)."""
    T, ld = 16, torch.tensor([-0.37, -1.13, -1.9], device=DEV)
    q = torch.zeros(T, 1, 3, Dk, device=DEV)
    k, v = torch.zeros_like(q), torch.ones(T, 1, 3, Dv, device=DEV)
    q[..., 0] = 1
    k[0, ..., 0] = 1
    d = torch.exp(ld.double() * torch.arange(T + 1, device=DEV, dtype=torch.double)[:, None])[:, None, :, None]
    out, final = _seq().linear_attention(q, k, v, ld)
    _near(out, d[:T].expand(out.shape), 2.0 ** -21, ld)
    _near(final[:, :, :1], d[T - 1][..., None].expand(final[:, :, :1].shape), 2.0 ** -21, ld)
    state = torch.zeros(1, 3, Dk, Dv, device=DEV)
    state[:, :, 0] = 1
    out, final = _seq().linear_attention(q, torch.zeros_like(k), v, ld, state)
    _near(out, d[1:].expand(out.shape), 2.0 ** -21, ld)
    _near(final[:, :, :1], d[T][..., None].expand(final[:, :, :1].shape), 2.0 ** -21, ld)
    # reversed: dv_0 = sum_t g^t dout_t, one at a time
    for t in (1, 7, 15):
        x = torch.zeros(T, 1, 3, Dv, device=DEV).requires_grad_()
        dout = torch.zeros_like(x)
        dout[t] = 1
        out, _ = _seq().linear_attention(q, k, x, ld)
        dv, = torch.autograd.grad(out, x, dout)
        _near(dv[:1], d[t:t + 1].expand(dv[:1].shape), 2.0 ** -21, ld)


@pytest.mark.parametrize("Dv", [16, 3])
def test_steps_without_decay_and_without_memory(Dv):
    z = lambda d: torch.zeros(2, 2, d, device=DEV)
    state = torch.randn(2, 2, 16, Dv, device=DEV)
    want = state.clone()
    want[:, 1] = 0
    _seq().linear_attention_step(z(16), z(16), z(Dv), torch.tensor([0.0, -float("inf")], device=DEV), state)
    assert torch.equal(state, want)


# ------------------------------------------------------------------ bad numbers over a long time
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [None, 600])
@pytest.mark.parametrize("what", ["state", "q", "k", "v", "dout", "dfinal"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_bad_numbers_over_time_segments(bad, what, start, dtype):
    """1100 tokens of one sequence run in time segments; with these decays what a segment multiplies a state with is less
    than float32 holds.  An infinity or a NaN still reaches every later token (earlier, in the gradients) up to an episode
    start, as the recurrence has it, and nothing else."""
    from oracle import sequence_oracle as R
    T = 1100
    gen = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen)
    c = dict(q=rn(T, 1, 2, 16).to(dtype), k=rn(T, 1, 2, 16).to(dtype), v=rn(T, 1, 2, 16).to(dtype), state=rn(1, 2, 16, 16),
             dout=rn(T, 1, 2, 16).to(dtype), dfinal=rn(1, 2, 16, 16))
    if what in ("state", "dfinal"):
        c[what][0, 1, 3, 5] = bad
    else:
        c[what][5 if what in "kv" else 1093, 0, 1, 3] = bad
    ld = torch.tensor([-1.3, -0.9])
    starts = torch.zeros(T, 1, dtype=torch.uint8)
    if start:
        starts[start] = 1
    d = {n: x.to(DEV) for n, x in c.items()}
    leaves = [d[n].requires_grad_() for n in ("q", "k", "v", "state")]
    out, final = _seq().linear_attention(*leaves[:3], ld.to(DEV), leaves[3], starts.to(DEV))
    got = (out, final) + torch.autograd.grad([out, final], leaves, [d["dout"], d["dfinal"]])
    ref = R.linear_attention(c["q"], c["k"], c["v"], ld, c["state"], starts, None, c["dout"], c["dfinal"])
    for name, g, r in zip(("out", "final", "dq", "dk", "dv", "dstate"), got, ref):
        wrong = g.cpu().isfinite() != r.isfinite()
        assert not bool(wrong.any()), "%s: %d of %d, first at %s" % (name, int(wrong.sum()), wrong.numel(),
                                                                     wrong.nonzero()[0].tolist())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv,T", [(20, 40, 75), (24, 72, 75), (63, 63, 75), (101, 97, 75), (127, 20, 75), (3, 5, 75),
                                     (128, 120, 75), (63, 63, 600), (101, 97, 600), (24, 72, 600)])
@pytest.mark.parametrize("what", ["state", "q", "k", "v", "dout", "dfinal"])
def test_bad_numbers_in_heads_of_any_size(what, Dk, Dv, T, dtype):
    """Heads that do not fill their tiles, rows that are no whole vectors, the last key and value column: as the oracle."""
    from oracle import sequence_oracle as R
    gen = torch.Generator().manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=gen)
    c = dict(q=rn(T, 1, 2, Dk).to(dtype), k=rn(T, 1, 2, Dk).to(dtype), v=rn(T, 1, 2, Dv).to(dtype), state=rn(1, 2, Dk, Dv),
             dout=rn(T, 1, 2, Dv).to(dtype), dfinal=rn(1, 2, Dk, Dv))
    if what in ("state", "dfinal"):
        c[what][0, 1, -1, -1] = float("inf")
        c[what][0, 0, 0, -2] = float("nan")
    else:
        c[what][T // 2, 0, 1, -1] = float("inf")
        c[what][T // 2 + 3, 0, 0, 0] = float("nan")
    ld = torch.tensor([-0.3, -0.01])
    starts = torch.zeros(T, 1, dtype=torch.uint8)
    starts[T // 4] = starts[3 * T // 4] = 1
    d = {n: x.to(DEV) for n, x in c.items()}
    leaves = [d[n].requires_grad_() for n in ("q", "k", "v", "state")]
    out, final = _seq().linear_attention(*leaves[:3], ld.to(DEV), leaves[3], starts.to(DEV))
    got = (out, final) + torch.autograd.grad([out, final], leaves, [d["dout"], d["dfinal"]])
    ref = R.linear_attention(c["q"], c["k"], c["v"], ld, c["state"], starts, None, c["dout"], c["dfinal"])
    for name, g, r in zip(("out", "final", "dq", "dk", "dv", "dstate"), got, ref):
        wrong = g.cpu().isfinite() != r.isfinite()
        assert not bool(wrong.any()), "%s: %d of %d, first at %s" % (name, int(wrong.sum()), wrong.numel(),
                                                                     wrong.nonzero()[0].tolist())

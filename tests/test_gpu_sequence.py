"""GPU: linear attention with a decay per head (sequence.py) against the float64 oracle.

Tolerances.  Every output is a sum of products of the inputs with weights g^m.  In float32 arithmetic its error is at
most K 2^-24 times the same sum over the inputs' absolute values ("bulk", from the oracle on absolute values), where
K counts the roundings a product goes through: at most Dk + Dv for the dot products, one per token for the state
(T + 64 with the block sums), a handful for the weight; on top comes half a step of the output's own type.  The
16-bit types' two-term operands are exact to 2^-16 of a term, which their outputs' tolerance counts as 2^-15 bulk; the
states' operands are exact.
"""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _seq():
    from tum_adlr_deep_reinforcement_learning_amd import sequence
    return sequence


def _case(T, N, H, Dk, Dv, dtype, seed=0, starts=0.0, lengths=None, state=True, tau=30.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    c = dict(q=(rn(T, N, H, Dk) * Dk ** -0.5).to(dtype), k=rn(T, N, H, Dk).to(dtype), v=rn(T, N, H, Dv).to(dtype),
             log_decay=-torch.rand(H, generator=gen) * 4 / tau - 1 / tau)
    c["state"] = rn(N, H, Dk, Dv) if state else None
    c["starts"] = (torch.rand(T, N, generator=gen) < starts).to(torch.uint8) if starts else None
    c["lengths"] = torch.tensor(lengths, dtype=torch.int32) if lengths is not None else None
    c["dout"], c["dfinal"] = rn(T, N, H, Dv).to(dtype), rn(N, H, Dk, Dv)
    return c


def _dev(c):
    return {k: v.to(DEV) if v is not None else None for k, v in c.items()}


def _oracle(c, grad):
    a = [c["q"], c["k"], c["v"], c["log_decay"], c["state"], c["starts"], c["lengths"]]
    b = [x.abs() if x is not None and i in (0, 1, 2, 4) else x for i, x in enumerate(a)]
    if not grad:
        return R.linear_attention(*a), R.linear_attention(*b)
    return R.linear_attention(*a, c["dout"], c["dfinal"]), \
        R.linear_attention(*b, c["dout"].abs(), c["dfinal"].abs())


def _close(name, got, ref, bulk, steps):
    dt = got.dtype
    assert got.shape == ref.shape, name
    tol = steps * 2.0 ** -24 * bulk
    if dt != torch.float32:
        tol = tol + 2.0 ** -15 * bulk
    tol = tol + torch.finfo(dt).eps / 2 * (ref.abs() + tol) + torch.finfo(dt).tiny
    err = (got.detach().cpu().double() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, worst %.3g times its tolerance" % (
        name, int(bad.sum()), bad.numel(), float((err / tol).max()))


def _check(c, grad=True, view=lambda x: x):
    s = _seq()
    d = _dev(c)
    T, N, H, Dk = c["q"].shape
    steps = T + 64 + Dk + c["v"].shape[3]
    q, k, v = (view(d[x]) for x in "qkv")
    leaves = [x.detach().requires_grad_(grad) for x in (q, k, v)]
    st = d["state"].requires_grad_(grad) if d["state"] is not None else None
    out, final = s.linear_attention(*leaves, d["log_decay"], st, d["starts"], d["lengths"])
    ref, bulk = _oracle(c, grad)
    _close("out", out, ref[0], bulk[0], steps)
    _close("final_state", final, ref[1], bulk[1], steps)
    if not grad:
        return
    wrt = leaves + ([st] if st is not None else [])
    grads = torch.autograd.grad([out, final], wrt, [d["dout"], d["dfinal"]])
    for i, name in enumerate(["dq", "dk", "dv", "dstate"][:len(wrt)]):
        _close(name, grads[i], ref[2 + i], bulk[2 + i], steps)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(16, 16), (64, 64), (128, 128), (32, 64), (128, 16), (16, 128), (20, 40), (1, 1),
                                   (7, 33), (96, 80), (127, 65)])
def test_head_sizes(Dk, Dv, dtype):
    _check(_case(50, 3, 2, Dk, Dv, dtype, seed=Dk * 131 + Dv, starts=0.05))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100])
def test_lengths_of_time(T, dtype):
    _check(_case(T, 2, 3, 32, 16, dtype, seed=T))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("state", [False, True])
def test_time_segments(state, dtype):
    """Few sequences, a long time axis: the scan is cut into segments and joined."""
    _check(_case(1100, 1, 2, 32, 48, dtype, seed=5, starts=0.004, state=state, tau=200.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_time_segments_with_lengths(dtype):
    _check(_case(700, 3, 1, 64, 64, dtype, seed=6, starts=0.01, lengths=[700, 130, 0]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_token_a_start_and_none(dtype):
    c = _case(40, 2, 2, 16, 32, dtype, seed=8)
    c["starts"] = torch.zeros(40, 2, dtype=torch.uint8)
    c["starts"][:, 0] = 255  # any value but 0
    _check(c)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_with_garbage_behind_them(dtype):
    """Rows behind a length may hold anything, NaN too: they are not read into any result."""
    lengths = [0, 1, 16, 37, 70, 70, 500, -3]  # beyond T and below 0: clamped
    c = _case(70, 8, 2, 32, 32, dtype, seed=9, starts=0.05, lengths=lengths)
    clean = {k: v.clone() if v is not None else None for k, v in c.items()}
    for n, m in enumerate(lengths):
        for x in ("q", "k", "v", "dout"):
            clean[x][max(m, 0):, n] = 0
            c[x][max(m, 0):, n] = float("nan")
    s, d = _seq(), _dev(c)
    leaves = [d[x].requires_grad_() for x in ("q", "k", "v", "state")]
    out, final = s.linear_attention(*leaves[:3], d["log_decay"], leaves[3], d["starts"], d["lengths"])
    grads = torch.autograd.grad([out, final], leaves, [d["dout"], d["dfinal"]])
    ref, bulk = _oracle(clean, True)
    for name, got, r, b in zip(["out", "final", "dq", "dk", "dv", "dstate"], (out, final) + grads, ref, bulk):
        _close(name, got, r, b, 70 + 64 + 64)
    for n, m in enumerate(lengths):
        assert not bool(out[max(m, 0):, n].any()) and not bool(grads[0][max(m, 0):, n].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["q", "k", "v", "state"])
def test_nan_reaches_only_what_the_recurrence_lets_it(what, dtype):
    """A NaN at token 37 of one head, an episode start at 45: which outputs are NaN is the oracle's answer."""
    c = _case(60, 2, 2, 16, 32, dtype, seed=10)
    c["starts"] = torch.zeros(60, 2, dtype=torch.uint8)
    c["starts"][45, 0] = 1
    if what == "state":
        c["state"][0, 1, 3, 5] = float("nan")
    else:
        c[what][37, 0, 1, 3] = float("nan")
    s, d = _seq(), _dev(c)
    out, final = s.linear_attention(d["q"], d["k"], d["v"], d["log_decay"], d["state"], d["starts"])
    ref, _ = _oracle(c, False)
    assert torch.equal(out.isnan().cpu(), ref[0].isnan()) and torch.equal(final.isnan().cpu(), ref[1].isnan())
    clean = _case(60, 2, 2, 16, 32, dtype, seed=10)
    clean["starts"] = c["starts"]
    (ro, rf), (bo, bf) = _oracle(clean, False)
    ok = ~ref[0].isnan()
    for got, r, b, m in ((out, ro, bo, ok), (final, rf, bf, ~ref[1].isnan())):
        _close(what, torch.where(m.to(DEV), got, 0), torch.where(m, r, 0), b, 60 + 64 + 48)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    """Batch-major, head-major and offset views, and rows that are not 16-byte aligned."""
    _check(_case(37, 3, 2, 16, 16, dtype, seed=11), view=lambda x: x.transpose(0, 1).contiguous().transpose(0, 1))
    _check(_case(37, 3, 2, 16, 16, dtype, seed=12), view=lambda x: x.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3))

    def odd(x):
        y = torch.zeros(x.shape[:3] + (x.shape[3] + 5,), dtype=x.dtype, device=x.device)
        y[..., 3:-2] = x
        return y[..., 3:-2]
    _check(_case(37, 3, 2, 16, 48, dtype, seed=13), view=odd)
    _check(_case(37, 3, 2, 16, 48, dtype, seed=14), view=lambda x: x.transpose(2, 3).contiguous().transpose(2, 3))
    _check(_case(37, 3, 2, 16, 48, dtype, seed=15), view=lambda x: x.flip(0).contiguous().flip(0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_shared_heads(dtype):
    """q and k broadcast over the heads (stride 0): their gradient is the sum over the heads."""
    c = _case(45, 2, 4, 16, 16, dtype, seed=16)
    for x in "qk":
        c[x] = c[x][:, :, :1].expand(45, 2, 4, 16)
    s, d = _seq(), _dev({k: (v[:, :, :1] if k in "qk" and v is not None else v) for k, v in c.items()})
    q, k = d["q"].requires_grad_(), d["k"].requires_grad_()
    out, final = s.linear_attention(q.expand(45, 2, 4, 16), k.expand(45, 2, 4, 16), d["v"], d["log_decay"], d["state"])
    ref, bulk = _oracle(c, True)
    _close("out", out, ref[0], bulk[0], 45 + 64 + 32)
    grads = torch.autograd.grad([out, final], [q, k], [d["dout"], d["dfinal"]])
    for g, r, b in zip(grads, ref[2:4], bulk[2:4]):
        # the heads' gradients are rounded to the type one by one before the framework's sum (4 roundings + the sum's)
        eps = torch.finfo(dtype).eps
        err = (g.cpu().double() - r.sum(2, keepdim=True)).abs()
        assert bool((err <= 4 * eps * b.sum(2, keepdim=True) + 2.0 ** -14 * b.sum(2, keepdim=True)).all())


def test_decay_bounds():
    """No decay (1), and a decay so strong that the memory is the last token."""
    c = _case(60, 2, 3, 16, 16, torch.float32, seed=17)
    c["log_decay"] = torch.tensor([0.0, -50.0, -float("inf")])
    _check(c)


def test_empty():
    s = _seq()
    z = lambda *a: torch.zeros(*a, device=DEV)
    ld = torch.tensor([-0.1, -0.2], device=DEV)
    st = torch.randn(3, 2, 4, 5, device=DEV)
    out, final = s.linear_attention(z(0, 3, 2, 4), z(0, 3, 2, 4), z(0, 3, 2, 5), ld, st)
    assert out.shape == (0, 3, 2, 5) and torch.equal(final, st)
    out, final = s.linear_attention(z(0, 3, 2, 4), z(0, 3, 2, 4), z(0, 3, 2, 5), ld)
    assert not bool(final.any())
    out, final = s.linear_attention(z(7, 0, 2, 4), z(7, 0, 2, 4), z(7, 0, 2, 5), ld)
    assert out.shape == (7, 0, 2, 5) and final.shape == (0, 2, 4, 5)
    q = z(0, 3, 2, 4).requires_grad_()
    st.requires_grad_()
    out, final = s.linear_attention(q, z(0, 3, 2, 4), z(0, 3, 2, 5), ld, st)
    g = torch.autograd.grad(final, [q, st], torch.ones_like(final))
    assert g[0].shape == q.shape and torch.equal(g[1], torch.ones_like(st))
    out = s.linear_attention_step(z(0, 2, 4), z(0, 2, 4), z(0, 2, 5), ld, z(0, 2, 4, 5))
    assert out.shape == (0, 2, 5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,Dk,Dv", [(1, 1, 1, 1), (5, 2, 16, 16), (3, 4, 64, 64), (2, 3, 128, 128), (7, 1, 20, 40),
                                       (3, 2, 33, 7), (67, 4, 16, 16), (2, 2, 5, 126), (9, 1, 128, 4)])
def test_step(N, H, Dk, Dv, dtype):
    c = _case(1, N, H, Dk, Dv, dtype, seed=Dk + Dv)
    c["starts"] = torch.zeros(1, N, dtype=torch.uint8)
    c["starts"][0, ::3] = 1
    s, d = _seq(), _dev(c)
    ref, bulk = _oracle(c, False)
    other = torch.full_like(d["state"], float("nan"))
    args = (d["q"][0], d["k"][0], d["v"][0], d["log_decay"])
    out = s.linear_attention_step(*args, d["state"], d["starts"][0], state_out=other)
    assert torch.equal(d["state"].cpu(), c["state"])
    _close("out", out, ref[0][0], bulk[0][0], Dk + 16)
    _close("state", other, ref[1], bulk[1], 16)
    again = s.linear_attention_step(*args, d["state"], d["starts"][0].bool())  # in place
    assert torch.equal(again, out) and torch.equal(d["state"], other)


def test_step_ignores_the_state_of_a_started_row():
    s, d = _seq(), _dev(_case(1, 4, 2, 16, 16, torch.float32))
    d["state"][1] = float("nan")
    x = torch.tensor([0, 1, 0, 0], dtype=torch.uint8, device=DEV)
    out = s.linear_attention_step(d["q"][0], d["k"][0], d["v"][0], d["log_decay"], d["state"], x)
    assert not bool(out.isnan().any()) and not bool(d["state"].isnan().any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_one_by_one_equal_the_blocks(dtype):
    """A prompt through linear_attention, then single tokens, against one call over everything."""
    c = _case(90, 3, 2, 32, 32, dtype, seed=20, starts=0.05)
    s, d = _seq(), _dev(c)
    ref, bulk = _oracle(c, False)
    out, state = s.linear_attention(d["q"][:70], d["k"][:70], d["v"][:70], d["log_decay"], d["state"], d["starts"][:70])
    outs = [out]
    for t in range(70, 90):
        outs.append(s.linear_attention_step(d["q"][t], d["k"][t], d["v"][t], d["log_decay"], state, d["starts"][t])[None])
    _close("out", torch.cat(outs), ref[0], bulk[0], 90 + 64 + 64)
    _close("state", state, ref[1], bulk[1], 90 + 64 + 64)


def test_gradient_against_differences():
    """d loss = <gradient, direction> for a small step in each input, float32 (quadratic error cancelled by a central
    difference; the loss is linear in each input, so the difference is exact up to float32 rounding)."""
    c = _case(48, 2, 2, 16, 16, torch.float32, seed=21, starts=0.05)
    s, d = _seq(), _dev(c)
    leaves = [d[x].requires_grad_() for x in ("q", "k", "v", "state")]

    def loss(xs):
        out, final = s.linear_attention(xs[0], xs[1], xs[2], d["log_decay"], xs[3], d["starts"])
        return (out.double() * d["dout"]).sum() + (final.double() * d["dfinal"]).sum()
    grads = torch.autograd.grad(loss(leaves), leaves)
    for i in range(4):
        step = torch.randn_like(leaves[i]) * 0.5
        hi, lo = list(leaves), list(leaves)
        hi[i], lo[i] = leaves[i] + step, leaves[i] - step
        with torch.no_grad():
            diff = (loss(hi) - loss(lo)) / 2
        # float32 roundings of about 1e4 outputs of size about 10, weighted by numbers of size 1
        assert abs(float(diff - (grads[i].double() * step).sum())) < 1e-3 * (1 + abs(float(diff)))


def test_results_repeat_bit_for_bit():
    c = _dev(_case(300, 2, 2, 64, 64, torch.bfloat16, seed=22, starts=0.02))
    s = _seq()
    leaves = [c[x].requires_grad_() for x in ("q", "k", "v", "state")]

    def go():
        out, final = s.linear_attention(*leaves[:3], c["log_decay"], leaves[3], c["starts"])
        return [out, final] + list(torch.autograd.grad([out, final], leaves, [c["dout"], c["dfinal"]]))
    a, b = go(), go()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_stream_and_capture():
    """On a side stream, and captured into two graphs whose workspaces are their own; replayed in turn with eager
    work between."""
    s = _seq()
    cs = [_dev(_case(600, 1, 2, 32, 32, torch.float32, seed=30 + i, tau=100.0)) for i in range(2)]
    call = lambda c: s.linear_attention(c["q"], c["k"], c["v"], c["log_decay"], c["state"])
    with torch.no_grad():
        want = [call(c) for c in cs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call(cs[0])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1])
        graphs, outs = [], []
        for c in cs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(c))
            graphs.append(g)
        for _ in range(3):
            for g in graphs:
                g.replay()
            eager = call(cs[0])
            torch.cuda.synchronize()
            assert torch.equal(eager[0], want[0][0])
            for o, w in zip(outs, want):
                assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
                o[0].zero_(), o[1].zero_()


def test_refusals():
    s = _seq()
    z = lambda *a, **k: torch.zeros(*a, device=DEV, **k)
    ld = z(2)
    q, v = z(4, 3, 2, 8), z(4, 3, 2, 8)
    bad = [
        dict(k=z(4, 3, 2, 9)), dict(v=z(4, 3, 1, 8)), dict(q=q.cpu()), dict(q=q.double()), dict(v=v.half()),
        dict(q=z(4, 3, 2, 129), k=z(4, 3, 2, 129)), dict(v=z(4, 3, 2, 129)), dict(q=z(4, 3, 16)),
        dict(log_decay=z(3)), dict(log_decay=ld.double()), dict(log_decay=ld.clone().requires_grad_()),
        dict(initial_state=z(3, 2, 8, 9)), dict(initial_state=z(3, 2, 8, 8).half()),
        dict(episode_starts=z(4, 3)), dict(episode_starts=z(3, 4, dtype=torch.uint8)),
        dict(lengths=z(3)), dict(lengths=z(4, dtype=torch.int32)), dict(lengths=torch.zeros(3, dtype=torch.int32)),
    ]
    for b in bad:
        with pytest.raises(ValueError):
            s.linear_attention(**{**dict(q=q, k=q, v=v, log_decay=ld), **b})
    t = dict(q=q[0], k=q[0], v=v[0], log_decay=ld, state=z(3, 2, 8, 8))
    big = z(2 * 3 * 2 * 8 * 8)
    for b in [dict(q=q), dict(state=z(3, 2, 8, 9)), dict(state=z(3, 2, 8, 8).transpose(2, 3)),
              dict(state=z(3, 2, 8, 8).bfloat16()), dict(state_out=z(3, 2, 8, 9)),
              dict(state=big[1:385].view(3, 2, 8, 8)),
              dict(state=big[:384].view(3, 2, 8, 8), state_out=big[4:388].view(3, 2, 8, 8)),
              dict(episode_starts=z(3)), dict(q=q[0].clone().requires_grad_())]:
        with pytest.raises(ValueError):
            s.linear_attention_step(**{**t, **b})

"""GPU: group norm with an activation (sequence.py) against the float64 oracle.

Tolerances.  u = 2^-24.  With n values per group, x of size X around a mean: the mean is off by at most (n / threads +
log) u X and the deviations by u (|x| + |mean|) besides; sums run over at most 64 values per thread and then a tree, so
72 u covers a sum's relative error.  xh = d r is then off by e = 80 u (1 + |xh|)(1 + (|x| + |mean|) r), z by
|w| e + 2u |z|, y by 1.2 (an activation's steepest slope) times that + 8 u (|y| + 1) for the function itself, and half
a step of x's type.  The gradient's terms carry the same errors: dx within 400 u r (1 + X r) times the sums of absolute
terms, dweight and dbias within 400 u (1 + X r) sum |dy| (1 + |xh|)(1 + |w|).  For float32 a floor of 2^-24 of the
tensor's largest value is added.
"""
import pytest
import torch

from oracle import sequence_oracle as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "gelu", "tanh"]
U = 2.0 ** -24


def _seq():
    from tum_adlr_deep_reinforcement_learning_amd import sequence
    return sequence


def _half(t):
    return torch.finfo(t.dtype).eps / 2


def _check(N, L, C, G, dtype, act="silu", seed=0, affine=True, shift=0.5, wdtype=torch.float32, view=None, eps=1e-5,
           x=None):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)
    x = ((rn(N, L, C) * 1.5 + shift) if x is None else x).to(dtype)
    w = (1 + 0.3 * rn(C)).to(wdtype) if affine else None
    b = (0.3 * rn(C)).to(wdtype) if affine else None
    dy = rn(N, L, C).to(dtype)
    ref = R.group_norm_act(x, G, w, b, eps, act, dy)
    if act == "relu":  # the slope jumps at z = 0: keep the gradient's oracle away from it
        z = R.group_norm_act(x, G, w, b, eps, "none")
        dy = torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)
        ref = R.group_norm_act(x, G, w, b, eps, act, dy)
    s = _seq()
    put = (lambda t: t.to(DEV)) if view is None else (lambda t: view(t.to(DEV)))
    xd = put(x).requires_grad_()
    leaves = [xd] + [t.to(DEV).requires_grad_() for t in (w, b) if t is not None]
    y = s.group_norm_act(xd, G, *(leaves[1:] if affine else (None, None)), eps=eps, activation=act)
    grads = torch.autograd.grad(y, leaves, put(dy))
    with torch.no_grad():
        assert torch.equal(s.group_norm_act(xd, G, *(leaves[1:] if affine else (None, None)), eps=eps, activation=act), y)

    # sizes of the terms
    X = x.double()
    g4 = X.reshape(N, L, G, C // G)
    mean = g4.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(((g4 - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xh = ((g4 - mean) * r).reshape(N, L, C)
    size = ((g4.abs() + mean.abs()) * r)
    full = lambda t: t.expand(N, L, G, C // G).reshape(N, L, C)
    wa = w.double().abs() if affine else torch.ones(C, dtype=torch.double)
    z = R.group_norm_act(x, G, w, b, eps, "none")
    e = 80 * U * (1 + xh.abs()) * (1 + size.reshape(N, L, C))
    tol = 1.2 * (wa * e + 2 * U * z.abs()) + 8 * U * (ref[0].abs() + 1)
    _close("y", y, ref[0], tol)
    worst = full((1 + size).amax((1, 3), keepdim=True))
    a = (dy.double().abs() * 1.2 * wa).reshape(N, L, G, C // G)
    axh = xh.abs().reshape(N, L, G, C // G)
    terms = r * (a + a.mean((1, 3), keepdim=True) + axh * (a * axh).mean((1, 3), keepdim=True))
    _close("dx", grads[0], ref[1], 400 * U * worst * terms.reshape(N, L, C))
    if affine:
        t = (dy.double().abs() * (1 + xh.abs()) * (1 + wa) * worst).sum((0, 1))
        _close("dweight", grads[1], ref[2], 400 * U * t * (1 + xh.abs().max()))
        _close("dbias", grads[2], ref[3], 400 * U * t)


def _close(name, got, ref, tol):
    assert got.shape == ref.shape
    tol = tol + _half(got) * (ref.abs() + tol) + torch.finfo(got.dtype).tiny + U * float(ref.abs().max())
    err = (got.detach().cpu().double() - ref).abs()
    assert bool((err <= tol).all()), "%s: %d of %d off, worst %.3g times its tolerance" % (
        name, int((err > tol).sum()), err.numel(), float((err / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,L,C,G", [(1, 1, 1, 1), (8, 1, 64, 4), (1000, 1, 64, 4), (3, 1, 48, 3), (5, 1, 7, 7),
                                     (130, 1, 30, 3), (4, 1, 320, 32), (2, 5, 24, 3), (3, 17, 40, 4), (70, 3, 10, 5),
                                     (1, 1, 2048, 1), (2, 1, 1000, 1), (9, 64, 32, 32)])
def test_small_groups(N, L, C, G, dtype):
    _check(N, L, C, G, dtype, seed=N + L + C)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,L,C,G", [(3, 900, 40, 4), (2, 1000, 64, 4), (1, 4096, 16, 1), (5, 333, 21, 3), (2, 60, 512, 2),
                                     (1, 2, 3000, 1), (2, 9, 2050, 2), (1, 257, 33, 1)])
def test_groups_of_a_block(N, L, C, G, dtype):
    _check(N, L, C, G, dtype, seed=N + L + C)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,L,C,G", [(1, 20000, 16, 1), (2, 9000, 20, 2), (1, 9001, 15, 1), (1, 40, 5000, 1),
                                     (1, 7, 1500, 1), (1, 1, 1501, 1), (2, 3, 40002, 2)])
def test_groups_beyond_a_block(N, L, C, G, dtype):
    _check(N, L, C, G, dtype, seed=N + L + C)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(40, 1, 64, 4), (2, 300, 64, 4), (1, 9000, 24, 1)])
def test_activations(shape, act):
    _check(*shape, torch.float32, act=act, seed=3)
    _check(*shape, torch.bfloat16, act=act, seed=4)


def test_activation_tails():
    """z of +-100 and +-20: no overflow, the right limits, zero slope on the flat side."""
    s = _seq()
    x = torch.tensor([[-1.0, 1.0]], device=DEV).repeat(4, 1).requires_grad_()
    for scale in (20.0, 100.0):
        w = torch.full((2,), scale, device=DEV)
        for act in ACTS:
            y = s.group_norm_act(x, 1, w, activation=act)
            ref = R.group_norm_act(x[:, None], 1, w, act=act, dy=torch.ones(4, 1, 2))
            assert bool(y.isfinite().all())
            g, = torch.autograd.grad(y.sum(), x)
            assert float((y.cpu().double() - ref[0][:, 0]).abs().max()) < 1e-4 * scale
            assert float((g.cpu().double() - ref[1][:, 0]).abs().max()) < 1e-3


@pytest.mark.parametrize("shape", [(40, 1, 64, 4), (2, 300, 64, 4), (1, 9000, 24, 1)])
def test_large_mean_and_constant_rows(shape):
    _check(*shape, torch.float32, seed=5, shift=300.0)
    N, L, C, G = shape
    _check(*shape, torch.float32, seed=6, x=torch.full((N, L, C), 2.5))  # no spread: y = act(bias)


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16])
def test_parameter_types_and_none(wdtype):
    _check(50, 1, 64, 4, torch.bfloat16, wdtype=wdtype)
    _check(2, 300, 64, 4, torch.bfloat16, wdtype=wdtype)
    _check(50, 1, 64, 4, torch.bfloat16, affine=False)
    _check(1, 9000, 24, 1, torch.float32, affine=False)


def test_weight_without_bias_and_frozen_input():
    s = _seq()
    x, w = torch.randn(9, 5, 12, device=DEV), torch.randn(12, device=DEV, requires_grad=True)
    y = s.group_norm_act(x, 3, w, activation="none")
    g, = torch.autograd.grad(y, w, torch.ones_like(y))
    ref = R.group_norm_act(x, 3, w, act="none", dy=torch.ones(9, 5, 12))
    assert float((g.cpu().double() - ref[2]).abs().max()) < 1e-4
    y = s.group_norm_act(x, 3, None, w, activation="none")
    g, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(g, torch.full_like(g, 45.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,L,C,G", [(6, 5, 16, 2), (3, 300, 32, 2), (1, 9000, 24, 1)])
def test_strides(N, L, C, G, dtype):
    _check(N, L, C, G, dtype, view=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))

    def odd(t):
        y = torch.zeros(t.shape[:2] + (t.shape[2] + 3,), dtype=t.dtype, device=t.device)
        y[..., 1:-2] = t
        return y[..., 1:-2]
    _check(N, L, C, G, dtype, view=odd)
    _check(N, L, C, G, dtype, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))


def test_shapes_and_empty():
    s = _seq()
    x = torch.randn(2, 3, 4, 5, 8, device=DEV)
    y = s.group_norm_act(x, 2)
    assert y.shape == x.shape and torch.equal(y.view(2, 60, 8), s.group_norm_act(x.view(2, 60, 8), 2))
    rows = torch.randn(6, 8, device=DEV)
    assert torch.equal(s.group_norm_act(rows, 2), s.group_norm_act(rows[:, None], 2)[:, 0])
    w = torch.ones(8, device=DEV, requires_grad=True)
    for shape in ((0, 8), (0, 5, 8), (3, 0, 8)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        y = s.group_norm_act(e, 2, w)
        g = torch.autograd.grad(y.sum(), [e, w])
        assert y.shape == shape and g[0].shape == shape and not bool(g[1].any())


def test_gradient_against_differences():
    """float32, central differences of a smooth loss: error h^2 x third derivative + rounding / h."""
    s = _seq()
    gen = torch.Generator(device=DEV).manual_seed(1)
    rn = lambda *a: torch.randn(*a, device=DEV, generator=gen)
    x, w, b, dy = rn(7, 30, 24), rn(24), rn(24), rn(7, 30, 24)
    for act in ("silu", "gelu", "tanh", "none"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        f = lambda a: (s.group_norm_act(a[0], 3, a[1], a[2], activation=act).double() * dy).sum()
        grads = torch.autograd.grad(f(leaves), leaves)
        for i in range(3):
            d = rn(*leaves[i].shape)
            hi, lo = [t.detach() for t in leaves], [t.detach() for t in leaves]
            h = 1e-3
            hi[i], lo[i] = hi[i] + h * d, lo[i] - h * d
            diff = float((f(hi) - f(lo)) / (2 * h))
            assert abs(diff - float((grads[i].double() * d).sum())) < 2e-2 * (1 + abs(diff) * 1e-2)


@pytest.mark.parametrize("shape", [(3000, 1, 64, 4), (4, 900, 40, 4), (1, 20000, 16, 1)])
def test_repeats_other_stream_and_capture(shape):
    s = _seq()
    N, L, C, G = shape
    x = torch.randn(N, L, C, device=DEV, requires_grad=True)
    w, b, dy = torch.randn(C, device=DEV, requires_grad=True), torch.randn(C, device=DEV, requires_grad=True), \
        torch.randn(N, L, C, device=DEV)

    def go():
        y = s.group_norm_act(x, G, w, b)
        return [y.detach()] + list(torch.autograd.grad(y, [x, w, b], dy))
    want = go()
    assert all(torch.equal(p, q) for p, q in zip(want, go()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = go()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    del got
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = go()
    for _ in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(want, go()))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, outs))


def test_refusals():
    s = _seq()
    x = torch.zeros(4, 3, 12, device=DEV)
    z = lambda *a, **k: torch.zeros(*a, device=DEV, **k)
    for args, kw in [((x.cpu(), 3), {}), ((x.double(), 3), {}), ((x, 5), {}), ((x, 0), {}), ((z(12), 3), {}),
                     ((x, 3, z(11)), {}), ((x, 3, z(12).double()), {}), ((x, 3, z(12).half()), {}),
                     ((x.half(), 3, z(12), z(12).half()), {}), ((x, 3), dict(activation="swish")),
                     ((x, 3), dict(eps=-1.0)), ((x, 3), dict(eps=float("nan"))), ((x, 3, torch.zeros(12)), {})]:
        with pytest.raises(ValueError):
            s.group_norm_act(*args, **kw)

"""GPU: the sequence operators at their edges: what a start cuts in the gradients, offsets beyond 32 bits, views whose
strides mean nothing, a training step captured into graphs, sizes that divide unevenly among waves.  Tolerances as in
test_gpu_sequence.py and test_gpu_groupnorm.py, whose helpers these use."""
import pytest
import torch

from oracle import sequence_oracle as R
from test_gpu_groupnorm import _check as _check_norm
from test_gpu_sequence import DEV, DTYPES, _case, _check, _close, _dev, _oracle, _seq

pytestmark = pytest.mark.gpu


@pytest.fixture
def large():
    """Gives the memory of a test with large allocations back to the other tests."""
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("at", [0, 20, 31, 45])
def test_gradients_of_bad_numbers_end_at_the_start(what, dtype, at):
    """An infinity in the row of an episode start (and a NaN right behind it): the gradients of the rows before the
    start are finite and right, whatever that row holds."""
    c = _case(60, 2, 2, 16, 32, dtype, seed=40)
    c["starts"] = torch.zeros(60, 2, dtype=torch.uint8)
    c["starts"][at, 0] = 1
    clean = dict(c)
    clean[what] = c[what].clone()
    c[what] = c[what].clone()
    for t, x in ((at, float("inf")), (at + 1, float("nan"))):
        clean[what][t, 0, 1] = 0
        c[what][t, 0, 1] = x
    s, d = _seq(), _dev(c)
    leaves = [d[x].requires_grad_() for x in ("q", "k", "v", "state")]
    out, final = s.linear_attention(*leaves[:3], d["log_decay"], leaves[3], d["starts"])
    grads = torch.autograd.grad([out, final], leaves, [d["dout"], d["dfinal"]])
    ref, bulk = _oracle(clean, True)
    for name, got, r, b in zip(["out", "dq", "dk", "dv"], (out,) + grads[:3], (ref[0],) + ref[2:5], (bulk[0],) + bulk[2:5]):
        if at:
            _close(name, got[:at], r[:at], b[:at], 60 + 64 + 48)
        _close(name, got[:, 1], r[:, 1], b[:, 1], 60 + 64 + 48)
        _close(name, got[:, :, 0], r[:, :, 0], b[:, :, 0], 60 + 64 + 48)
    _close("dstate", grads[3], ref[5], bulk[5], 60 + 64 + 48)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(128, 80), (70, 100), (100, 70), (128, 33), (72, 128), (65, 127)])
def test_head_sizes_that_fill_no_slice(Dk, Dv, dtype):
    _check(_case(50, 2, 2, Dk, Dv, dtype, seed=41, starts=0.05, lengths=[50, 23]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_of_single_rows_mean_nothing(dtype):
    """One sequence, one head or one token, as views whose stride there is odd."""
    for shape in ((40, 1, 3, 32), (40, 3, 1, 32), (1, 5, 2, 32), (1, 1, 1, 32)):
        T, N, H, D = shape

        def view(x):
            y = x.contiguous()
            st = [7 if n == 1 else a for n, a in zip(y.shape, y.stride())]
            return y.as_strided(y.shape, st)
        _check(_case(T, N, H, D, D, dtype, seed=42), view=view)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("strides", ["tokens", "tokens far apart", "tokens at the limit", "tokens beyond it", "sequences"])
def test_offsets_beyond_32_bits(strides, dtype, large):
    """Views whose rows lie gigabytes apart (a block's rows are addressed by 32-bit offsets up to 2^26 elements apart)."""
    T, N, H, D = 70, 2, 2, 32
    st, sn = {"tokens": (2 ** 24 - 64, H * D), "tokens far apart": (2 ** 25 + 64, H * D), "sequences": (H * D, 2 ** 31),
              "tokens at the limit": (2 ** 26, H * D), "tokens beyond it": (2 ** 26 + 64, H * D)}[strides]
    n = (T - 1) * st + (N - 1) * sn + H * D

    def view(x):
        room = torch.empty(n, dtype=x.dtype, device=DEV)
        y = room.as_strided(x.shape, (st, sn, D, 1))
        y.copy_(x)
        return y
    _check(_case(T, N, H, D, D, dtype, seed=43, starts=0.05), view=view)


def test_states_beyond_32_bits(large):
    """70 000 states of 64 KB, in place; the last ones against the oracle."""
    N, D = 70000, 128
    gen = torch.Generator(device=DEV).manual_seed(1)
    state = torch.randn(N, 1, D, D, device=DEV, generator=gen)
    q, k, v = (torch.randn(N, 1, D, device=DEV, generator=gen) for _ in range(3))
    ld = torch.tensor([-0.3], device=DEV)
    pick = torch.tensor([0, 32767, 32768, 65535, 65536, N - 1], device=DEV)
    c = [x[pick].cpu() for x in (q, k, v, state)]
    out = _seq().linear_attention_step(q, k, v, ld, state)
    args = [c[0][None], c[1][None], c[2][None], ld.cpu(), c[3]]
    ref, bulk = R.linear_attention(*args), R.linear_attention(*[a.abs() if i != 3 else a for i, a in enumerate(args)])
    _close("out", out[pick], ref[0][0], bulk[0][0], D + 16)
    _close("state", state[pick], ref[1], bulk[1], 16)
    # and through whole columns of one token, from these states
    out2, final = _seq().linear_attention(q[None], k[None], v[None], ld, state)
    c = [x[pick].cpu() for x in (state,)]
    args[4] = c[0]
    ref, bulk = R.linear_attention(*args), R.linear_attention(*[a.abs() if i != 3 else a for i, a in enumerate(args)])
    _close("out", out2[0][pick], ref[0][0], bulk[0][0], D + 80)
    _close("state", final[pick], ref[1], bulk[1], 80)


def test_norm_offsets_beyond_32_bits(large):
    def view(x):
        N, L, C = x.shape
        room = torch.empty((N - 1) * 2 ** 31 + L * C, dtype=x.dtype, device=DEV)
        y = room.as_strided(x.shape, (2 ** 31, C, 1))
        y.copy_(x)
        return y
    _check_norm(3, 70, 64, 8, torch.bfloat16, view=view)
    _check_norm(3, 1, 64, 8, torch.bfloat16, view=view)
    _check_norm(2, 900, 64, 2, torch.bfloat16, view=view)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_in_graphs(dtype):
    """Memory and norm, forward and backward, captured twice into graphs that share a memory pool (so that the second
    capture reuses the first one's freed workspaces) and replayed in turn, on new inputs, with eager steps between."""
    s = _seq()
    T, N, H, D = 300, 2, 4, 32
    ld = torch.tensor([-0.5, -0.1, -0.02, -0.005], device=DEV)
    data = [torch.randn(T, N, 3, H, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)).to(dtype)
            for i in range(4)]
    starts = (torch.arange(T, device=DEV)[:, None] % 41 == torch.tensor([3, 17], device=DEV)).to(torch.uint8)
    w, b = torch.linspace(0.5, 1.5, H * D, device=DEV), torch.linspace(-1, 1, H * D, device=DEV)

    def step(x):
        x, wl, bl = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
        q, k, v = x.unbind(2)
        m, final = s.linear_attention(q, k, v, ld, None, starts)
        y = s.group_norm_act(m.reshape(T * N, H * D), H, wl, bl)
        loss = y.float().square().sum() + final.square().sum()
        return (y.detach(), final.detach()) + torch.autograd.grad(loss, [x, wl, bl])
    want = [step(x) for x in data]
    slots = [torch.empty_like(data[0]).copy_(data[0]) for _ in range(2)]
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for x in slots:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(x))
        graphs.append(g)
    for turn in range(4):
        for x, g, o in zip(slots, graphs, outs):
            x.copy_(data[turn])
            g.replay()
            eager = step(data[(turn + 1) % 4])
            torch.cuda.synchronize()
            assert all(torch.equal(p, r) for p, r in zip(o, want[turn]))
            assert all(torch.equal(p, r) for p, r in zip(eager, want[(turn + 1) % 4]))


def test_two_streams_at_once():
    """The same operators with their workspaces on two streams, queued without waiting."""
    s = _seq()
    cs = [_dev(_case(800, 1, 2, 64, 64, torch.bfloat16, seed=50 + i, tau=200.0)) for i in range(2)]
    x = [torch.randn(4, 9000, 64, device=DEV) for _ in range(2)]

    def go(i):
        c = cs[i]
        leaves = [c[n].detach().requires_grad_() for n in ("q", "k", "v")]
        out, final = s.linear_attention(*leaves, c["log_decay"], c["state"])
        y = x[i].detach().requires_grad_()
        z = s.group_norm_act(y, 2)
        return [out.detach(), final.detach(), z.detach()] + list(torch.autograd.grad([out, z], leaves + [y], [c["dout"], z.detach()]))
    want = [go(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(go(i))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(p, r) for p, r in zip(g, w))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 2), (3, 9), (4, 4), (5, 8), (7, 17), (9, 31), (17, 65), (66, 127), (127, 64), (101, 97)])
def test_rows_of_any_length_and_address(Dk, Dv, dtype):
    """Rows that are no whole vectors, packed and behind one odd element."""
    _check(_case(75, 2, 2, Dk, Dv, dtype, seed=Dk, starts=0.05, lengths=[75, 38]))

    def odd(x):
        y = torch.full((x.numel() + 1,), float("nan"), dtype=x.dtype, device=DEV)
        y[1:] = x.reshape(-1)
        return y[1:].view(x.shape)
    _check(_case(34, 3, 1, Dk, Dv, dtype, seed=Dv), view=odd)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,Dk,Dv", [(3, 2, 9, 1), (2, 2, 70, 2), (5, 1, 128, 3), (3, 2, 8, 5), (2, 3, 20, 17), (70, 2, 64, 35),
                                       (2, 2, 128, 69), (40, 4, 100, 101), (3000, 1, 10, 127), (700, 3, 33, 33)])
def test_step_rows_of_any_length(N, H, Dk, Dv, dtype):
    c = _case(1, N, H, Dk, Dv, dtype, seed=Dv, starts=0.2)
    s, d = _seq(), _dev(c)
    ref, bulk = _oracle(c, False)
    out = s.linear_attention_step(d["q"][0], d["k"][0], d["v"][0], d["log_decay"], d["state"], d["starts"][0])
    _close("out", out, ref[0][0], bulk[0][0], Dk + 16)
    _close("state", d["state"], ref[1], bulk[1], 16)


def test_second_derivatives_are_refused():
    """A graph of the gradients can be asked for (another term of the loss may want one), but not run through them."""
    s = _seq()
    d = _dev(_case(20, 2, 2, 8, 8, torch.float32, seed=60))
    q = d["q"].requires_grad_()
    out, _ = s.linear_attention(q, d["k"], d["v"], d["log_decay"])
    plain, = torch.autograd.grad(out, q, d["dout"], retain_graph=True)
    g, = torch.autograd.grad(out, q, d["dout"].requires_grad_(), create_graph=True)
    assert torch.equal(g, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), d["dout"])
    x = torch.randn(6, 16, device=DEV, requires_grad=True)
    dy = torch.randn(6, 16, device=DEV)
    y = s.group_norm_act(x, 4)
    plain, = torch.autograd.grad(y, x, dy, retain_graph=True)
    g, = torch.autograd.grad(y, x, dy.requires_grad_(), create_graph=True)
    assert torch.equal(g, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), dy)


@pytest.mark.parametrize("backward", [False, True])
def test_accumulated_gradients_and_a_captured_step(backward):
    """Leaves that an eager step gave gradients, its graph gone: a captured forward (and backward) on them replays right."""
    s = _seq()
    d = _dev(_case(64, 2, 2, 16, 16, torch.float32, seed=61))
    leaves = [d[n].requires_grad_() for n in ("q", "k", "v")]

    def step():
        out, final = s.linear_attention(*leaves, d["log_decay"], d["state"], None)
        if not backward:
            return [out.detach(), final.detach()]
        return list(torch.autograd.grad([out, final], leaves, [d["dout"], d["dfinal"]]))
    out, final = s.linear_attention(*leaves, d["log_decay"], d["state"], None)
    torch.autograd.backward([out, final], [d["dout"], d["dfinal"]])
    del out, final
    want = step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(again, want))

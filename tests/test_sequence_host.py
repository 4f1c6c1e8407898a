"""CPU: the oracle of the sequence operators against differences and a second formula, the structs against the header,
and every refusal that needs no device (the C entries check before they launch)."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from oracle import sequence_oracle as R
from tum_adlr_deep_reinforcement_learning_amd import _native, sequence

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = 4096  # a "pointer" that is never followed: every call below is refused before a launch


def _rand(*shape, seed=0):
    return torch.randn(*shape, dtype=torch.double, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------ the oracle
def test_oracle_is_the_decayed_sum():
    """out_t = sum over s <= t, with no start in (s, t], of g^(t-s) (q_t . k_s) v_s."""
    T, N, H, Dk, Dv = 13, 2, 2, 3, 4
    q, k, v, ld = _rand(T, N, H, Dk), _rand(T, N, H, Dk, seed=1), _rand(T, N, H, Dv, seed=2), torch.tensor([-0.3, -0.05])
    starts = torch.zeros(T, N, dtype=torch.uint8)
    starts[4, 0] = starts[9, 0] = starts[0, 1] = 1
    out, final = R.linear_attention(q, k, v, ld, None, starts)
    want = torch.zeros_like(out)
    for t in range(T):
        for s in range(t + 1):
            clear = (starts[s + 1:t + 1].sum(0) == 0).double()[:, None, None]
            g = torch.exp(ld.double() * (t - s))[None, :, None]
            want[t] += clear * g * (q[t] * k[s]).sum(-1, keepdim=True) * v[s]
    assert float((out - want).abs().max()) < 1e-12
    assert float(((q[-1][..., None] * final).sum(-2) - out[-1]).abs().max()) < 1e-12


@pytest.mark.parametrize("lengths", [None, [9, 4, 0]])
def test_oracle_gradients_against_differences(lengths):
    T, N, H, Dk, Dv = 9, 3, 2, 3, 2
    xs = [_rand(T, N, H, Dk), _rand(T, N, H, Dk, seed=1), _rand(T, N, H, Dv, seed=2), _rand(N, H, Dk, Dv, seed=3)]
    ld = torch.tensor([-0.3, -0.05])
    starts = (_rand(T, N, seed=4) > 1).to(torch.uint8)
    lens = torch.tensor(lengths) if lengths else None
    dout, dfinal = _rand(T, N, H, Dv, seed=5), _rand(N, H, Dk, Dv, seed=6)
    if lens is not None:
        dout = torch.where((torch.arange(T)[:, None] < lens)[..., None, None], dout, torch.zeros_like(dout))

    def loss(a):
        out, final = R.linear_attention(a[0], a[1], a[2], ld, a[3], starts, lens)
        return float((out * dout).sum() + (final * dfinal).sum())
    grads = R.linear_attention(xs[0], xs[1], xs[2], ld, xs[3], starts, lens, dout, dfinal)[2:]
    for i in range(4):
        step = _rand(*xs[i].shape, seed=7)
        hi, lo = list(xs), list(xs)
        hi[i], lo[i] = xs[i] + step, xs[i] - step  # the loss is linear in each input
        diff = (loss(hi) - loss(lo)) / 2
        assert abs(diff - float((grads[i] * step).sum())) < 1e-10 * (1 + abs(diff))


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "tanh"])
def test_norm_oracle_against_differences(act):
    x, w, b, dy = _rand(3, 5, 8), _rand(8, seed=1), _rand(8, seed=2), _rand(3, 5, 8, seed=3)
    _, dx, dw, db = R.group_norm_act(x, 2, w, b, 1e-5, act, dy)
    h = 1e-5
    for i, g in ((0, dx), (1, dw), (2, db)):
        a = [x, w, b]
        step = _rand(*a[i].shape, seed=4)
        f = lambda s: float((R.group_norm_act(*[t if j != i else t + s * step for j, t in enumerate(a)][:1], 2,
                                              *[t if j != i else t + s * step for j, t in enumerate(a)][1:], 1e-5, act)
                             * dy).sum())
        diff = (f(h) - f(-h)) / (2 * h)
        # rounding 1e-16 x about 100 / h, curvature h^2
        assert abs(diff - float((g * step).sum())) < 1e-7 * (1 + abs(diff))


def test_norm_oracle_is_group_norm():
    x, w, b = _rand(4, 6, 12), _rand(12, seed=1), _rand(12, seed=2)
    want = torch.nn.functional.group_norm(x.transpose(1, 2), 3, w, b, 1e-3).transpose(1, 2)
    assert float((R.group_norm_act(x, 3, w, b, 1e-3, "relu") - want.relu()).abs().max()) < 1e-12


# ------------------------------------------------------------------ structs
def test_struct_layout_matches_the_header(tmp_path):
    pairs = [("fw_seq_tensor", _native.FwSeqTensor), ("fw_linattn", _native.FwLinattn),
             ("fw_linattn_token", _native.FwLinattnToken), ("fw_rows", _native.FwRows),
             ("fw_group_norm", _native.FwGroupNorm)]
    lines = []
    for name, cls in pairs:
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f[0]) for f in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"fwrollout.h\"\nint main(void) {\n%s\n}\n"
                   % "\n".join(lines))
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def test_types_and_activations_match_the_header():
    text = open(os.path.join(ROOT, "include", "fwrollout.h")).read()
    codes = dict((a, int(b)) for a, b in re.findall(r"#define (FW_(?:DT|ACT)_\w+) (\d)", text))
    assert [sequence._DT[t] for t in (torch.float32, torch.bfloat16, torch.float16)] == \
        [codes["FW_DT_" + n] for n in ("F32", "BF16", "F16")]
    assert sequence._ACT == {n: codes["FW_ACT_" + n.upper()] for n in sequence._ACT}


# ------------------------------------------------------------------ refusals of the C entries
def _refused(fn, args, words):
    assert fn(ctypes.byref(args) if args is not None else None, None) == -1
    assert words in _native.last_error(), _native.last_error()


def _scan(**kw):
    a = _native.FwLinattn()
    a.T, a.N, a.H, a.Dk, a.Dv, a.dtype = 8, 2, 2, 16, 16, 0
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        s = getattr(a, n)
        s.p, s.st, s.sn, s.sh = BUF, 64, 32, 16
    a.log_decay = BUF
    for k, v in kw.items():
        if isinstance(v, tuple):
            for f, y in v:
                setattr(getattr(a, k), f, y)
        else:
            setattr(a, k, v)
    return a


NULL = (("p", None),)


@pytest.mark.parametrize("kw,words", [
    (dict(T=-1), "T and N"), (dict(N=-1), "T and N"), (dict(H=0), "H >= 1"), (dict(Dk=0), "head sizes"),
    (dict(Dk=129), "head sizes"), (dict(Dv=0), "head sizes"), (dict(Dv=129), "head sizes"), (dict(dtype=3), "dtype"),
    (dict(dtype=-1), "dtype"), (dict(q=NULL), "NULL q"), (dict(k=NULL), "NULL q, k"), (dict(v=NULL), "NULL q, k or v"),
    (dict(log_decay=None), "log_decay"), (dict(N=2 ** 40), "too many"), (dict(N=2 ** 30, H=1), "too many"),
    (dict(starts=BUF, starts_st=-1), "starts_st"), (dict(starts=BUF, starts_st=2 ** 26), "starts_st"),
    (dict(T=4096, N=1), "workspace"), (dict(T=4096, N=1, workspace=BUF, workspace_bytes=64), "workspace"),
    (dict(T=4096, N=1, workspace=BUF + 4, workspace_bytes=2 ** 40), "16-byte"),
])
def test_scan_refusals(kw, words):
    lib = _native.load()
    _refused(lib.fw_linattn_forward, _scan(**kw), words)
    _refused(lib.fw_linattn_backward, _scan(**kw), words)


def test_scan_refusals_of_one_direction():
    lib = _native.load()
    _refused(lib.fw_linattn_forward, None, "NULL")
    _refused(lib.fw_linattn_backward, None, "NULL")
    _refused(lib.fw_linattn_forward, _scan(out=NULL), "NULL out")
    for n in ("dout", "dq", "dk", "dv"):
        _refused(lib.fw_linattn_backward, _scan(**{n: NULL}), "NULL dout")
    for a in (_scan(N=0), _scan(N=0, T=0)):  # nothing to do
        assert lib.fw_linattn_forward(ctypes.byref(a), None) == 0
        assert lib.fw_linattn_backward(ctypes.byref(a), None) == 0


def test_scan_workspace():
    lib = _native.load()
    ws = lib.fw_linattn_workspace_bytes
    assert ws(8, 65536, 4, 16, 16, 0, 0) == 0          # enough sequences: no time segments
    assert ws(4096, 1, 4, 64, 64, 1, 0) > 0
    assert ws(4096, 1, 4, 64, 64, 1, 1) == 2 * ws(4096, 1, 4, 64, 64, 1, 0)
    assert ws(10 ** 9, 1, 1, 128, 128, 0, 1) < 2 ** 32  # bounded by the number of waves, not by the length
    for bad in ((0, 1, 1, 4, 4, 0, 0), (8, 0, 1, 4, 4, 0, 0), (8, 1, 0, 4, 4, 0, 0), (8, 1, 1, 0, 4, 0, 0),
                (8, 1, 1, 4, 200, 0, 0)):
        assert ws(*bad) == 0


def _token(**kw):
    a = _native.FwLinattnToken()
    a.N, a.H, a.Dk, a.Dv, a.dtype = 2, 2, 16, 16, 0
    for n in ("q", "k", "v", "out"):
        s = getattr(a, n)
        s.p, s.sn, s.sh = BUF, 32, 16
    a.log_decay, a.state, a.state_out = BUF, BUF, BUF
    for k, v in kw.items():
        if isinstance(v, tuple):
            setattr(getattr(a, k), "p", None)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,words", [
    (dict(N=-1), "N must be"), (dict(H=0), "H >= 1"), (dict(Dk=0), "head sizes"), (dict(Dk=129), "head sizes"),
    (dict(Dv=0), "head sizes"), (dict(Dv=129), "head sizes"), (dict(dtype=3), "dtype"), (dict(q=NULL), "NULL buffer"),
    (dict(out=NULL), "NULL buffer"), (dict(log_decay=None), "NULL buffer"), (dict(state=None), "NULL buffer"),
    (dict(state_out=None), "NULL buffer"), (dict(state=BUF + 4), "aligned"), (dict(state_out=BUF + 8), "aligned"),
    (dict(N=2 ** 40), "too many"), (dict(N=2 ** 30 - 1, H=1, Dk=100, Dv=100), "too many"),
])
def test_step_refusals(kw, words):
    lib = _native.load()
    _refused(lib.fw_linattn_step, _token(**kw), words)
    _refused(lib.fw_linattn_step, None, "NULL")
    assert lib.fw_linattn_step(ctypes.byref(_token(N=0)), None) == 0


def _norm(**kw):
    a = _native.FwGroupNorm()
    a.N, a.L, a.C, a.G, a.eps = 4, 3, 64, 4, 1e-5
    for n in ("x", "y", "dy", "dx"):
        s = getattr(a, n)
        s.p, s.sn, s.sl = BUF, 192, 64
    for k, v in kw.items():
        if isinstance(v, tuple):
            setattr(getattr(a, k), "p", None)
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,words", [
    (dict(N=-1), "multiple"), (dict(L=-1), "multiple"), (dict(C=0), "multiple"), (dict(G=0), "multiple"),
    (dict(G=5), "multiple"), (dict(dtype=3), "dtype"), (dict(wdtype=1), "wdtype"), (dict(act=5), "activation"),
    (dict(act=-1), "activation"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=NULL), "NULL x"),
    (dict(N=2 ** 40), "too many"), (dict(N=2 ** 24, L=600, C=64, G=1, workspace=BUF, workspace_bytes=2 ** 50,
                                         stats=BUF), "too many"),
])
def test_norm_refusals(kw, words):
    lib = _native.load()
    _refused(lib.fw_group_norm_forward, _norm(**kw), words)
    if "workspace" not in kw:
        kw = dict(kw, workspace=BUF, workspace_bytes=2 ** 50, stats=BUF)
    _refused(lib.fw_group_norm_backward, _norm(**kw), words)


def test_norm_refusals_of_one_direction():
    lib = _native.load()
    _refused(lib.fw_group_norm_forward, None, "NULL")
    _refused(lib.fw_group_norm_backward, None, "NULL")
    _refused(lib.fw_group_norm_forward, _norm(y=NULL), "NULL")
    _refused(lib.fw_group_norm_backward, _norm(dy=NULL), "NULL")
    _refused(lib.fw_group_norm_backward, _norm(dx=NULL), "NULL")
    _refused(lib.fw_group_norm_backward, _norm(), "workspace")
    _refused(lib.fw_group_norm_backward, _norm(L=0), "empty")
    large = dict(N=2, L=100000, C=64, G=4)
    _refused(lib.fw_group_norm_forward, _norm(**large), "workspace")
    _refused(lib.fw_group_norm_backward, _norm(**large), "stats")
    _refused(lib.fw_group_norm_backward, _norm(stats=BUF, **large), "workspace")
    for a in (_norm(N=0), _norm(L=0)):
        assert lib.fw_group_norm_forward(ctypes.byref(a), None) == 0
    assert lib.fw_group_norm_stats(ctypes.byref(_norm(**large))) == 1
    assert lib.fw_group_norm_stats(ctypes.byref(_norm())) == 0


# ------------------------------------------------------------------ refusals of the Python functions
def test_cpu_tensors_are_refused():
    z = torch.zeros
    ld = z(2)
    with pytest.raises(ValueError, match="on the GPU"):
        sequence.linear_attention(z(4, 3, 2, 8), z(4, 3, 2, 8), z(4, 3, 2, 8), ld)
    with pytest.raises(ValueError, match="on the GPU"):
        sequence.linear_attention_step(z(3, 2, 8), z(3, 2, 8), z(3, 2, 8), ld, z(3, 2, 8, 8))
    with pytest.raises(ValueError, match="on the GPU"):
        sequence.group_norm_act(z(4, 8), 2)
    with pytest.raises(ValueError, match=r"\[T, N, H, D\]"):
        sequence.linear_attention(z(4, 3, 8), z(4, 3, 8), z(4, 3, 8), ld)
    with pytest.raises(ValueError, match=r"\[N, \.\.\., C\]"):
        sequence.group_norm_act(z(8), 2)
    with pytest.raises(ValueError):
        sequence.linear_attention(None, None, None, ld)


def test_memory_policy_arguments():
    from tum_adlr_deep_reinforcement_learning_amd.rollout import RetentionActorCritic
    with pytest.raises(ValueError, match="heads"):
        RetentionActorCritic(14, 3, width=64, heads=5)
    p = RetentionActorCritic(14, 3)
    assert p.new_memory(5).shape == (5, 4, 16, 16)
    tau = -1.0 / p.log_decay
    assert abs(float(tau[0]) - 4.0) < 1e-5 and abs(float(tau[-1]) - 1000.0) < 1e-2 and bool((tau[1:] > tau[:-1]).all())
    assert RetentionActorCritic(14, 3, heads=1).log_decay.shape == (1,)
    assert "log_decay" in p.state_dict() and not any(n == "log_decay" for n, _ in p.named_parameters())

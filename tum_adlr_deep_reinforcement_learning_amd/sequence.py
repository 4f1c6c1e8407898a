"""Operators of a policy with memory, in the layouts of the rollout slab (time-major, heads and channels last).

  linear_attention       a decaying key-value memory per head over whole rollout columns [T][N], with resets at the
                         episode starts, ragged lengths, a state carried in and out, and gradients
  linear_attention_step  the same recurrence for one token per environment (the collect step)
  group_norm_act         group norm with an activation over channels-last rows or maps, with gradients

Every function launches on the current stream of its tensors' device, takes its workspace from torch's allocator on
that stream and never synchronises.  They may be captured into HIP graphs; torch.jit.trace is refused.  Tensors are
float32, bfloat16 or float16; states, statistics, sums and the gradients of parameters are float32.  There is no CPU
path: CPU tensors are refused.

The reference's policies are memoryless; these have no counterpart there.
"""
import ctypes
import functools
import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # include/fwrollout.h FW_DT_*
MAX_HEAD = 128


def _packer(cls):
    """A ctypes structure's fields as one struct.pack: a fifth of the time of setting them one by one, and a small call
    is bound by the host."""
    code = {ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_double: "d", ctypes.c_size_t: "N", ctypes.c_void_p: "P"}

    def flat(c):
        return "".join(code[t] if t in code else flat(t) for _, t in c._fields_)
    p = struct.Struct("@" + flat(cls))
    assert p.size == ctypes.sizeof(cls)
    return p.pack


_pack_linattn, _pack_token, _pack_norm = (_packer(c) for c in (_native.FwLinattn, _native.FwLinattnToken,
                                                               _native.FwGroupNorm))
_NO_ROWS = (0, 0, 0, 0)


def _ptr(t):
    return t.data_ptr() if t is not None else 0


def _launch(name, args, device):
    """lib.<name>(args, current stream) with `device` current, which it mostly is."""
    if torch._C._is_tracing():  # a trace would hold the allocation of the results and not what writes them
        raise RuntimeError("%s cannot be traced" % name)
    fn, i = getattr(_native.load(), name), device.index
    if torch._C._cuda_getDevice() == i:
        rc = fn(args, torch._C._cuda_getCurrentRawStream(i))
    else:
        with torch.cuda.device(device):
            rc = fn(args, torch._C._cuda_getCurrentRawStream(i))
    if rc:
        _native.check(rc, name)


def _once(backward):
    """once_differentiable, whose context is needed only where a graph of the gradients is asked for."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        if forward_ad._current_level >= 0:
            _no_tangents("the backward pass", *grads)
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


def _no_tangents(who, *tensors):
    """A tensor with a forward-mode tangent does not require a gradient: it would come out as a constant."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("%s has no forward-mode derivative" % who)


def _rows4(t):
    """The fields of an fw_seq_tensor for a [T][N][H][D] tensor with unit stride in D."""
    st = t.stride()
    return t.data_ptr(), st[0], st[1], st[2]


def _rows3(t):
    """The same for one token, [N][H][D]."""
    st = t.stride()
    return t.data_ptr(), 0, st[0], st[1]


def _dense(t):
    """Unit stride in the last dimension (a copy otherwise; broadcast leading dimensions stay views)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _heads(who, q, k, v, dims):
    try:
        dt, dev, sq, sv = q.dtype, q.get_device(), q.shape, v.shape
        if dev >= 0 and k.get_device() == dev == v.get_device() and dt in _DT and k.dtype is dt and v.dtype is dt and \
                len(sq) == dims and k.shape == sq and sv[:-1] == sq[:-1] and 1 <= sq[-1] <= MAX_HEAD and \
                1 <= sv[-1] <= MAX_HEAD and sq[-2] >= 1:
            return
    except (AttributeError, IndexError, TypeError):
        pass
    lay = "[T, N, H, D]" if dims == 4 else "[N, H, D]"  # what is wrong
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != dims:
            raise ValueError("%s: %s must be a %s tensor" % (who, name, lay))
        if t.device.type != "cuda":
            raise ValueError("%s: %s must be on the GPU (no CPU path exists)" % (who, name))
        if t.dtype not in _DT or t.dtype != q.dtype or t.device != q.device:
            raise ValueError("%s: q, k and v must share a device and one of float32, bfloat16, float16" % who)
    if q.shape != k.shape or q.shape[:-1] != v.shape[:-1]:
        raise ValueError("%s: q and k must have the same shape, v the same up to its last dimension; got %s %s %s"
                         % (who, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not (1 <= q.shape[-1] <= MAX_HEAD and 1 <= v.shape[-1] <= MAX_HEAD):
        raise ValueError("%s: head sizes must be 1..%d" % (who, MAX_HEAD))
    if q.shape[-2] < 1:
        raise ValueError("%s: at least one head" % who)


def _decay(who, log_decay, H, device):
    if not isinstance(log_decay, torch.Tensor) or log_decay.shape != (H,) or log_decay.dtype != torch.float32 or \
            log_decay.device != device:
        raise ValueError("%s: log_decay must be a float32 [H] tensor on the operands' device" % who)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s: log_decay is a fixed schedule and has no gradient; detach it" % who)
    return log_decay if log_decay.is_contiguous() else log_decay.contiguous()


def _starts(who, x, shape, device):
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.shape != shape or x.dtype not in (torch.uint8, torch.bool) or \
            x.device != device:
        raise ValueError("%s: episode_starts must be a uint8 or bool %s tensor on the operands' device"
                         % (who, list(shape)))
    return x


def _state(who, x, shape, device, name):
    if not isinstance(x, torch.Tensor) or x.shape != shape or x.dtype != torch.float32 or x.device != device:
        raise ValueError("%s: %s must be a float32 %s tensor on the operands' device" % (who, name, list(shape)))
    return x


def _step_state(who, x, shape, device, name):
    p = _state(who, x, shape, device, name).data_ptr()
    if p % 16 or not x.is_contiguous():
        raise ValueError("%s: %s must be contiguous and 16-byte aligned" % (who, name))
    return p


@functools.lru_cache(maxsize=256)
def _linattn_bytes(T, N, H, Dk, Dv, dtype, backward):  # of the sizes alone
    return _native.load().fw_linattn_workspace_bytes(T, N, H, Dk, Dv, dtype, backward)


def _linattn_head(q, v):
    T, N, H, Dk = q.shape
    return T, N, H, Dk, v.shape[3], _DT[q.dtype]


def _linattn_masks(log_decay, starts, lengths):
    if starts is None:
        return log_decay.data_ptr(), 0, 0, 0, _ptr(lengths)
    st = starts.stride()
    return log_decay.data_ptr(), starts.data_ptr(), st[0], st[1], _ptr(lengths)


def _workspace(n, device):
    # referenced until the launches are queued; the allocator reuses it in stream order
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _linattn_forward(q, k, v, log_decay, state, starts, lengths):
    head = T, N, H, Dk, Dv, code = _linattn_head(q, v)
    out = v.new_empty((T, N, H, Dv))
    final = log_decay.new_empty((N, H, Dk, Dv))
    n = _linattn_bytes(T, N, H, Dk, Dv, code, 0)
    ws = _workspace(n, q.device)
    _launch("fw_linattn_forward",
            _pack_linattn(*head, *_rows4(q), *_rows4(k), *_rows4(v), *_rows4(out),
                          *_linattn_masks(log_decay, starts, lengths), _ptr(state), final.data_ptr(),
                          *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, *_NO_ROWS, 0, 0, _ptr(ws), n), q.device)
    return out, final


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, starts, lengths):
        out, final = _linattn_forward(q, k, v, log_decay, state, starts, lengths)
        ctx.save_for_backward(q, k, v, log_decay, state, starts, lengths)
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    @_once
    def backward(ctx, dout, dfinal):
        q, k, v, log_decay, state, starts, lengths = ctx.saved_tensors
        head = T, N, H, Dk, Dv, code = _linattn_head(q, v)
        dout = _dense(dout) if dout is not None else v.new_zeros((T, N, H, Dv))
        dfinal = dfinal.contiguous() if dfinal is not None else None
        dq, dk, dv = q.new_empty((T, N, H, Dk)), k.new_empty((T, N, H, Dk)), v.new_empty((T, N, H, Dv))
        dstate = torch.empty_like(state) if state is not None and ctx.needs_input_grad[4] else None
        n = _linattn_bytes(T, N, H, Dk, Dv, code, 1)
        ws = _workspace(n, q.device)
        _launch("fw_linattn_backward",
                _pack_linattn(*head, *_rows4(q), *_rows4(k), *_rows4(v), *_NO_ROWS,
                              *_linattn_masks(log_decay, starts, lengths), _ptr(state), 0,
                              *_rows4(dout), *_rows4(dq), *_rows4(dk), *_rows4(dv), _ptr(dfinal), _ptr(dstate),
                              _ptr(ws), n), q.device)
        return dq, dk, dv, None, dstate, None, None


def linear_attention(q, k, v, log_decay, initial_state=None, episode_starts=None, lengths=None):
    """Linear attention with a decay per head over the columns of a rollout; returns (out, final_state).

    With ``g = exp(log_decay[h])``, per column n and head h::

        S_t = (0 if episode_starts[t, n] else g S_{t-1}) + k_t v_t^T,   S_{-1} = initial_state (None: zeros)
        out_t = S_t^T q_t,                                              final_state = S_{len-1}

    q, k [T, N, H, Dk] and v [T, N, H, Dv] (head sizes 1..128) share a dtype; any strides, broadcast views too
    (a q and k shared by the heads: ``expand`` them, and their gradient is summed).  Batch-major data is passed as
    ``x.transpose(0, 1)``.  log_decay: float32 [H], <= 0, without a gradient.  initial_state, final_state: float32
    [N, H, Dk, Dv].  episode_starts: uint8 or bool [T, N].  lengths: int [N]; rows behind a column's length are not
    read, come out as zeros and get zero gradients (values are clamped to 0..T).  out has v's shape and dtype.

    Differentiable in q, k, v and initial_state (in reverse, once); nothing but the inputs is kept for the backward
    pass, which is deterministic.  A non-finite input reaches the outputs that the recurrence lets it reach, and no
    others."""
    _heads("linear_attention", q, k, v, 4)
    T, N, H, Dk = q.shape
    dev = q.device
    log_decay = _decay("linear_attention", log_decay, H, dev)
    starts = _starts("linear_attention", episode_starts, (T, N), dev)
    state = None
    if initial_state is not None:
        state = _state("linear_attention", initial_state, (N, H, Dk, v.shape[3]), dev, "initial_state").contiguous()
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.shape != (N,) or lengths.device != dev or \
                lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError("linear_attention: lengths must be an int32 or int64 [N] tensor on the operands' device")
        lengths = lengths.clamp(0, T).to(torch.int32).contiguous() if lengths.dtype == torch.int64 \
            else lengths.contiguous()
    if forward_ad._current_level >= 0:
        _no_tangents("linear_attention", q, k, v, log_decay, state)
    q, k, v = _dense(q), _dense(k), _dense(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (state is not None and state.requires_grad)):
        return _LinearAttention.apply(q, k, v, log_decay, state, starts, lengths)
    return _linattn_forward(q, k, v, log_decay, state, starts, lengths)


def linear_attention_step(q, k, v, log_decay, state, episode_starts=None, state_out=None):
    """One token per environment of ``linear_attention``: q, k [N, H, Dk], v [N, H, Dv] -> out [N, H, Dv].

    ``state`` (float32 [N, H, Dk, Dv], contiguous) is read once and the new state written once, in place or into
    ``state_out``, which must not overlap it otherwise; autograd sees it as written in place.  A row with
    episode_starts [N] set begins from zeros.  Has no gradient (the training form is ``linear_attention``): tensors that
    require one are refused outside ``torch.no_grad()``."""
    who = "linear_attention_step"
    _heads(who, q, k, v, 3)
    N, H, Dk = q.shape
    dev = q.device
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    getattr(state, "requires_grad", False) or
                                    getattr(state_out, "requires_grad", False)):
        raise ValueError("%s has no gradient: use linear_attention, or torch.no_grad()" % who)
    log_decay = _decay(who, log_decay, H, dev)
    starts = _starts(who, episode_starts, (N,), dev)
    shape = (N, H, Dk, v.shape[2])
    new = state if state_out is None else state_out
    at = _step_state(who, state, shape, dev, "state")
    to = at
    if new is not state:
        to = _step_state(who, new, shape, dev, "state_out")
        if to != at and abs(to - at) < new.numel() * 4:
            raise ValueError("%s: state_out overlaps state" % who)
    if forward_ad._current_level >= 0:
        _no_tangents(who, q, k, v, log_decay, state, new)
    q, k, v = _dense(q), _dense(k), _dense(v)
    out = v.new_empty((N, H, shape[3]))
    _launch("fw_linattn_step",
            _pack_token(N, H, Dk, shape[3], _DT[q.dtype], *_rows3(q), *_rows3(k), *_rows3(v), *_rows3(out),
                        log_decay.data_ptr(), _ptr(starts), starts.stride(0) if starts is not None else 0,
                        at, to), dev)
    written(new)
    return out


def written(t):
    """Tells autograd that a kernel has written into ``t``, so that a backward pass that saved it refuses to run."""
    if not t.is_inference():  # (those have no version, and nothing saves them)
        torch.autograd.graph.increment_version(t)


# ------------------------------------------------------------------ group norm
_ACT = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "tanh": 4}  # include/fwrollout.h FW_ACT_*


@functools.lru_cache(maxsize=256)
def _norm_stats(N, L, C, groups):  # of the sizes alone
    return _native.load().fw_group_norm_stats(_pack_norm(N, L, C, groups, 0, 0, 0, 0, 0.0, *(0,) * 19))


def _rows(t):
    st = t.stride()
    return t.data_ptr(), st[0], st[1]


def _norm_forward(x, groups, weight, bias, eps, act, keep):
    N, L, C = x.shape
    y = x.new_empty((N, L, C))
    stats = ws = None
    n = 0
    p = weight if weight is not None else bias
    head = (N, L, C, groups, _DT[x.dtype], _DT[p.dtype] if p is not None else 0, act, 0, eps, *_rows(x), *_rows(y),
            0, 0, 0, 0, 0, 0, _ptr(weight), _ptr(bias), 0, 0)
    if _norm_stats(N, L, C, groups):  # (units that need neither fit a block)
        n = _native.load().fw_group_norm_workspace_bytes(_pack_norm(*head, 0, 0, 0), 0)
        ws = _workspace(n, x.device)
        stats = torch.empty((N, groups, 2), dtype=torch.float32, device=x.device) if keep else None
    _launch("fw_group_norm_forward", _pack_norm(*head, _ptr(stats), _ptr(ws), n), x.device)
    return y, stats


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        y, stats = _norm_forward(x, groups, weight, bias, eps, act, True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.conf = (groups, eps, act)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        groups, eps, act = ctx.conf
        dy = _dense(dy)
        N, L, C = x.shape
        dx = x.new_empty((N, L, C))
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        if x.numel() == 0:
            return (dx,) + tuple(t.zero_() if t is not None else None for t in (dw, db)) + (None, None, None)
        p = weight if weight is not None else bias
        head = (N, L, C, groups, _DT[x.dtype], _DT[p.dtype] if p is not None else 0, act, 0, eps, *_rows(x), 0, 0, 0,
                *_rows(dy), *_rows(dx), _ptr(weight), _ptr(bias), _ptr(dw), _ptr(db), _ptr(stats))
        n = _native.load().fw_group_norm_workspace_bytes(_pack_norm(*head, 0, 0), 1)
        ws = _workspace(n, x.device)
        _launch("fw_group_norm_backward", _pack_norm(*head, _ptr(ws), n), x.device)
        return dx, dw, db, None, None, None


def _channels(name, p, x, C):
    if p is None:
        return None
    if not isinstance(p, torch.Tensor) or p.shape != (C,) or p.get_device() != x.get_device() or \
            (p.dtype is not torch.float32 and p.dtype is not x.dtype):
        raise ValueError("group_norm_act: %s must be a [C] tensor of x's dtype or float32 on its device" % name)
    return p if p.is_contiguous() else p.contiguous()


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, activation="silu"):
    """``activation(group_norm(x))``, channels last: x [N, ..., C] of float32, bfloat16 or float16.

    The C channels form ``num_groups`` groups of neighbours; the statistics of a sample's group run over its channels
    and over every dimension between the first and the last (none of them: per row, as for a policy's features).
    weight, bias: [C] in x's dtype or float32 (both the same), or None.  activation: "none", "relu", "silu", "gelu" (by
    erf) or "tanh".  Returns a contiguous tensor of x's shape and dtype.  Any strides with unit channel stride are
    read in place.  Differentiable in x, weight and bias (in reverse, once); deterministic."""
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise ValueError("group_norm_act: x must be an [N, ..., C] tensor")
    if not x.is_cuda:
        raise ValueError("group_norm_act: x must be on the GPU (no CPU path exists)")
    if x.dtype not in _DT:
        raise ValueError("group_norm_act: x must be float32, bfloat16 or float16")
    C, groups = x.shape[-1], int(num_groups)
    if groups != num_groups:
        raise ValueError("group_norm_act: num_groups must be a whole number")
    if groups < 1 or C < 1 or C % groups:
        raise ValueError("group_norm_act: %d channels do not form %d groups" % (C, groups))
    if activation not in _ACT:
        raise ValueError("group_norm_act: activation must be one of %s" % ", ".join(_ACT))
    if not float(eps) >= 0.0:
        raise ValueError("group_norm_act: eps must be >= 0")
    weight, bias = _channels("weight", weight, x, C), _channels("bias", bias, x, C)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("group_norm_act: weight and bias must share a dtype")
    if forward_ad._current_level >= 0:
        _no_tangents("group_norm_act", x, weight, bias)
    shape = x.shape
    if len(shape) != 3:
        rows = 1
        for d in shape[1:-1]:
            rows *= d
        x = x.reshape(shape[0], rows, C)
    x = _dense(x)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        y = _GroupNormAct.apply(x, weight, bias, groups, float(eps), _ACT[activation])
    else:
        y = _norm_forward(x, groups, weight, bias, float(eps), _ACT[activation], False)[0]
    return y if len(shape) == 3 else y.view(shape)

"""float64 restatements of the sequence operators, token by token from their definitions (torch, CPU; test oracle)."""
import math

import torch


def _mask(T, N, starts, lengths):
    fresh = torch.zeros(T, N, dtype=torch.bool) if starts is None else starts.cpu() != 0
    n = torch.full((N,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    return fresh, torch.arange(T)[:, None] < n[None, :]


def linear_attention(q, k, v, log_decay, state=None, starts=None, lengths=None, dout=None, dfinal=None):
    """Returns (out, final) or, with dout, (out, final, dq, dk, dv, dstate).  Rows behind a length are zeros."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    T, N, H, Dk = q.shape
    Dv = v.shape[3]
    g = torch.exp(log_decay.detach().cpu().double())[None, :, None, None]
    fresh, live = _mask(T, N, starts, lengths)
    S = torch.zeros(N, H, Dk, Dv, dtype=torch.double) if state is None else state.detach().cpu().double().clone()
    out = torch.zeros(T, N, H, Dv, dtype=torch.double)
    states = []
    sel = lambda m, a, b: torch.where(m[:, None, None, None], a, b)
    for t in range(T):
        new = sel(fresh[t], torch.zeros_like(S), g * S) + k[t][..., None] * v[t][..., None, :]
        S = sel(live[t], new, S)
        o = (q[t][..., None] * S).sum(-2)
        out[t] = torch.where(live[t][:, None, None], o, torch.zeros_like(o))
        states.append(S)
    if dout is None:
        return out, S
    dout = dout.detach().cpu().double()
    R = torch.zeros_like(S) if dfinal is None else dfinal.detach().cpu().double().clone()
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    row = lambda m, a: torch.where(m[:, None, None], a, torch.zeros_like(a))
    for t in reversed(range(T)):
        dq[t] = row(live[t], (states[t] * dout[t][..., None, :]).sum(-1))
        R1 = R + q[t][..., None] * dout[t][..., None, :]
        dk[t] = row(live[t], (R1 * v[t][..., None, :]).sum(-1))
        dv[t] = row(live[t], (R1 * k[t][..., None]).sum(-2))
        R = sel(live[t], sel(fresh[t], torch.zeros_like(R), g * R1), R)
    return out, S, dq, dk, dv, R


def activation(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        c = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    y = torch.tanh(z)
    return y, 1 - y * y


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="silu", dy=None):
    """x [N][L][C]; returns y or, with dy, (y, dx, dweight, dbias)."""
    x = x.detach().cpu().double()
    N, L, C = x.shape
    per = C // groups
    w = torch.ones(C, dtype=torch.double) if weight is None else weight.detach().cpu().double()
    b = torch.zeros(C, dtype=torch.double) if bias is None else bias.detach().cpu().double()
    xg = x.reshape(N, L, groups, per)
    mean = xg.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(((xg - mean) ** 2).mean((1, 3), keepdim=True) + eps)
    xh = ((xg - mean) * r).reshape(N, L, C)
    y, slope = activation(xh * w + b, act)
    if dy is None:
        return y
    dz = dy.detach().cpu().double() * slope
    dxh = (dz * w).reshape(N, L, groups, per)
    xhg = xh.reshape(N, L, groups, per)
    dx = r * (dxh - dxh.mean((1, 3), keepdim=True) - xhg * (dxh * xhg).mean((1, 3), keepdim=True))
    return y, dx.reshape(N, L, C), (dz * xh).sum((0, 1)), dz.sum((0, 1))

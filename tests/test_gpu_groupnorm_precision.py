"""GPU: group norm where few bits or small numbers decide: groups without spread, variances that float32
does not hold, the activations' far sides."""
import pytest
import torch

from oracle import sequence_oracle as R
from test_gpu_groupnorm import ACTS, DEV, DTYPES, _seq

pytestmark = pytest.mark.gpu
# lanes, a block, a bundle of groups, streams
SHAPES = [(40, 1, 64, 4), (30, 1, 60, 4), (2, 300, 64, 4), (3, 900, 40, 4), (1, 9000, 24, 1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [2.5, 300.0, 1000.0])
@pytest.mark.parametrize("shape", SHAPES)
def test_groups_without_spread(shape, value, dtype):
    """Equal numbers of few bits: their sums are exact (below 2^24 of the last bit), so the mean is their value, x - mean is
    0 whatever 1 / sqrt(eps) = 316 would make of it, y is the bias and the weight's gradient 0: all of it exactly."""
    N, L, C, G = shape
    x = torch.full((N, L, C), value, dtype=dtype, device=DEV)
    w, b = torch.linspace(0.5, 1.5, C, device=DEV).requires_grad_(), torch.linspace(-1, 1, C, device=DEV)
    y = _seq().group_norm_act(x, G, w, b, activation="none")
    assert torch.equal(y.detach(), b.to(dtype).expand(N, L, C))
    dw, = torch.autograd.grad(y, w, torch.randn_like(y))
    assert not bool(dw.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_variances_beyond_float32(shape, act, dtype):
    """Deviations of 1e20: their squares are infinite in float32, 1 / sqrt of that is 0, and what follows is finite."""
    N, L, C, G = shape
    x = (torch.arange(N * L * C, device=DEV).reshape(N, L, C) % 3 - 1.0).mul_(1e20).to(dtype).requires_grad_()
    w, b = torch.linspace(0.5, 1.5, C, device=DEV).requires_grad_(), torch.linspace(-1, 1, C, device=DEV).requires_grad_()
    y = _seq().group_norm_act(x, G, w, b, activation=act)
    want = R.activation(b.detach().cpu().double(), act)[0]
    # the activation's own roundings and half a step
    tol = 2.0 ** -20 + torch.finfo(dtype).eps / 2 * want.abs()
    assert bool(((y.detach().cpu().double() - want).abs() <= tol).all())
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
    assert not bool(dx.any()) and not bool(dw.any()) and bool(db.isfinite().all())


def _activated(z, act, dtype):
    """act(z) and its slope, through groups of two channels -1 and 1: no mean, a spread of 1 (eps = 0), z the weight."""
    w = torch.stack([z, z], 1).reshape(-1).to(DEV)
    x = torch.tensor([-1.0, 1.0], device=DEV).repeat(len(z))[None].to(dtype)
    b = torch.zeros_like(w).requires_grad_()
    y = _seq().group_norm_act(x, len(z), w, b, eps=0.0, activation=act)
    slope, = torch.autograd.grad(y, b, torch.ones_like(y))
    signed = (w * x[0].float()).cpu().double()
    return signed, y.detach()[0].cpu().double(), slope.cpu().double()


def _held(got, want, tol):
    err = (got - want).abs()
    worst = int((err / tol).argmax())
    assert bool((err <= tol).all()), "%g for %g, %.3g times the tolerance" % (got[worst], want[worst], err[worst] / tol[worst])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_far_from_zero_in_16_bits(dtype):
    """Half a step of the type, relative to the value itself also where it is small.  The tail's polynomial is off by
    2^-18, the exponential's argument z^2 / 2 by two roundings: 123 x 2^-23 where float32 ends; a few roundings more:
    2^-15 together."""
    z, y, slope = _activated(torch.linspace(0.01, 13.0, 1300), "gelu", dtype)
    want, dwant = R.activation(z, "gelu")
    half, least = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny
    # below the smallest normal number: half of float16's last step; bfloat16's numbers there may be 0
    least = least * torch.finfo(dtype).eps / 2 if dtype == torch.float16 else least
    _held(y, want, 2.0 ** -15 * want.abs() + half * want.abs() * (1 + 2.0 ** -15) + least)
    q, p = 0.5 * torch.erfc(z.abs() * 0.5 ** 0.5), torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5 * z.abs()
    # the slope in float32: its terms' errors, and a rounding of the sum
    _held(slope, dwant, 2.0 ** -15 * (q + p) + 2.0 ** -23 * dwant.abs() + 1e-37)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_slopes_near_zero_in_16_bits(dtype):
    """The slopes are summed in float32 over all rows: their own error adds up.  The tail's 9e-8 of at most 1/2, its
    exponential's argument (4.5 at most, 2^-22 of it, of values below 1/4), and a few roundings of numbers up to 1.2: 2^-20."""
    z, _, slope = _activated(torch.linspace(0.001, 3.0, 1500), "gelu", dtype)
    _held(slope, R.activation(z, "gelu")[1], torch.full_like(slope, 2.0 ** -20))


@pytest.mark.parametrize("act", ["silu", "gelu", "tanh"])
def test_activations_in_float32(act):
    """Relative to the value at every z.  A handful of roundings and units of the hardware's exponential and reciprocal, 2^-23
    each: 2^-20.  What is below float32's normal numbers may be 0."""
    z, y, slope = _activated(torch.cat([torch.linspace(0.003, 1.5, 1000), torch.linspace(1.5, 13, 1000)] +
                                       ([torch.linspace(13, 100, 500)] if act != "gelu" else [])), act, torch.float32)
    want, dwant = R.activation(z, act)
    _held(y, want, 2.0 ** -20 * want.abs() + 100 * 2.0 ** -126)
    if act == "silu":
        s = torch.sigmoid(z)
        size = s * (1 + z.abs())
    elif act == "gelu":
        size = 0.5 * torch.erfc(-z * 0.5 ** 0.5) + z.abs() * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
    else:
        size = torch.ones_like(z)
    _held(slope, dwant, 2.0 ** -20 * size + 100 * 2.0 ** -126)


@pytest.mark.parametrize("groups", [2.5, "2", float("nan")])
def test_groups_are_a_whole_number(groups):
    with pytest.raises(ValueError):
        _seq().group_norm_act(torch.zeros(4, 8, device=DEV), groups)

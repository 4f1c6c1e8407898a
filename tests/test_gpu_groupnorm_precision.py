"""GPU: group norm where few bits or small numbers decide: groups without spread, variances that float32
does not hold."""
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

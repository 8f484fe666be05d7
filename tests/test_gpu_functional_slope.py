"""The gradient of GELU where it is small: between the passes 16-bit types keep its slope in 16 bits, which may not cost
the gradient its digits."""
import math

import pytest
import torch

from oracle import float_oracle as O
from test_gpu_functional import IDS, TYPES, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def F(gpu):
    from qnn import functional
    return functional


def gradient(F, z, dy):
    """dy gelu'(z) as the residual's gradient, of exactly these z: the product is of zeros."""
    r = z.clone().requires_grad_(True)
    x, w = torch.zeros(z.shape[0], 8, dtype=z.dtype, device="cuda"), torch.zeros(z.shape[1], 8, dtype=z.dtype, device="cuda")
    return torch.autograd.grad(F.linear_act(x, w, None, r, "gelu"), r, dy)[0].cpu().double()


def definition(z):
    """gelu'(z) in float64 and what its computation in fp32 may be off by.  Of the two terms Phi(-a) and a phi(a), a = |z|,
    the exponential is off by (z^2 + 8) e, the fit of the tail by 1.2e-6 up to a = 6.5 and by 1 % past it (where the tail
    is under 1 / a^2 of the other term)."""
    z = z.cpu().double()
    a = z.abs()
    tail, second = 0.5 * torch.special.erfc(a / math.sqrt(2)), a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    below = tail - second
    err = (z * z + 8) * O.E * (tail + second) + torch.where(a <= 6.5, 1.2e-6, 1e-2) * tail
    return torch.where(z < 0, below, 1 - below), err + torch.where(z < 0, 0.0, 2 * O.E)


@pytest.mark.parametrize("scale", [1.0, 300.0, 1e-3])
@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_gelu_gradient_keeps_its_digits(F, dt, scale):
    """Every z of the type in [-14, 7] (fp32: a million), within what the oracle's `slope_code` allows beside the rounding."""
    if dt == torch.float32:
        z = torch.linspace(-12, 7, 1 << 20, device="cuda")
    else:
        z = torch.arange(-32768, 32768, device="cuda").to(torch.int16).view(dt)
        z = z[(z >= -14) & (z <= 7)]
    z = z[:z.numel() // 8 * 8].view(-1, 8)
    dy = torch.full_like(z, scale)
    d, err = definition(z)
    want, err = d * dy.cpu().double(), (err + O.slope_code(d, err, dt)) * dy.cpu().double()
    near(gradient(F, z, dy), O._out(want, err, dt), "dz")


@pytest.mark.parametrize("dt", TYPES[:2], ids=IDS[:2])
def test_gelu_gradient_far_below(F, dt):
    """Where fixed point of d was off by 3 % and then 0.  In half steps of the type, one of them the rounding's: bf16 1 + 1/8 by the
    code; fp16 1 + 5e-5 |d|^(-1/4) 2^11, which is 1.14 at -0.25, 1.19, 1.31, 1.69, 3.0 and 8.5 at -6; and 0.01 for fp32."""
    z = torch.tensor([[-0.25, -2.0, -3.0, -4.0, -5.0, -6.0]], device="cuda", dtype=dt)
    d, _ = definition(z)
    scale = 2.0 ** 14  # as a loss's scale keeps such gradients among fp16's normal numbers
    got = gradient(F, z, torch.full_like(z, scale)) / scale
    steps = torch.tensor([1.14] * 6 if dt == torch.bfloat16 else [1.16, 1.22, 1.34, 1.72, 3.1, 8.7], dtype=torch.float64)
    assert ((got - d).abs() <= steps * torch.finfo(dt).eps / 2 * d.abs()).all(), (got, d)


@pytest.mark.parametrize("dt", TYPES, ids=IDS)
def test_gelu_gradient_at_the_ends(F, dt):
    inf = math.inf
    z = torch.tensor([[-inf, inf, math.nan, -0.0, 0.0, torch.finfo(dt).min, torch.finfo(dt).max, -20.0]], device="cuda").to(dt)
    got = gradient(F, z, torch.ones_like(z))[0]
    assert got[2].isnan() and got[[0, 1, 3, 4, 5, 6]].tolist() == [0.0, 1.0, 0.5, 0.5, 0.0, 1.0] and abs(got[7]) < 1e-30

"""SiLU and its slope at given z, over the whole range where they are not zero in FP32.

With weight 0 the value before the activation is the bias itself, so z is exact. u = 2^-24.

Value. The logistic function is r = 1 / (1 + t) for z >= 0 and t r below, with t = exp(-|z|).
32-bit tensors: t is off by 1 ulp (2 u) and, where it is below FP32's normal numbers, by half
their step 2^-150; the sum, the reciprocal and two products round once each: 6 u, 8 u allowed,
and |z| 2^-150 twice. 16-bit tensors: exp(-z) is a power of two with relative error 2^-22, whose
exponent is rounded (|z| u); a sum, a reciprocal's 2 u and a product: |z| u + 2^-22 + 4 u, below
|z| u + 2^-20. Then half a step of the type. Where exp(-z) is beyond FP32, from z = -88.72 down,
they may have 0 for s, as 1 / (1 + exp(-z)) in FP32 has.

Slope s (1 + z (1 - s)): the same for s and for 1 - s, the sum by the larger of its terms, and
dy s is formed first (a subnormal's rounding, 2^-150, times 1 + |z|).
"""

import math

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t, ref):
    f = torch.finfo(t)
    return (ref.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)


def relative(dtype, z):
    return 8 * U if dtype == F32 else z.abs() * U + 2.0 ** -20


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("pixels", [1, 3])
def test_every_z(dtype, pixels):
    z = torch.cat([torch.linspace(-95, -80, 4096), torch.linspace(-80, 30, 4000),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 88.0, 100.0, 1e4, 1e30, -1e4, -1e30] * 8 + [-104.0] * 16)])
    c = z.numel()
    assert c % 8 == 0
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 1, pixels, c, generator=g).to(dtype).cuda().permute(0, 3, 1, 2)
    bias = z.cuda().requires_grad_(True)
    y = fb.group_norm_act(x, 1, torch.zeros(c, device="cuda"), bias)
    zd = z.double().cuda()
    s, rest = torch.sigmoid(zd), torch.sigmoid(-zd)
    want = (zd * s).view(1, c, 1, 1).expand_as(y)
    zz = zd.view(1, c, 1, 1)
    gone = (dtype != F32) & (zd < -math.log(torch.finfo(F32).max))
    tol = (relative(dtype, zz) + gone.view(1, c, 1, 1)) * want.abs() + zz.abs() * 2.0 ** -149 + half_step(dtype, want)
    beyond = want.abs() > torch.finfo(dtype).max  # rounds to an infinity in x's type
    assert y[beyond].isinf().all() and (y[beyond] > 0).all()
    off = (y.double() - want).abs().masked_fill(beyond, 0.0)
    assert (off <= tol).all(), (zz.expand_as(y)[off > tol][:5], y[off > tol][:5], want[off > tol][:5])
    # dbias: the slope times the sum of dy
    dy = torch.ones_like(y)
    db, = torch.autograd.grad(y, bias, dy)
    ref = pixels * s * (1 + zd * rest)
    size = pixels * s * (1 + zd.abs() * rest)
    tol = (2 * relative(dtype, zd) + 8 * U + gone) * size + pixels * (1 + zd.abs()) * 2.0 ** -148
    off = (db.double() - ref).abs()
    assert (off <= tol).all(), (z[(off > tol).cpu()][:5], db[off > tol][:5], ref[off > tol][:5])

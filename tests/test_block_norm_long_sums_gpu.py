"""The vectors' gradients over many rows of terms of one sign, in which a long chain of FP32 sums drifts.

u = 2^-24. A thread adds the terms of at most 256 rows, and five steps of a warp, eight warps and three steps
between CTAs follow in FP32, all else in FP64: the sum of n equal terms t is off by at most (256 + 16) u n t,
and the term's own roundings. One running sum of FP32 loses the part of t below half a step of the sum
each time: with t = 1 + 3 * 2^-14 from 2^10 on, where a step is 2^-13, 2^-14 of each or more."""

import numpy as np
import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
T = 1.0 + 3 * 2.0 ** -14


def bound(rows):
    return (256 + 16 + 6) * U * rows * T


@pytest.mark.parametrize("rows,c", [(400_000, 8), (80_000, 24), (120_000, 96), (60_000, 264), (30_000, 1001)])
def test_sums_of_one_sign(rows, c):
    # rows of +-1 in turn, which are their own norm but for a rounding of rstd
    x = torch.ones(1, rows, c, device="cuda")
    x[..., 1::2] = -1.0
    y = torch.ones_like(x, requires_grad=True)
    gate, weight, bias = (torch.ones(c, device="cuda", requires_grad=True) for _ in range(3))
    scale, shift = (torch.zeros(1, c, device="cuda", requires_grad=True) for _ in range(2))
    r, z = fb.gated_residual_norm(x - 1.0, y, gate, weight, bias, scale=scale, shift=shift, kind="rms", eps=0.0)
    assert torch.equal(r, x)
    dr, dz = torch.zeros_like(r), torch.full_like(z, T)
    dz[..., 1::2] = -T  # dz rhat is T everywhere, and dR = dz - rhat <dz rhat> nothing
    dweight, dbias, dscale, dshift = torch.autograd.grad((r, z), (weight, bias, scale, shift), (dr, dz), retain_graph=True)
    sign = x[0, 0].double()
    for got, want in ((dweight, torch.ones_like(sign)), (dbias, sign), (dscale[0], 1.0 + sign), (dshift[0], sign)):
        assert (got.double() - rows * T * want).abs().max() <= 2 * bound(rows)
    (dgate,) = torch.autograd.grad((r, z), (gate,), (torch.full_like(r, T), torch.zeros_like(z)))
    assert (dgate.double() - rows * T).abs().max() <= bound(rows)


def test_a_running_sum_would_not_do():
    total, t, rows = np.float32(0.0), np.float32(T), 30_000
    for _ in range(rows):
        total = np.float32(total + t)
    assert abs(float(total) - rows * T) > 2 * bound(rows)

"""Gradient sums and statistics of tensors so large that each thread adds up over a thousand terms.

u = 2^-24. A thread adds at most 64 terms in FP32 before they go into an FP64 sum: 64 u of the sum
of magnitudes. The CTA's rows are added in FP32 (here at most 16 of them, one rounding each), the
part's sum is rounded to FP32 once and the result once: 64 + 16 + 4 = 84 u.
"""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SUM = 84 * U
F32 = torch.float32

# (N, C, H, W), groups; a CTA of 296 has one row of threads and some 1,000 or 3,400 spans for each
LONG = [
    ((1, 255, 547, 549), 5),    # one number a vector
    ((1, 255, 997, 1001), 5),
    ((1, 1024, 547, 549), 32),  # four numbers a vector
]


@pytest.mark.parametrize("case", range(len(LONG)))
def test_equal_gradients(case):
    """A constant dy without an activation: dbias = count * dy, and with weights of one dx = 0,
    both in closed form. The terms are equal, so that roundings do not average out."""
    shape, groups = LONG[case]
    n, c, h, w = shape
    g = torch.Generator(device="cuda").manual_seed(case)
    x = torch.randn(n, h, w, c, generator=g, device="cuda").permute(0, 3, 1, 2).requires_grad_(True)
    weight = torch.ones(c, device="cuda", requires_grad=True)
    bias = torch.zeros(c, device="cuda", requires_grad=True)
    for value in (0.1, 0.3, 0.7):
        y = fb.group_norm_act(x, groups, weight, bias, activation=None)
        dy = torch.full((), value, device="cuda").expand_as(y)
        dx, db = torch.autograd.grad(y, (x, bias), dy)
        v = dy.double()[0, 0, 0, 0].item()
        off = (db.double() - n * h * w * v).abs().max().item() / (n * h * w * v)
        assert off <= SUM, f"dbias is off by {off / U:.0f} u"
        # dx = rstd (dy - <dy> - xhat <dy xhat>); rstd is 1 to 1 %, |xhat| below 7, <dy xhat> is off
        # by the sum's error and the mean's (32 u), <|xhat|> below 1
        off = dx.abs().max().item() / (1.01 * v)
        assert off <= SUM + 4 * U + 7 * (SUM + 32 * U), f"dx is {off / U:.0f} u"


def test_equal_distances():
    """x = +-v in turn along each channel: mean 0 and variance v^2 exactly, so |y| = v / sqrt(v^2 + eps).
    A batch's 8 squares are added in FP32 (8 u), as are at most 16 batches and 16 rows (32 u): 40 u of
    the variance, 20 u of y, and 12 u for the mean and a few roundings."""
    for (n, c, h, w), _ in LONG:
        h += 1  # an even number of pixels
        for v in (0.37, 0.63, 0.74):
            sign = torch.ones(h * w, device="cuda")
            sign[1::2] = -1
            x = (v * sign).view(1, h, w, 1).expand(n, h, w, c).contiguous().permute(0, 3, 1, 2)
            y = fb.group_norm_act(x, 1, eps=1e-5, activation=None).double()
            vd = x.double().abs().max().item()
            want = vd / (vd * vd + 1e-5) ** 0.5
            off = (y.abs() - want).abs().max().item() / want
            assert off <= 32 * U, f"y is off by {off / U:.0f} u"

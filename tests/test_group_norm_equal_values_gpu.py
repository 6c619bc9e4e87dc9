"""group_norm_act of groups whose numbers are all equal: their mean is that number and their
variance zero, exactly, so z = (x - mean) rstd w + b is b itself, whatever the number, and every
term of dweight is zero. No tolerance: y is b rounded to x's type.
"""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# numbers of few and of many digits; near the ends of the type's range too
VALUES = {F32: [1000.25, 1000.1, 0.1, 1 / 3, -7e-3, 3e19, -1e30, 3e38, 1e-30],
          F16: [1000.25, 1000.1, 0.1, 1 / 3, -7e-3, 65504.0],
          BF16: [1000.25, 1000.1, 0.1, 1 / 3, -7e-3, 3e19, -1e30, 3e38, 1e-30]}


def check(shape, groups, dtype, values):
    """values: one for each channel, the same within a group."""
    n, c, h, w = shape
    g = torch.Generator().manual_seed(c * 1000 + h * w)
    x = values.to(dtype).cuda().view(1, c, 1, 1).expand(shape).contiguous(
        memory_format=torch.channels_last).requires_grad_(True)
    weight = (1 + 0.3 * torch.randn(c, generator=g)).cuda().requires_grad_(True)
    bias = torch.randn(c, generator=g).cuda().requires_grad_(True)
    y = fb.group_norm_act(x, groups, weight, bias, activation=None)
    want = bias.detach().to(dtype).view(1, c, 1, 1).expand_as(y)
    assert torch.equal(y, want), (shape, groups, (y != want).sum().item())
    dy = torch.randn(n, h, w, c, generator=g).to(dtype).cuda().permute(0, 3, 1, 2)
    dx, dw = torch.autograd.grad(y, (x, weight), dy)
    assert torch.equal(dw, torch.zeros_like(dw)) and dx.isfinite().all()


SHAPES = (
    # one launch, a thread's vectors from one to eight and more, the last batch of each length
    [(200, 16, 1, 64 * k) for k in range(1, 17)] + [(3, 16, 1, 200 * k + 7) for k in range(1, 9)] +
    # the passes: spans of one to several pixels, a thread's from one to a batch and more
    [(1, 5, 1, 51 * k) for k in range(1, 18)] + [(2, 6, 1, 85 * k + 1) for k in range(1, 9)] +
    [(1, 64, 300, 300 + k) for k in range(0, 8)] +
    # a group over several slices
    [(1, 1283, 40, 30), (3, 2056, 20, 21)])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_one_number_everywhere(dtype):
    for i, shape in enumerate(SHAPES):
        for value in VALUES[dtype][i % 3::3]:
            check(shape, 1, dtype, torch.full((shape[1],), value))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_a_number_for_each_channel(dtype):
    for shape in SHAPES:
        g = torch.Generator().manual_seed(shape[3])
        check(shape, shape[1], dtype, 100 * torch.randn(shape[1], generator=g))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_numbers_that_differ_little(dtype):
    # 3e19 squared is beyond FP32, the distances squared are not: y = (x - mean) / std
    step = torch.finfo(dtype).eps * 2 ** 65
    for shape in ((2, 16, 16, 16), (1, 16, 300, 301)):
        x = torch.full(shape, 2.0 ** 65)
        x[:, :, :, ::2] += step
        share = (shape[3] + 1) // 2 / shape[3]
        x = x.to(dtype).cuda().contiguous(memory_format=torch.channels_last)
        y = fb.group_norm_act(x, 1, activation=None).double()
        # two values of known shares: the statistics in closed form. The mean, an FP32 number near
        # 2^65, is off by a few of its steps (bf16 steps are 2^16 of those; FP32's are one, and the
        # two values lie one apart, so there y is only bounded).
        std = step * (share * (1 - share)) ** 0.5
        hi, lo = step * (1 - share) / std, -step * share / std
        assert y.isfinite().all()
        if dtype == BF16:
            assert ((y[:, :, :, ::2] - hi).abs() <= 2.0 ** -7 * abs(hi)).all()
            assert ((y[:, :, :, 1::2] - lo).abs() <= 2.0 ** -7 * abs(lo)).all()

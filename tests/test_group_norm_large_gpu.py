"""group_norm_act of tensors beyond L2: short applying parts and L2 priorities (from 80 MB and six
waves of parts up), a part's sums in FP64. Every output is compared, against the definition in 64
bits and with the tolerances of test_group_norm_gpu.py.
"""

import pytest
import torch

import fussim_b200 as fb

from .test_group_norm_gpu import BF16, F16, F32, check_backward, check_forward, grads

pytestmark = pytest.mark.gpu

LARGE = [
    ((2, 64, 993, 1001), 16, BF16, F32, "silu"),    # 254 MB, 8 channels a vector
    ((5, 64, 620, 647), 4, F16, F16, None),
    ((1, 48, 1303, 1001), 16, F32, F32, "silu"),    # 250 MB
    ((3, 6, 1999, 2000), 3, F32, F32, "relu"),      # two pixels a span
    ((1, 3, 5000, 4004), 1, BF16, BF16, "silu"),    # eight pixels a span
    ((1, 2064, 247, 251), 8, BF16, F32, "silu"),    # two slices
    ((1, 255, 701, 703), 5, F16, F32, "silu"),      # one number a vector
    ((500, 64, 61, 63), 8, BF16, F32, "silu"),      # more samples than a wave of CTAs
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_values_and_gradients(case):
    (n, c, h, w), groups, dtype, wdtype, act = LARGE[case]
    g = torch.Generator(device="cuda").manual_seed(case)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    x = (randn(n, h, w, c) * (0.5 + randn(c).abs()) + randn(c)).to(dtype).permute(0, 3, 1, 2)
    dy = randn(n, h, w, c).to(dtype).permute(0, 3, 1, 2)
    weight, bias = (1 + 0.3 * randn(c)).to(wdtype), (0.3 * randn(c)).to(wdtype)
    assert x.numel() * x.element_size() > 80 << 20
    y, dx, dw, db = grads(x, groups, weight, bias, 1e-5, act, dy)
    check_forward(y, x, groups, weight, bias, 1e-5, act)
    check_backward(dx, dw, db, x, groups, weight, bias, 1e-5, act, dy)
    again = grads(x, groups, weight, bias, 1e-5, act, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, (y, dx, dw, db)))
    with torch.no_grad():
        assert torch.equal(fb.group_norm_act(x, groups, weight, bias, 1e-5, act), y)

"""A 16-bit sum with a branch that has no norm is formed in the same steps of 32 bits wherever its rows
begin: the product of scale and gate, that with the branch, the sum, and the type's rounding."""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("c", [40, 1000, 4104, 5000, 9000, 16384, 4999, 9001])
def test_bits(c, dtype):
    rows = 2_000_000 // c
    g = torch.Generator().manual_seed(c)
    x, y = ((torch.randn(rows * c + 1, generator=g) + 0.1).to(dtype).cuda() for _ in range(2))
    gate = torch.randn(c, generator=g).cuda()
    want = (x[1:].view(rows, c).float() + (gate * 0.7) * y[1:].view(rows, c).float()).to(dtype)
    apart = fb.gated_residual(x[1:].view(rows, c), y[1:].view(rows, c), gate, residual_scale=0.7)
    whole = fb.gated_residual(x[1:].clone().view(rows, c), y[1:].clone().view(rows, c), gate, residual_scale=0.7)
    assert torch.equal(apart, want) and torch.equal(whole, want)

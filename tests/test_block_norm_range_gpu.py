"""Norms of finite rows whose numbers lie further apart than FP32 (and BF16) reaches, or whose squares add up
to more than it holds.

Tolerances as in test_block_norm_gpu. The reciprocal of a deviation of 2^127 is a multiple of 2^-149 and
so off by at most 2^-22 of itself, 4 u, besides; a thread's sums are of at most 32 numbers and a row's of
41 roundings in all, which leaves those 4 u inside D(v).
"""

import pytest
import torch

import fussim_b200 as fb
from tests.test_block_norm_gpu import BF16, F32, check, near, normed

pytestmark = pytest.mark.gpu

COLS = (2, 24, 96, 600, 1003, 1024, 3000, 5001, 8192, 16384)


def rows(c, dtype, seed=0):
    """Both signs, one number against all others, and rows of ordinary numbers beside them."""
    g = torch.Generator().manual_seed(seed + c)
    t = torch.randn(7, c, generator=g)
    t[0] = torch.where(torch.arange(c) % 2 == 0, 2.5e38, -2.5e38)
    t[2] = torch.where(t[2] > 0, 3e38, -3e38)
    t[2, 0], t[2, 1] = 3e38, -3e38
    t[4] = 3e38
    t[4, -1] = -3e38
    t[5] = (t[5].clamp(-3, 3) / 3) * 3.2e38
    t[5, 0], t[5, -1] = 3.2e38, -3.2e38
    return t.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("c", COLS)
def test_norm_before(c, dtype):
    x = rows(c, dtype).unsqueeze(0).requires_grad_(True)
    w, b = (torch.randn(c, device="cuda", requires_grad=True) for _ in range(2))
    z = fb.block_norm(x, w, b, kind="layer")
    assert z.isfinite().all()
    up = torch.randn(z.shape, device="cuda").to(dtype)
    grads = dict(zip(("x", "weight", "bias"), torch.autograd.grad(z, (x, w, b), up)))
    check({"x": x, "weight": w, "bias": b}, "before", None, z, kind="layer", ups=(None, up), grads=grads)
    with torch.no_grad():
        assert torch.equal(fb.block_norm(x, w, b, kind="layer"), z)
        # rows beside those keep their bits
        small = [1, 3, 6]
        alone = x.detach().clone()
        alone[:, [0, 2, 4, 5]] = 1.0
        assert torch.equal(fb.block_norm(alone, w, b, kind="layer")[:, small], z[:, small])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("c", COLS)
def test_norm_of_the_branch(c, dtype):
    x = torch.randn(1, 7, c, device="cuda").to(dtype).requires_grad_(True)
    y = rows(c, dtype, 1).unsqueeze(0).requires_grad_(True)
    w = torch.randn(c, device="cuda", requires_grad=True)
    r = fb.gated_residual(x, y, branch_kind="layer", branch_weight=w)
    up = torch.randn(r.shape, device="cuda").to(dtype)
    grads = dict(zip(("x", "branch", "branch_weight"), torch.autograd.grad(r, (x, y, w), up)))
    check({"x": x, "branch": y, "branch_weight": w}, "after", r, None, branch_kind="layer", ups=(up, None), grads=grads)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("c", COLS)
def test_rms(c, dtype):
    x = rows(c, dtype).unsqueeze(0).requires_grad_(True)
    x.data[:, 1] = 3.3e38
    z = fb.block_norm(x)
    up = torch.randn(z.shape, device="cuda").to(dtype)
    check({"x": x}, "before", None, z, ups=(None, up), grads={"x": torch.autograd.grad(z, x, up)[0]})
    r = fb.gated_residual(torch.zeros_like(x), x, branch_kind="rms")
    check({"x": torch.zeros_like(x), "branch": x}, "after", r, None, branch_kind="rms")


def test_residual_stream():
    """r itself lies that far apart."""
    for c in (48, 1000, 4104):
        x = rows(c, F32).unsqueeze(0)
        y = torch.randn(1, 7, c, device="cuda").to(BF16)
        r, z = fb.gated_residual_norm(x, y, kind="layer", branch_kind="rms")
        h, off, _ = normed(r.double(), "layer", 1e-6)
        near("z", z, h, off)

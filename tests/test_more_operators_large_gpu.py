"""Block norms and AdamW on tensors of more than 2^31 numbers: what lies behind that is compared."""

import pytest
import torch

import fussim_b200 as fb
from tests import adamw_oracle as O
from tests.test_adamw_gpu import unlike
from tests.test_block_norm_gpu import check

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [1024, 1001])
def test_rows_behind_2_31(cols):
    rows = (1 << 31) // cols + 300
    x = torch.zeros(1, rows, cols, device="cuda", dtype=BF16)
    y = torch.zeros_like(x)
    parts = [slice(0, 200), slice(rows - 250, rows)]
    for p in parts:
        x[:, p] = torch.randn(1, p.stop - p.start, cols, device="cuda").to(BF16)
        y[:, p] = torch.randn(1, p.stop - p.start, cols, device="cuda").to(BF16)
    gate, weight = (torch.randn(cols, device="cuda").to(BF16) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (x, y)]
    r, z = fb.gated_residual_norm(x, y, gate, weight, kind="layer", residual_scale=0.7)
    ups = torch.randn(2, 1, 250, cols, device="cuda").to(BF16)
    dr, dz = torch.zeros_like(r), torch.zeros_like(z)
    dr[:, parts[1]], dz[:, parts[1]] = ups[0], ups[1]
    dx, dy = torch.autograd.grad((r, z), leaves, (dr, dz))
    for p in parts:
        d = {"x": x[:, p].detach(), "branch": y[:, p].detach(), "gate": gate, "weight": weight}
        check(d, "both", r[:, p], z[:, p], kind="layer", s=0.7, ups=(dr[:, p], dz[:, p]),
              grads={"x": dx[:, p], "branch": dy[:, p]})


@pytest.mark.parametrize("bits", [32, 8])
def test_numbers_behind_2_31(bits):
    n, first = (1 << 31) + 777, (1 << 31) - 512
    p = torch.zeros(n, device="cuda", dtype=BF16)
    g = torch.zeros_like(p)
    m, v, scales = fb.adamw_moments(p, bits)
    tail = slice(first, n)
    p[tail] = (torch.randn(n - first, device="cuda") * 0.1).to(BF16)
    g[tail] = (torch.randn(n - first, device="cuda") * 0.01).to(BF16)
    before = [t[tail].cpu().clone() for t in (p, g, m, v)]
    old = None if scales is None else scales[first // 256:].cpu().clone()
    fb.adamw_step_([p], [g], [m], [v], None if scales is None else [scales], step=3, lr=1e-2, seed=5)
    want = O.step32(*before, old, step=3, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, wd=1e-2, seed=5, first_block=first // 256)
    for name, got, ref in zip(("param", "exp_avg", "exp_avg_sq"), (p, m, v), want):
        found = unlike(got[tail].cpu(), ref.to(got.dtype))
        assert not found, f"{name}: {found}"
    if scales is not None:
        assert not unlike(scales[first // 256:].cpu(), want[3])
    assert not p[:1000].any() and not m.view(torch.uint8)[:1000].any()

"""The sum that gated_residual returns may be written in place, as that of x + s * gate * y: its backward
pass has no use for it. gated_residual_norm's may not, since it is what the norm took."""

import pytest
import torch

import fussim_b200 as fb
from tests.test_block_norm_gpu import BF16, F16, F32, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("branch_kind", [None, "rms", "layer"])
@pytest.mark.parametrize("types", [(F32, F32), (F32, BF16), (F16, F16)], ids=str)
def test_in_place(types, branch_kind):
    for shape in ((2, 9, 40), (1, 33, 1001), (3, 0, 16)):
        d = make(*shape, *types, "sample", branch_kind, form="after")
        for t in d.values():
            t.requires_grad_(True)
        kw = dict(residual_scale=0.5, branch_kind=branch_kind, branch_weight=d.get("branch_weight"),
                  branch_bias=d.get("branch_bias"))
        r = fb.gated_residual(d["x"], d["branch"], d["gate"], **kw)
        kept = r.detach().clone()
        r += 1.0
        up = torch.randn(r.shape, device="cuda").to(r.dtype)
        grads = dict(zip(d, torch.autograd.grad(r, list(d.values()), up)))
        for k, t in d.items():
            assert grads[k].dtype == t.dtype and grads[k].shape == t.shape
        if r.numel():
            check(d, "after", kept, None, branch_kind=branch_kind, s=0.5, ups=(up, None), grads=grads)


def test_some_gradients():
    for names in (["x"], ["branch"], ["gate"]):
        d = make(2, 9, 40, F32, BF16, "channel", None, form="after")
        for k in names:
            d[k].requires_grad_(True)
        r = fb.gated_residual(d["x"], d["branch"], d["gate"])
        r.mul_(2.0)
        (got,) = torch.autograd.grad(r.sum(), [d[k] for k in names])
        assert got.dtype == d[names[0]].dtype and got.shape == d[names[0]].shape and got.any()


def test_the_norms_input_may_not():
    x = torch.randn(3, 16, device="cuda", requires_grad=True)
    r, z = fb.gated_residual_norm(x, torch.randn(3, 16, device="cuda"))
    r += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()

"""The vectors' gradients of rows within a warp, whose sums are laid where the ring of rows was: with
even and odd numbers of turns of a CTA they are those of the definition, and the same bits each time."""

import pytest
import torch

from tests.test_block_norm_gpu import BF16, F16, F32, call, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("types", [(F32, F32), (F16, F16), (F32, BF16)], ids=str)
@pytest.mark.parametrize("c", [8, 24, 96, 256, 512])
def test_repeats_after_even_and_odd_turns(c, types):
    kw = dict(kind="layer", branch_kind="layer", s=0.7)
    for rows in (1, 2, 33, 64, 129, 256, 511, 768, 1024, 1281, 5000, 20_001):
        d = make(2, rows, c, *types, "sample", "layer", "layer", True, seed=rows)
        for t in d.values():
            t.requires_grad_(True)
        r, z = call(d, "both", **kw)
        g = torch.Generator(device="cuda").manual_seed(rows)
        ups = [torch.randn(o.shape, generator=g, device="cuda").to(o.dtype) for o in (r, z)]
        first = torch.autograd.grad((r, z), list(d.values()), ups, retain_graph=True)
        check(d, "both", r, z, ups=ups, grads=dict(zip(d, first)), **kw)
        for _ in range(5):
            again = torch.autograd.grad((r, z), list(d.values()), ups, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(first, again)), rows


@pytest.mark.parametrize("c", [8, 96, 512])
def test_before_and_plain(c):
    """The kernels of fewer sums."""
    for form, kw in (("before", dict(kind="layer")), ("both", dict(kind="rms")), ("after", dict(branch_kind=None))):
        for rows in (64, 700, 1536):
            d = make(1, rows, c, F32, F32, "channel" if form != "before" else "none", None, kw.get("kind", "rms"), True,
                     form, seed=rows)
            for t in d.values():
                t.requires_grad_(True)
            outs = [o for o in call(d, form, **kw) if o is not None]
            ups = [torch.randn_like(o) for o in outs]
            first = torch.autograd.grad(outs, list(d.values()), ups, retain_graph=True)
            r, z = (None, outs[0]) if form == "before" else (outs[0], outs[1] if form == "both" else None)
            check(d, form, r, z, ups=(ups[0] if r is not None else None, ups[-1] if z is not None else None),
                  grads=dict(zip(d, first)), **kw)
            for _ in range(5):
                again = torch.autograd.grad(outs, list(d.values()), ups, retain_graph=True)
                assert all(torch.equal(a, b) for a, b in zip(first, again)), (form, rows)

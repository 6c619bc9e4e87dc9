"""Steps of AdamW that are refused leave parameters, moments and counts as they were, in every group; the
next one goes as if they had not been tried."""

import pytest
import torch

import fussim_b200 as fb
from tests.test_adamw_optimizer_gpu import equal

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def pair(dtype, **kw):
    """(parameters, optimiser) of two groups, twice."""
    out = []
    for _ in range(2):
        g = torch.Generator().manual_seed(3)
        p = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in ((5, 7), (300,), (4, 6))]
        out.append((p, fb.AdamW([dict(params=p[:1]), dict(params=p[1:], lr=1e-2)], **kw)))
    return out


def give(p, step):
    g = torch.Generator().manual_seed(step)
    for t in p:
        t.grad = (0.01 * torch.randn(t.shape, generator=g)).to(t.dtype).cuda()


def sparse(p, opt):
    p[2].grad = p[2].grad.to_sparse()


def gaps(p, opt):
    p[2].data = torch.zeros(4, 12, device="cuda", dtype=p[2].dtype)[:, ::2]


def rate(p, opt):
    opt.param_groups[1]["lr"] = -1.0


def moments(p, opt):
    if opt.state.get(p[2]):
        opt.state[p[2]]["exp_avg"] = opt.state[p[2]]["exp_avg"].t()
    else:
        sparse(p, opt)


@pytest.mark.parametrize("kw", [dict(), dict(state_bits=8, max_norm=0.05), dict(capturable=True),
                                dict(master_weights=True), dict(capturable=True, state_bits=8)], ids=str)
@pytest.mark.parametrize("spoil", [sparse, gaps, rate, moments], ids=lambda f: f.__name__)
@pytest.mark.parametrize("after", [0, 2])
def test_refused(after, spoil, kw):
    dtype = BF16 if "master_weights" in kw else F32
    (a, opt), (b, ref) = pair(dtype, **kw)
    for step in range(after):
        for p, o in ((a, opt), (b, ref)):
            give(p, step)
            o.step()
    give(a, after)
    kept = a[2].data, opt.param_groups[1]["lr"], dict(opt.state.get(a[2], {})), opt.grad_norm
    spoil(a, opt)
    for _ in range(2):
        with pytest.raises((ValueError, RuntimeError)):
            opt.step()
    a[2].data, opt.param_groups[1]["lr"] = kept[:2]
    assert opt.grad_norm is kept[3]
    assert bool(opt.state.get(a[2])) == bool(after)
    if after:
        opt.state[a[2]].update(kept[2])
    assert equal(a, b)
    for step in range(after, after + 3):
        for p, o in ((a, opt), (b, ref)):
            give(p, step)
            o.step()
        assert equal(a, b)
    for p, q in zip(a, b):
        assert int(opt.state[p]["step"]) == int(ref.state[q]["step"]) == after + 3
        assert equal([opt.state[p]["exp_avg"]], [ref.state[q]["exp_avg"]])

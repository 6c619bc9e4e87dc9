"""A refused step leaves counts and states as they were (here the GPU is what is missing)."""

import pytest
import torch

import fussim_b200 as fb


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
@pytest.mark.parametrize("kw", [dict(), dict(state_bits=8), dict(capturable=True), dict(max_norm=1.0)], ids=str)
def test_no_gpu(kw):
    p = torch.nn.Parameter(torch.ones(3, 5))
    p.grad = torch.ones(3, 5)
    opt = fb.AdamW([p], **kw)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="CUDA is not available"):
            opt.step()
    assert not opt.state.get(p) and opt.grad_norm is None
    opt.state[p] = dict(step=7, exp_avg=torch.zeros(3, 5), exp_avg_sq=torch.zeros(3, 5))
    if not kw:
        with pytest.raises(RuntimeError, match="CUDA is not available"):
            opt.step()
        assert opt.state[p]["step"] == 7 and torch.equal(p, torch.ones(3, 5))


def test_a_later_group():
    """A group that cannot be served is found before the first one's parameters count."""
    p, q = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    opt = fb.AdamW([dict(params=[p]), dict(params=[q])])
    opt.param_groups[1]["amsgrad"] = True
    p.grad = q.grad = torch.ones(4)
    with pytest.raises(ValueError, match="amsgrad"):
        opt.step()
    assert not opt.state.get(p) and not opt.state.get(q)

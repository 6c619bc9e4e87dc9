"""States of AdamW are float32 whatever torch's default type is."""

import pytest
import torch

import fussim_b200 as fb


@pytest.fixture(params=[torch.float64, torch.bfloat16], ids=str)
def default(request):
    kept = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(kept)


def test_moments(default):
    p = torch.zeros(300, dtype=torch.float32)
    for bits in (32, 8):
        first, second, scales = fb.adamw_moments(p, bits)
        assert first.dtype == second.dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)
    assert scales.dtype == torch.float32


def test_counts(default):
    p = torch.nn.Parameter(torch.zeros(3, dtype=torch.float32))
    opt = fb.AdamW([p], capturable=True)
    assert opt._count(opt.param_groups[0], p.device).dtype == torch.float32
    state = dict(step=torch.tensor(4.0), exp_avg=torch.ones(3), exp_avg_sq=torch.ones(3))
    opt.load_state_dict(dict(state={0: state}, param_groups=[dict(opt.param_groups[0], params=[0])]))
    assert opt.state[p]["step"].dtype == torch.float32 and int(opt.state[p]["step"]) == 4
    assert opt.state[p]["exp_avg"].dtype == torch.float32

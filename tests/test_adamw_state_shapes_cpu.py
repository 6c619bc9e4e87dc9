"""State dicts whose states do not fit the parameters are refused before anything is loaded."""

import copy

import pytest
import torch

import fussim_b200 as fb

F8 = torch.float8_e4m3fn


def optimiser(bits=32):
    p = [torch.nn.Parameter(torch.randn(4, 6)), torch.nn.Parameter(torch.randn(300))]
    opt = fb.AdamW(p, state_bits=bits)
    for t in p:
        first, second, scales = fb.adamw_moments(t, bits)
        opt.state[t] = dict(step=3, exp_avg=first, exp_avg_sq=second)
        if scales is not None:
            opt.state[t]["scales"] = scales
    return p, opt


@pytest.mark.parametrize("name,shape", [("exp_avg", (1, 6)), ("exp_avg_sq", (6,)), ("exp_avg", ()), ("exp_avg", (6, 4))])
def test_shapes(name, shape):
    p, opt = optimiser()
    saved = copy.deepcopy(opt.state_dict())
    saved["state"][0][name] = torch.ones(shape)
    saved["param_groups"][0]["lr"] = 5.0
    kept = {k: dict(v) for k, v in opt.state.items()}
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 1e-3
    for k, v in opt.state.items():
        assert all(v[n] is t for n, t in kept[k].items())


def test_master():
    p = torch.nn.Parameter(torch.randn(4, 6).bfloat16())
    opt = fb.AdamW([p], master_weights=True)
    first, second, _ = fb.adamw_moments(p)
    opt.state[p] = dict(step=1, exp_avg=first, exp_avg_sq=second, master=p.detach().float())
    saved = copy.deepcopy(opt.state_dict())
    opt.load_state_dict(saved)
    saved["state"][0]["master"] = torch.ones(6)
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(saved)


def test_codes():
    p, opt = optimiser(8)
    saved = copy.deepcopy(opt.state_dict())
    opt.load_state_dict(saved)
    for change, match in ((dict(scales=torch.ones(1, 1)), "scales"), (dict(scales=torch.ones(2, 2).double()), None),
                          (dict(exp_avg=torch.zeros(30, 10).to(F8)), "shape")):
        other = copy.deepcopy(saved)
        other["state"][1].update(change)
        if match:
            with pytest.raises(ValueError, match=match):
                opt.load_state_dict(other)
        else:
            opt.load_state_dict(other)
            assert opt.state[p[1]]["scales"].dtype == torch.float32
    del saved["state"][1]["scales"]
    with pytest.raises(ValueError, match="scales"):
        opt.load_state_dict(saved)


def test_strides_are_checked_first():
    p = torch.nn.Parameter(torch.randn(2, 3, 4, 5).to(memory_format=torch.channels_last))
    q = torch.nn.Parameter(torch.randn(2, 3, 4, 5))
    opts = []
    for t in (p, q):
        opt = fb.AdamW([t], state_bits=8)
        first, second, scales = fb.adamw_moments(t, 8)
        opt.state[t] = dict(step=1, exp_avg=first, exp_avg_sq=second, scales=scales)
        opts.append(opt)
    kept = dict(opts[1].state[q])
    with pytest.raises(ValueError, match="strides"):
        opts[1].load_state_dict(opts[0].state_dict())
    assert all(opts[1].state[q][n] is t for n, t in kept.items())


def test_counts_of_a_group():
    """Unequal counts of a capturable group are found first, too."""
    p, opt = optimiser()
    saved = copy.deepcopy(opt.state_dict())
    saved["state"][0]["step"] = 9
    opt.load_state_dict(saved)
    assert [opt.state[t]["step"] for t in p] == [9, 3]
    saved["param_groups"][0]["capturable"] = True
    with pytest.raises(ValueError, match="same number of steps"):
        opt.load_state_dict(saved)
    assert [opt.state[t]["step"] for t in p] == [9, 3] and not opt.param_groups[0]["capturable"]

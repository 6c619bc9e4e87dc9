"""What records or differentiates a call in ways that the training operators do not support is
refused, before anything else looks at the tensors (runs without a GPU)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

import fussim_b200 as fb

X, W = torch.randn(2, 12, 4, 5), torch.ones(12)


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode(which, requires_grad):
    args = {"x": X, "weight": W, "bias": W}
    with fwAD.dual_level():
        t = args[which].clone().requires_grad_(requires_grad)
        args[which] = fwAD.make_dual(t, torch.ones_like(t))
        with pytest.raises(RuntimeError, match="forward-mode.*" + which):
            fb.group_norm_act(args["x"], 3, args["weight"], args["bias"])


CALLS = {
    "group_norm_act": lambda x: fb.group_norm_act(x, 3),
    "grad_norm": lambda x: fb.grad_norm([x]),
    "clip_grad_norm": lambda x: fb.clip_grad_norm([x], 1.0)[1],
}


@pytest.mark.parametrize("name", CALLS)
def test_tracing(name):
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        torch.jit.trace(CALLS[name], X)
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        make_fx(CALLS[name])(X)

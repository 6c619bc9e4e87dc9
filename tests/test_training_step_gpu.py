"""The operators together, as a training step uses them: a small image network of
convolutions and GroupNormAct layers, the fused loss, its backward pass, and clipping."""

import copy

import pytest
import torch

import fussim_b200 as fb
from fussim_b200 import synthetic

pytestmark = pytest.mark.gpu


class Plain(torch.nn.Module):
    """GroupNormAct in torch's own operators."""

    def __init__(self, layer):
        super().__init__()
        self.weight, self.bias, self.layer = layer.weight, layer.bias, layer

    def forward(self, x):
        y = torch.nn.functional.group_norm(x, self.layer.num_groups, self.weight, self.bias,
                                           self.layer.eps)
        return torch.nn.functional.silu(y)


def network(seed):
    torch.manual_seed(seed)
    layers = [torch.nn.Conv2d(3, 16, 3, padding=1), fb.GroupNormAct(4, 16),
              torch.nn.Conv2d(16, 24, 3, padding=1), fb.GroupNormAct(8, 24),
              torch.nn.Conv2d(24, 3, 3, padding=1), torch.nn.Sigmoid()]
    return torch.nn.Sequential(*layers).cuda().to(memory_format=torch.channels_last)


def step(net, a, b, limit, clip):
    net.zero_grad(set_to_none=True)
    loss = fb.l1_dssim_loss(net(a).contiguous(), b)
    loss.backward()
    norm = clip(net.parameters(), limit)
    return loss.item(), norm.item(), [p.grad for p in net.parameters()]


@pytest.fixture
def full_precision():
    kept = torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32
    torch.backends.cudnn.allow_tf32 = torch.backends.cuda.matmul.allow_tf32 = False
    yield
    torch.backends.cudnn.allow_tf32, torch.backends.cuda.matmul.allow_tf32 = kept


@pytest.mark.parametrize("limit", [0.01, 100.0])
def test_step_matches_torch(limit, full_precision):
    a, b = (t.cuda() for t in synthetic.pair_noise((2, 3, 61, 75), 0.1, seed=3))
    net = network(1)
    ref = copy.deepcopy(net)
    for i, layer in enumerate(ref):
        if isinstance(layer, fb.GroupNormAct):
            ref[i] = Plain(layer)
    got = step(net, a, b, limit, fb.clip_grad_norm_)
    want = step(ref, a, b, limit, torch.nn.utils.clip_grad_norm_)
    assert abs(got[0] - want[0]) <= 1e-5 and abs(got[1] - want[1]) <= 1e-4 * want[1]
    scale = max(w.abs().max().item() for w in want[2])
    for g, w in zip(got[2], want[2]):
        # convolutions and the loss round alike on both sides but for the layers' differences
        # of a few 2^-24, amplified by at most the layers' 1/std
        assert (g - w).abs().max().item() <= 1e-4 * scale


def test_step_in_a_graph():
    a, b = (t.cuda() for t in synthetic.pair_noise((1, 3, 48, 64), 0.1, seed=4))
    net = network(2)
    params = list(net.parameters())

    def forward_backward():
        loss = fb.l1_dssim_loss(net(a).contiguous(), b)
        grads = torch.autograd.grad(loss, params)
        return loss.detach(), fb.clip_grad_norm(grads, 0.05)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            loss, (clipped, norm) = forward_backward()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = forward_backward()
    graph.replay()
    torch.cuda.synchronize()
    assert abs(captured[0].item() - loss.item()) <= 1e-6
    assert abs(captured[1][1].item() - norm.item()) <= 1e-4 * norm.item()
    scale = max(g.abs().max().item() for g in clipped)
    for g, w in zip(captured[1][0], clipped):
        assert (g - w).abs().max().item() <= 1e-4 * scale

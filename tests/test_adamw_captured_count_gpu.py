"""A step whose count is a host number is not captured, nor one that makes states: each replay would take
the same count, or begin with zeros."""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_refused_under_capture(bits):
    p, q = (torch.nn.Parameter(torch.randn(300, generator=torch.Generator().manual_seed(1)).cuda()) for _ in range(2))
    opt, ref = (fb.AdamW([t], state_bits=bits) for t in (p, q))
    p.grad = torch.randn_like(p)
    q.grad = p.grad.clone()
    opt.step()
    ref.step()
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capturable"):
            opt.step()
    graph.replay()
    for o in (opt, ref):
        o.step()
    assert torch.equal(p, q) and opt.state[p]["step"] == 2
    # the function's caller gives the count: a captured call with a host number stays as it was
    m, v, scales = fb.adamw_moments(p, bits)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        fb.adamw_step_([p.detach()], [p.grad], [m], [v], None if scales is None else [scales], step=1, lr=1e-3)


def test_first_step_under_capture():
    p, q = (torch.nn.Parameter(torch.ones(40, device="cuda")) for _ in range(2))
    opt = fb.AdamW([p, q], capturable=True)
    p.grad = torch.ones_like(p)
    opt.step()
    q.grad = torch.ones_like(q)  # q's first
    x = torch.zeros(8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="states"):
            opt.step()
    assert int(opt.state[p]["step"]) == 1 and not opt.state.get(q) and torch.equal(q, torch.ones_like(q))
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    assert int(opt.state[p]["step"]) == int(opt.state[q]["step"]) == 3


@pytest.mark.parametrize("first", [False, True])
def test_capturable_set_between_steps(first):
    """Counts go on where a group's setting changes."""
    sizes = (7, 300, 40)  # the first one may have its gradients late, when it counts with its group
    a, b = ([torch.nn.Parameter(torch.linspace(-1, 1, n, device="cuda")) for n in sizes] for _ in range(2))
    opt, ref = fb.AdamW(a, capturable=first), fb.AdamW(b)
    for step in range(6):
        if step in (2, 4):
            opt.param_groups[0]["capturable"] ^= True
        for p, q in list(zip(a, b))[step < 2 and not first:]:
            p.grad = torch.full_like(p, 0.1 * (step + 1))
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
        assert all(torch.equal(p, q) for p, q in zip(a[1:], b[1:])), step
        assert [int(opt.state[p]["step"]) for p in a[1:]] == [step + 1] * 2
        assert all(isinstance(opt.state[p]["step"], torch.Tensor) == opt.param_groups[0]["capturable"] for p in a[1:])
        if step >= 2 or first:
            assert int(opt.state[a[0]]["step"]) == step + 1


def test_unequal_counts_do_not_become_capturable():
    a = [torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2)]
    opt = fb.AdamW(a)
    for skip in (0, None):
        for i, p in enumerate(a):
            p.grad = None if i == skip else torch.ones_like(p)
        opt.step()
    opt.param_groups[0]["capturable"] = True
    kept = [p.detach().clone() for p in a]
    with pytest.raises(ValueError, match="same number of steps"):
        opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a, kept)) and [opt.state[p]["step"] for p in a] == [1, 2]

"""Tensors whose memory does not hold their numbers as they are: lazily negated views (the imaginary
part of a conjugate), and tensors that have no memory, give the same results as copies of them, or
are refused."""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu


def negated(t):
    """t as a view of -t that is negated when it is read, and dense like t."""
    v = torch._neg_view(-t)
    assert v.is_neg() and v.stride() == t.stride() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("layout", [torch.contiguous_format, torch.channels_last])
def test_group_norm(layout):
    x = torch.randn(2, 12, 6, 8, device="cuda").contiguous(memory_format=layout)
    w, b, dy = torch.randn(12, device="cuda"), torch.randn(12, device="cuda"), torch.randn_like(x)

    def run(x, w, b, dy):
        ins = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = fb.group_norm_act(ins[0], 3, ins[1], ins[2])
        return (y, fb.group_norm_act(x, 3, w, b)) + torch.autograd.grad(y, ins, dy)

    want = run(x, w, b, dy)
    for i in range(4):
        args = [x, w, b, dy]
        args[i] = negated(args[i])
        assert all(torch.equal(p, q) for p, q in zip(run(*args), want)), i


def test_clipping():
    grads = [torch.randn(1000, device="cuda"), torch.randn(7, 5, device="cuda")]
    want, norm = fb.clip_grad_norm(grads, 1.0)
    lazy = [negated(g) for g in grads]
    assert torch.equal(fb.grad_norm(lazy), norm)
    for given in (lazy, [lazy[0], grads[1]]):
        out, got = fb.clip_grad_norm(given, 1.0)
        assert torch.equal(got, norm) and all(torch.equal(p, q) for p, q in zip(out, want))
        out = [torch._neg_view(torch.zeros_like(g)) for g in grads]
        _, got = fb.clip_grad_norm(given, 1.0, out=out)
        assert torch.equal(got, norm) and all(torch.equal(p, q) for p, q in zip(out, want))
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, lazy):
        p.grad = g
    assert torch.equal(fb.clip_grad_norm_(params, 1.0), norm)
    assert all(torch.equal(p.grad, q) for p, q in zip(params, want))
    # the public way there: one number fills its memory whatever its stride
    z = torch.complex(torch.ones(1, device="cuda"), torch.full((1,), 3.0, device="cuda"))
    g = z.conj().imag
    assert g.is_neg() and fb.clip_grad_norm([g], 10.0)[0][0].item() == -3.0


def test_a_weight_without_memory():
    # no pointer means no weight in the C call; it must not be taken for that
    x = torch.randn(2, 12, 6, 8, device="cuda")
    zero = torch._efficientzerotensor(12, device="cuda")
    for args in ((zero, None), (None, zero)):
        with pytest.raises(RuntimeError, match="memory"):
            fb.group_norm_act(x, 3, *args)

"""Outputs of clip_grad_norm that do not fill their memory: refused exactly where one of them gives a
number two places, or two of them share one; results are right everywhere else.

Whether they do is counted here from the indices of every number's bytes. Tolerances as in
test_grad_clip_gpu.py (5 u and half a step, u = 2^-24).
"""

import random

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def places(t):
    """First byte of every number."""
    at = torch.full((), t.storage_offset())
    for d in range(t.dim()):
        at = at.unsqueeze(-1) + torch.arange(t.size(d)) * t.stride(d)
    return [i * t.element_size() for i in at.flatten().tolist()]


def in_conflict(outs):
    taken = set()
    for t in outs:
        for first in places(t):
            for byte in range(first, first + t.element_size()):
                if byte in taken:
                    return True
                taken.add(byte)
    return False


def attempt(outs):
    """Clips into outs; returns whether the call was refused, and checks it if not."""
    gen = torch.Generator().manual_seed(len(outs))
    grads = [torch.randn(t.shape, generator=gen).to(t.dtype).cuda() for t in outs]
    try:
        _, norm = fb.clip_grad_norm(grads, 0.5, out=outs)
    except ValueError as e:
        assert "overlap" in str(e)
        return True
    coef = min(1.0, 0.5 / (norm.double().item() + 1e-6))
    for g, o in zip(grads, outs):
        ref = g.double() * coef
        assert ((o.double() - ref).abs() <= ref.abs() * (10 * 2.0 ** -24 + torch.finfo(o.dtype).eps / 2)).all()
    return False


def test_slices_of_one_buffer():
    b = torch.zeros(24, 36, device="cuda")
    flat = b.view(-1)
    for outs, refused in (
        ([flat[0::2][:50], flat[2::2][:50]], True),     # the even numbers, twice
        ([flat[0::2], flat[1::2]], False),              # even and odd
        ([flat[0:400:2], flat[400::2]], False),         # one behind the other
        ([flat[0:402:2], flat[400::2]], True),
        ([b[:, ::2], b[:, 1::2]], False),
        ([b[:, ::2], b[:, 2::2]], True),
        ([b[:, :20], b[:, 20:]], False),
        ([b[:, :21], b[:, 20:]], True),
        ([b[:, :10], b[5]], True),                      # columns and a row
        ([b[:, :10], b[5, 10:]], False),
        ([b[:12, ::3], b[12:]], False),
        ([b.t()[1::2], b[:, ::2]], False),
        ([b.t()[1::2], b[:, 1::4]], True),
        ([b[:, i] for i in range(36)], False),
        ([b[:, i] for i in range(36)] + [b[23:, 35]], True),
        ([flat.as_strided((4, 4), (1, 1))], True),      # overlap themselves
        ([flat.as_strided((4, 6), (5, 1))], True),
        ([flat.as_strided((4, 5), (6, 1))], False),
        ([flat.as_strided((4, 4), (2, 3))], True),
        ([flat.as_strided((3, 4), (2, 3))], False),
        ([flat.as_strided((3, 2), (2, 3))], False),
    ):
        assert in_conflict(outs) == refused
        for order in (outs, outs[::-1]):
            assert attempt(order) == refused, [(t.shape, t.stride(), t.storage_offset()) for t in order]


def test_column_views_in_place():
    b = torch.randn(40, 300, device="cuda")
    kept = b.clone()
    params = [torch.nn.Parameter(torch.zeros(40, device="cuda")) for _ in range(300)]
    for i, p in enumerate(params):
        p.grad = b[:, i]
    norm = fb.clip_grad_norm_(params, 1.0).item()
    assert ((b - kept / (norm + 1e-6)).abs() <= 10 * 2.0 ** -24 * kept.abs()).all()
    params[7].grad = b[:, 8]
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm_(params, 1.0)


@pytest.mark.parametrize("count", [1, 2, 3])
@pytest.mark.parametrize("seed", range(4))
def test_any_views(count, seed):
    r = random.Random(100 * count + seed)
    seen = {True: 0, False: 0}
    for _ in range(100):
        store = torch.zeros(512, device="cuda")
        outs = []
        for _ in range(count):
            t = store if r.random() < 0.7 else store.view(BF16)
            while True:
                shape = [r.randint(1, 4) for _ in range(r.randint(0, 3))]
                stride = [r.choice([1, 1, 2, 3, 4, 5, 7, 8, 12, 16, 20, 32, 60]) for _ in shape]
                offset = r.randint(0, 80)
                if offset + sum((n - 1) * s for n, s in zip(shape, stride)) < t.numel():
                    break
            outs.append(t.as_strided(shape, stride, offset))
        want = in_conflict(outs)
        assert attempt(outs) == want, [(t.dtype, t.shape, t.stride(), t.storage_offset()) for t in outs]
        seen[want] += 1
    assert all(seen.values())  # both answers came up


def test_large_nested_strides_are_quick():
    # found without walking the numbers: two interleaved views of 64 million numbers, six dimensions
    b = torch.zeros(2 ** 27, device="cuda").view(8, 16, 32, 64, 64, 8)
    a, c = b[..., ::2], b[..., 1::2]
    grads = [torch.ones_like(a), torch.ones_like(c)]
    _, norm = fb.clip_grad_norm(grads, 1e9, out=[a, c])
    assert abs(norm.item() - 2.0 ** 13.5) <= 4 * 2.0 ** -24 * 2.0 ** 13.5
    assert (b == 1).all()
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm(grads, 1e9, out=[a, b[..., ::2]])

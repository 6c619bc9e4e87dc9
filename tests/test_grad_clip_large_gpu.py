"""Clipping calls so large that the scaling comes in several pieces for each range of the norm's pass
(from twice 444 x 16 units of 2,048 numbers, 29 million, into other buffers), over one table of
tensors or several. Tolerances as in test_grad_clip_gpu.py.
"""

import pytest
import torch

import fussim_b200 as fb

from .test_grad_clip_gpu import BF16, F16, F32, check

pytestmark = pytest.mark.gpu

UNIT = 2048
ONE_CUT = 444 * 16 * UNIT  # numbers from which on a range has one cut, two from twice as many


def fill(shape, dtype, gen, scale):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


LARGE = {
    # just below and above two cuts, one tensor
    "one_below": ([2 * ONE_CUT - UNIT], F32, F32),
    "one_at": ([2 * ONE_CUT - UNIT + 1], F32, F32),
    "one_odd": ([3 * ONE_CUT + 12_345], F32, F32),
    # many cuts, ragged tensors of every size among long ones
    "ragged": ([20_000_003, 1, 7, 0, 33_333_333, 2047, 2049, 5, 40_000_001, 16, 1_000_001], BF16, F32),
    "ragged_same": ([20_000_003, 1, 7, 0, 33_333_333, 2047, 2049, 5, 40_000_001, 16, 1_000_001], F16, F16),
    # several tables, the first with one cut, or all with several
    "tables": ([(i * 7919) % 30_011 for i in range(1700)] + [70_000_001], BF16, BF16),
    "all_tables": ([40_000 + i for i in range(1700)], F32, F32),
}


@pytest.mark.parametrize("case", LARGE)
def test_into_other_buffers(case):
    sizes, dtype, out_dtype = LARGE[case]
    gen = torch.Generator(device="cuda").manual_seed(len(sizes))
    grads = [fill(n, dtype, gen, 0.1 + (i % 5)) for i, n in enumerate(sizes)]
    kept = [g.clone() for g in grads]
    outs = [torch.full((n,), 7.0, device="cuda", dtype=out_dtype) for n in sizes]
    first = None
    for _ in range(2):
        _, norm = fb.clip_grad_norm(grads, 3.0, out=outs)
        check(outs, norm, grads, 3.0)
        first = first or (norm.clone(), [o.clone() for o in outs])
    assert torch.equal(norm, first[0]) and all(torch.equal(p, q) for p, q in zip(outs, first[1]))
    assert all(torch.equal(g, k) for g, k in zip(grads, kept))
    # within the limit: copies
    _, norm = fb.clip_grad_norm(grads, float("inf"), out=outs)
    check(outs, norm, grads, float("inf"))


@pytest.mark.parametrize("packed", [False, True])
def test_some_in_place_some_not(packed):
    gen = torch.Generator(device="cuda").manual_seed(9)
    sizes = [30_000_001, 5, 12_000_000, 3001]
    if packed:  # pieces of one buffer without gaps, into pieces of another with another offset
        src, dst = fill(sum(sizes) + 3, F32, gen, 1.0), torch.full((sum(sizes) + 8,), 7.0, device="cuda")
        grads = list(src[3:].split(sizes))
        outs = list(dst[1:-7].split(sizes))
    else:
        grads = [fill(n, F32, gen, 1.0) for n in sizes]
        outs = [torch.zeros_like(g) for g in grads]
    outs[2] = grads[2]
    kept = [g.clone() for g in grads]
    _, norm = fb.clip_grad_norm(grads, 3.0, out=outs)
    check(outs, norm, kept, 3.0)
    assert all(torch.equal(grads[i], kept[i]) for i in (0, 1, 3))
    if packed:
        assert (dst[:1] == 7).all() and (dst[-7:] == 7).all()
        assert (dst[1:-7].split(sizes)[2] == 7).all()


def test_in_a_graph():
    gen = torch.Generator(device="cuda").manual_seed(10)
    grads = [fill(n, BF16, gen, 1.0) for n in (25_000_000, 9, 11_000_001)]
    outs = [torch.zeros(g.shape, device="cuda") for g in grads]
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        _, norm = fb.clip_grad_norm(grads, 2.0, out=outs)
    for scale in (1.0, 3.0):
        for g in grads:
            g.copy_(fill(g.shape, BF16, gen, scale))
        graph.replay()
        torch.cuda.synchronize()
        check(outs, norm, grads, 2.0)

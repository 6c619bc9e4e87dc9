"""grad_norm, clip_grad_norm and clip_grad_norm_ against their definition in 64 bits.

Tolerances. u = 2^-24. Squares of up to 32 numbers are summed in FP32 as a tree with at most six
roundings on the way of any term (all positive: 6 u relative), everything else in FP64, so the
norm before its rounding is off by 3 u and by 4 u after; the factor by 4 u (3 u and its own
rounding), a scaled number by 5 u (the product's) and half a step of its type.
"""

import math

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t, ref):
    f = torch.finfo(t)
    return (ref.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)


def exact(grads, max_norm):
    norm = math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in grads))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def check(outs, norm, grads, max_norm):
    want, coef = exact(grads, max_norm)
    assert norm.dtype == F32 and norm.shape == () and norm.is_cuda
    assert abs(norm.item() - want) <= 4 * U * want
    for o, g in zip(outs, grads):
        ref = g.double() * coef
        tol = 5 * U * ref.abs() + half_step(o.dtype, ref)
        assert ((o.double() - ref).abs() <= tol).all()


def tensors(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda()
            for i, s in enumerate(sizes)]


SIZES = {
    "one": [1],
    "small": [1, 2, 7, 8, 9, 0, 15, 16, 17],
    "units": [2047, 2048, 2049, 4096, 0, 0, 6145],
    "long": [1_000_003],
    "ragged": [5, 300_001, 1, 64, 77_777, 2, 0, 1024],
    "gaussians": [(997, 3), (997, 1, 3), (997, 15, 3), (997, 1), (997, 3), (997, 4)],
}


@pytest.mark.parametrize("dtypes", [(F32,), (F16,), (BF16,), (F32, BF16, F16)],
                         ids=["f32", "f16", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", SIZES)
def test_values(sizes, dtypes):
    grads = tensors(SIZES[sizes], dtypes, 3)
    norm, _ = exact(grads, 1.0)
    assert abs(fb.grad_norm(grads).item() - norm) <= 4 * U * norm
    for limit in (0.0, 0.25 * norm, 4 * norm, float("inf")):
        kept = [g.clone() for g in grads]
        out, got = fb.clip_grad_norm(grads, limit)                      # new tensors
        check(out, got, grads, limit)
        assert [o.dtype for o in out] == [g.dtype for g in grads]
        wide = [torch.full(g.shape, 7.0, device="cuda") for g in grads]   # 32-bit buffers
        out, got = fb.clip_grad_norm(grads, limit, out=wide)
        assert all(o is w for o, w in zip(out, wide))
        check(wide, got, grads, limit)
        assert all(torch.equal(g, k) for g, k in zip(grads, kept))      # inputs as they were
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g.clone()
        got = fb.clip_grad_norm_(params, limit)                         # in place
        check([p.grad for p in params], got, grads, limit)
        if limit > norm:
            assert all(torch.equal(p.grad, g) for p, g in zip(params, grads))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_at_any_offset(dtype):
    # pieces of one buffer, packed without gaps, into a buffer with another offset
    sizes = [1, 3, 5000, 7, 4097, 2, 9001]
    for src_shift in range(0, 9):
        for dst_shift in (0, 1, src_shift):
            src = torch.randn(sum(sizes) + src_shift, device="cuda").to(dtype)
            dst = torch.full((sum(sizes) + dst_shift + 5,), 3.0, device="cuda", dtype=dtype)
            gs, os_, a, b = [], [], src_shift, dst_shift
            for n in sizes:
                gs.append(src[a:a + n])
                os_.append(dst[b:b + n])
                a, b = a + n, b + n
            _, norm = fb.clip_grad_norm(gs, 1.0, out=os_)
            check(os_, norm, gs, 1.0)
            assert (dst[:dst_shift] == 3).all() and (dst[b:] == 3).all()  # nothing beside them


def test_many_tensors():
    sizes = [(i * 37) % 900 for i in range(2100)]  # several tables
    grads = tensors(sizes, (F32, BF16), 5)
    check([], fb.grad_norm(grads), grads, 1.0)
    out, norm = fb.clip_grad_norm(grads, 2.0)
    check(out, norm, grads, 2.0)


def test_strided_tensors():
    base = torch.randn(64, 48, device="cuda")
    conv = torch.randn(8, 6, 3, 3, device="cuda").to(memory_format=torch.channels_last)
    grads = [base[:, ::2], base.t()[1::2], conv, torch.randn(5, device="cuda").expand(3, 5)]
    out, norm = fb.clip_grad_norm(grads, 1.0)
    check(out, norm, grads, 1.0)
    # in place: column views of one buffer, and a dense permuted tensor
    kept = [g.clone() for g in grads[:3]]
    untouched = base[1::2].clone()
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads[:3]]
    for p, g in zip(params, grads[:3]):
        p.grad = g
    norm = fb.clip_grad_norm_(params, 1.0)
    check(grads[:3], norm, kept, 1.0)
    # outputs of other strides than the gradients
    out = [torch.zeros(24, 64, device="cuda").t(), torch.zeros(8, 6, 3, 3, device="cuda")]
    _, norm = fb.clip_grad_norm([kept[0], kept[2]], 1.0, out=out)
    check(out, norm, [kept[0], kept[2]], 1.0)


def test_range_of_values():
    for value in (1e30, 1e-30, 3e38, 1e-42):
        g = torch.full((10_001,), value, device="cuda")
        want = g[0].double().item() * math.sqrt(10_001)
        got = fb.grad_norm([g]).item()
        if want > torch.finfo(F32).max:
            assert got == float("inf")
        else:
            assert abs(got - want) <= 4 * U * want + 2.0 ** -150
    zeros = [torch.zeros(100, device="cuda"), torch.zeros(7, device="cuda", dtype=BF16)]
    out, norm = fb.clip_grad_norm(zeros, 1.0)
    assert norm.item() == 0.0 and not any(o.any() for o in out)
    # beyond FP32's range the norm is infinite, the factor not: it comes from the FP64 norm
    g = torch.full((10_001,), 1e38, device="cuda")
    out, norm = fb.clip_grad_norm([g], 1.0)
    assert norm.item() == float("inf")
    want = 1.0 / math.sqrt(10_001)
    assert ((out[0].double() - want).abs() <= 8 * U * want).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_nonfinite(bad, dtype):
    grads = tensors([100, 3000, 5], (dtype,), 6)
    grads[1][1234] = bad
    mine = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    ref = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, q, g in zip(mine, ref, grads):
        p.grad, q.grad = g.clone(), g.clone()
    with pytest.raises(RuntimeError, match="norm is"):
        fb.clip_grad_norm_(mine, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(p.grad[:1000], g[:1000]) for p, g in zip(mine, grads))
    got = fb.clip_grad_norm_(mine, 1.0)
    want = torch.nn.utils.clip_grad_norm_(ref, 1.0, foreach=False)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    for p, q in zip(mine, ref):
        assert torch.equal(p.grad.isnan(), q.grad.isnan())
        assert torch.equal(p.grad.nan_to_num(), q.grad.nan_to_num())
    fb.clip_grad_norm_(mine[2:], 1.0, error_if_nonfinite=not math.isnan(bad))


def test_empty_lists():
    assert fb.grad_norm([]).item() == 0.0
    out, norm = fb.clip_grad_norm([], 1.0)
    assert out == [] and norm.item() == 0.0
    assert fb.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0).item() == 0.0
    assert fb.grad_norm([torch.zeros(0, device="cuda")]).item() == 0.0


def test_one_parameter_and_generators():
    p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
    p.grad = torch.ones(10, device="cuda")
    assert abs(fb.clip_grad_norm_(p, 1.0).item() - math.sqrt(10)) <= 1e-6
    fb.clip_grad_norm_((q for q in [p]), 0.5)
    assert abs(p.grad.norm().item() - 0.5) <= 1e-5
    assert abs(fb.grad_norm(q.grad for q in [p]).item() - 0.5) <= 1e-5


def test_refusals():
    a = torch.randn(100, device="cuda")
    b = torch.randn(100, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a, a], 1.0, out=[a, a])          # the same tensor twice
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a[:60], a[40:]], 1.0, out=[a[:60], a[40:]])
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a, b], 1.0, out=[b, a])          # onto each other
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a[:50], b[:50]], 1.0, out=[a[1:51], b[:50]])
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a, b], 1.0, out=[torch.zeros_like(a)] * 2)
    half = torch.zeros(100, device="cuda", dtype=F16)
    with pytest.raises(ValueError, match="overlap"):        # the gradient's memory as 32 bits
        fb.clip_grad_norm([half[:50]], 1.0, out=[half.view(F32)])
    wide = torch.zeros(100, 2, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a, b], 1.0, out=[wide[:, 0], wide[:, 0]])
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm([a], 1.0, out=[torch.zeros(1, device="cuda").expand(100)])
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = a
    with pytest.raises(ValueError, match="overlap"):
        fb.clip_grad_norm_([p, p], 1.0)
    with pytest.raises(ValueError, match="shape"):
        fb.clip_grad_norm([a], 1.0, out=[a.view(10, 10)])
    with pytest.raises(ValueError, match="float32"):
        fb.clip_grad_norm([a], 1.0, out=[torch.zeros(100, device="cuda", dtype=F16)])
    with pytest.raises(RuntimeError, match="one device"):
        fb.grad_norm([a, b.cpu()])
    with pytest.raises(RuntimeError, match="on cuda"):
        fb.clip_grad_norm([a], 1.0, out=[torch.zeros(100)])
    # read twice is no trouble
    out, norm = fb.clip_grad_norm([a, a], 1.0)
    check(out, norm, [a, a], 1.0)


def test_saved_tensors_notice():
    g = torch.randn(10, device="cuda")
    leaf = torch.randn(10, device="cuda", requires_grad=True)
    y = (leaf * g).sum()
    fb.clip_grad_norm([g], 0.1, out=[g])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_repeats_and_streams():
    grads = tensors([300_000, 5, 70_001, 1024], (F32, BF16), 7)
    want, norm = fb.clip_grad_norm(grads, 1.0)
    torch.cuda.synchronize()
    results = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            results += [fb.clip_grad_norm(grads, 1.0) for _ in range(4)]
    torch.cuda.synchronize()
    for out, n in results:
        assert torch.equal(n, norm) and all(torch.equal(p, q) for p, q in zip(out, want))


@pytest.mark.parametrize("more", [0, 400])
def test_graphs_replay_together(more):
    sizes = [50_000, 7, 3000] + [100 + i for i in range(more)]  # a small table and a large one
    graphs = []
    for k in range(2):
        grads = tensors([n + k for n in sizes], (F32, F16), 8 + k)
        params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(params, grads):
            p.grad = g
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            norm = fb.clip_grad_norm_(params, 0.5)
        graphs.append((graph, torch.cuda.Stream(), grads, norm))
    for round_ in range(3):
        fresh = []
        for k, (_, _, grads, _) in enumerate(graphs):
            fresh.append(tensors([n + k for n in sizes], (F32, F16), 40 + 2 * round_ + k))
            for g, f in zip(grads, fresh[-1]):
                g.copy_(f)
        torch.cuda.synchronize()
        for graph, s, _, _ in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, grads, norm), f in zip(graphs, fresh):
            check(grads, norm, f, 0.5)


def test_more_than_two_to_the_31_numbers():
    n = 2 ** 31 + 12_345
    g = torch.full((n,), 0.5, dtype=BF16, device="cuda")
    g[-1] = 64.0
    want = math.sqrt(0.25 * (n - 1) + 4096.0)
    norm = fb.grad_norm([g]).item()
    assert abs(norm - want) <= 4 * U * want
    _, got = fb.clip_grad_norm([g], 1.0, out=[g])
    assert got.item() == norm
    coef = 1.0 / (want + 1e-6)
    for at, v in ((0, 0.5), (n - 2, 0.5), (n - 1, 64.0), (2 ** 31 + 1, 0.5)):
        ref = torch.tensor(v * coef, dtype=torch.float64)
        assert abs(g[at].double().item() - ref.item()) <= (half_step(BF16, ref) + 5 * U * ref).item()
    assert (g[:-1] == g[0]).all()


def test_a_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    grads = tensors([300_000, 5], (F32,), 7)
    want, norm = fb.clip_grad_norm(grads, 1.0)
    out, got = fb.clip_grad_norm([g.to("cuda:1") for g in grads], 1.0)
    assert got.device.index == 1 and got.item() == norm.item()
    assert all(torch.equal(p.cpu(), q.cpu()) for p, q in zip(out, want))

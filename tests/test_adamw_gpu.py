"""adamw_step_ against its definition: in 64 bits, and bit for bit in its own steps of 32 bits.

Tolerances against 64 bits. u = 2^-24, c the relative error of g * coef: 0 without clipping, else
4 u (the norm) + 2 u (the factor's rounding and the product's) = 6 u. Each constant is rounded to
FP32 (u). m: two products (a constant's and its own rounding: 2 u of each term) and the sum (u of
the result, at most of the terms): 3 u (b1 |m| + (1-b1)|g|) + c (1-b1)|g|. v, of positive terms:
g^2, its product with a rounded constant and the sum, 4 u, and 2 c. The denominator: half of v's
(2 u + c), the root's u, the constant's u, the product's u, eps's u and the sum's u: 7 u + c. The
quotient 1 u more, its constant and product 2 u; p * decay 2 u of |p| and the last difference u of
both. p's type adds half a step. Products of roundings are covered by 1 % more.
"""

import math

import pytest
import torch

import fussim_b200 as fb
from tests import adamw_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SET = dict(step=7, lr=3e-3, betas=(0.9, 0.98), eps=1e-8, wd=0.05)
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
SIZES = {
    "one": [1],
    "edges": [255, 256, 257, 0, 7, 8, 9, 511, 512],
    "units": [2047, 2048, 2049, 6145, 1],
    "long": [1_000_003],
    "many": [1 + 37 * i % 700 for i in range(70)],       # the large table
    "more": [1 + 11 * i % 300 for i in range(900)],      # several launches
}


def half_step(t, ref):
    f = torch.finfo(t)
    return (ref.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)


def tensors(sizes, dtype, seed, scale=1.0, gap=None):
    """Tensors of their own memory, or pieces of one buffer that begin `gap` numbers apart."""
    g = torch.Generator().manual_seed(seed)
    data = [(torch.randn(n, generator=g) * scale).to(dtype) for n in sizes]
    if gap is None:
        return [d.cuda() for d in data]
    flat = torch.zeros(sum(sizes) + gap * (len(sizes) + 1), device="cuda", dtype=dtype)
    out, at = [], gap
    for d in data:
        out.append(flat[at:at + d.numel()])
        out[-1].copy_(d)
        at += d.numel() + gap
    return out


def make(sizes, pt, gt, bits, seed=0, gap=None, copy=None):
    s = {"params": tensors(sizes, pt, seed, 0.1, gap), "grads": tensors(sizes, gt, seed + 1, 0.02, gap)}
    ms, rs = tensors(sizes, F32, seed + 2, 0.01, gap), tensors(sizes, F32, seed + 3, 0.02, gap)
    for r in rs:
        r.abs_()
    if bits == 32:
        s["exp_avgs"], s["exp_avg_sqs"] = ms, [r.square_() for r in rs]
    else:
        s["scales"] = [torch.empty(-(-n // 256), 2, device="cuda") for n in sizes]
        for k, column, parts in (("exp_avgs", 0, ms), ("exp_avg_sqs", 1, rs)):
            s[k] = tensors(sizes, torch.float8_e4m3fn, 0, 0.0, gap)
            for codes, scale, part in zip(s[k], s["scales"], parts):
                b = O.blocks(part)
                top, scale[:, column:column + 1] = O.scale_of(b.cpu())
                codes.copy_((b / scale[:, column:column + 1]).view(-1)[:part.numel()])
    if copy:
        s["copies"] = tensors(sizes, copy, seed, 0.0, gap)
    return s


def snapshot(s):
    return {k: [t.detach().cpu().clone() for t in v] for k, v in s.items()}


def run(s, seed=5, **kw):
    d = dict(SET, **kw)
    d["weight_decay"] = d.pop("wd")
    return fb.adamw_step_(**s, seed=seed, **d)


def unlike(a, b):
    """Where two tensors' numbers differ (NaN counts as equal to NaN): "" if nowhere."""
    if a.dtype != b.dtype or a.shape != b.shape:
        return f"{a.dtype} {a.shape}, {b.dtype} {b.shape}"
    a, b = a.detach().cpu().double().flatten(), b.detach().cpu().double().flatten()
    at = ((a != b) & ~(a.isnan() & b.isnan())).nonzero().flatten()
    return f"{len(at)} of {len(a)}, at {at[:4].tolist()}: {a[at[:4]].tolist()}, {b[at[:4]].tolist()}" if len(at) else ""


def same(a, b):
    return not unlike(a, b)


def check_bits(before, s, coef=1.0, seed=5, first=0, **kw):
    """Every output equals the definition's own steps of 32 bits."""
    for i, p in enumerate(before["params"]):
        state = [before[k][i].flatten() for k in ("exp_avgs", "exp_avg_sqs")]
        scales = before["scales"][i] if "scales" in before else None
        want = O.step32(p.flatten(), before["grads"][i].flatten(), *state, scales, coef=coef, seed=seed,
                        tensor=first + i, **dict(SET, **kw))
        got = [s[k][i].cpu().flatten() for k in ("params", "exp_avgs", "exp_avg_sqs")]
        found = unlike(got[0], want[0].to(p.dtype))
        assert not found, f"parameter {i}: {found}"
        found = unlike(got[1], want[1])
        assert not found, f"exp_avg {i}: {found}"
        found = unlike(got[2], want[2])
        assert not found, f"exp_avg_sq {i}: {found}"
        if scales is not None:
            found = unlike(s["scales"][i].cpu(), want[3])
            assert not found, f"scales {i}: {found}"
        if "copies" in s:
            found = unlike(s["copies"][i].cpu().flatten(), want[0].to(s["copies"][i].dtype))
            assert not found, f"copy {i}: {found}"
        assert same(s["grads"][i].cpu(), before["grads"][i])


def check_definition(before, s, coef=1.0, c=0.0, **kw):
    d = dict(SET, **kw)
    b1, lr, t = d["betas"][0], d["lr"], d["step"]
    for i, p in enumerate(before["params"]):
        g = before["grads"][i].double().flatten() * coef
        if "scales" in before:
            m, r = (O.decode(before[k][i], before["scales"][i], j) for j, k in enumerate(("exp_avgs", "exp_avg_sqs")))
            v = r.double() ** 2
        else:
            m, v = before["exp_avgs"][i].flatten(), before["exp_avg_sqs"][i].flatten()
        want, wm, wv, change, den = O.step64(p.flatten(), before["grads"][i].flatten(), m, v, coef=coef, **d)
        tol_m = 3 * U * (b1 * m.double().abs() + (1 - b1) * g.abs()) + c * (1 - b1) * g.abs()
        rate = lr / (1 - b1 ** t)
        tol = rate * (tol_m / den + (10 * U + c) * change.abs()) + 3 * U * p.double().flatten().abs() + U * want.abs()
        for k in ("params", "copies"):
            if k in s:
                got = s[k][i].cpu().flatten()
                # (v's codes give g^2 + r^2 an extra rounding, of r^2)
                assert ((got.double() - want).abs() <= 1.01 * tol + half_step(got.dtype, want)).all()
        if "scales" not in s:
            tiny = 2.0 ** -149
            assert ((s["exp_avgs"][i].cpu().flatten().double() - wm).abs() <= 1.01 * tol_m + tiny).all()
            assert ((s["exp_avg_sqs"][i].cpu().flatten().double() - wv).abs() <= (4.04 * U + 2 * c) * wv + 4 * tiny).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gap", [None, 0, 1], ids=["own", "packed", "odd"])
@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("sizes", ["edges", "units"])
def test_step(sizes, types, gap, bits):
    s = make(SIZES[sizes], *types, bits, gap=gap)
    before = snapshot(s)
    assert run(s) is None
    check_bits(before, s)
    check_definition(before, s)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", ["one", "long", "many", "more"])
def test_sizes(sizes, bits):
    s = make(SIZES[sizes], BF16 if sizes == "many" else F32, F32, bits, seed=3)
    before = snapshot(s)
    run(s)
    check_bits(before, s)
    check_definition(before, s)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gt", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("ct", [F16, BF16], ids=str)
def test_copies(ct, gt, bits):
    for gap in (None, 1):
        s = make(SIZES["edges"], F32, gt, bits, gap=gap, copy=ct)
        before = snapshot(s)
        run(s)
        check_bits(before, s)
        check_definition(before, s)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("limit", [0.0, 1e-3, 0.05, 1e3])
def test_clipping(limit, bits):
    s = make(SIZES["units"] + SIZES["edges"], F32, BF16, bits, copy=BF16)
    before = snapshot(s)
    norm = run(s, max_norm=limit)
    exact = math.sqrt(math.fsum((g.double() ** 2).sum().item() for g in before["grads"]))
    assert norm.shape == () and abs(norm.item() - exact) <= 4 * U * exact
    ratio = limit / (norm.double().cpu() + 1e-6)
    check_bits(before, s, coef=min(1.0, ratio.item()))
    check_definition(before, s, coef=min(1.0, limit / (exact + 1e-6)), c=6 * U if limit < exact else 0.0)


def test_given_norm_and_maximize():
    s = make(SIZES["edges"], F32, F32, 32)
    before = snapshot(s)
    norm = torch.tensor(4.0, device="cuda")
    assert run(s, max_norm=1.0, norm=norm, maximize=True) is norm
    check_bits(before, s, coef=-1.0 / (4.0 + 1e-6))


def test_first_step_and_settings():
    for kw in (dict(step=1), dict(step=1, betas=(0.0, 0.0)), dict(step=100_000, lr=0.0), dict(wd=0.0, eps=0.1),
               dict(step=2, betas=(0.95, 0.9999))):
        for bits in (32, 8):
            s = make(SIZES["edges"], F32, F32, bits)
            if kw.get("step") == 1:
                for k in ("exp_avgs", "exp_avg_sqs", "scales"):
                    for t in s.get(k, []):
                        t.zero_()
            before = snapshot(s)
            run(s, **kw)
            check_bits(before, s, **kw)
            check_definition(before, s, **kw)


def test_zero_gradients_and_moments():
    """Numbers that have never had a gradient: only the decay moves them."""
    for bits in (32, 8):
        s = make([700], F32, F32, bits)
        for k in ("grads", "exp_avgs", "exp_avg_sqs"):
            s[k][0].zero_()
        before = snapshot(s)
        run(s)
        check_bits(before, s)
        assert same(s["params"][0].cpu(), before["params"][0] * torch.tensor(1.0 - SET["lr"] * SET["wd"]))
        assert not s["exp_avgs"][0].float().any() and not s["exp_avg_sqs"][0].float().any()


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits):
    """An infinite or NaN gradient spoils its own number and moments alone."""
    s = make([1000], F32, F32, bits)
    at = {3: math.inf, 300: -math.inf, 301: math.nan, 600: 1e30, 999: math.nan}
    for i, x in at.items():
        s["grads"][0][i] = x
    before = snapshot(s)
    run(s)
    check_bits(before, s)
    got = s["params"][0].cpu()
    assert got.isnan().nonzero().flatten().tolist() == [3, 300, 301, 999]
    if bits == 8:
        for k in ("exp_avgs", "exp_avg_sqs"):
            bad = s[k][0].float().isnan().nonzero().flatten().tolist()
            assert bad == ([3, 300, 301, 600, 999] if k == "exp_avg_sqs" else [3, 300, 301, 999])
        assert s["scales"][0].isfinite().all()
    before = snapshot(s)
    run(s, step=8)
    check_bits(before, s, step=8)


def test_roots_and_quotients():
    """All 2^24 roots of two binades, and as many quotients, are the correctly rounded ones: halved moments
    (exactly) and a rate of 1 leave a parameter of zero at minus the quotient."""
    n = 1 << 24
    v = (torch.arange(n, dtype=torch.int32, device="cuda") + 0x40000000).view(F32)  # [2, 8): halves in [1, 4)
    g = torch.Generator(device="cuda").manual_seed(1)
    m = torch.randn(n, device="cuda", generator=g) * torch.exp2(torch.randint(-30, 30, (n,), device="cuda", generator=g).float())
    s = {"params": [torch.zeros(n, device="cuda")], "grads": [torch.zeros(n, device="cuda")], "exp_avgs": [m],
         "exp_avg_sqs": [v]}
    before = snapshot(s)
    kw = dict(step=1, lr=0.5, betas=(0.5, 0.5), eps=2.0 ** -30, wd=0.0)
    run(s, **kw)
    check_bits(before, s, **kw)


@pytest.mark.parametrize("bits", [32, 8])
def test_norm_not_finite(bits):
    """A NaN norm makes everything NaN; an infinite one leaves finite gradients nothing."""
    for bad in (math.nan, math.inf):
        s = make([700, 3], F32, F32, bits)
        s["grads"][1][0] = bad
        before = snapshot(s)
        norm = run(s, max_norm=1.0)
        assert norm.isnan().item() if math.isnan(bad) else norm.isinf().item()
        check_bits(before, s, coef=math.nan if math.isnan(bad) else 0.0)
        assert s["params"][0].isnan().all().item() == math.isnan(bad)


def test_extremes_of_codes():
    """Blocks of one value, of tiny values, of a range beyond the codes', and of negative zeros."""
    s = make([256 * 6 + 5], F32, F32, 8)
    g = s["grads"][0]
    g[:256] = 0.25
    g[256:512] = 1e-38
    g[512:768] = torch.logspace(-30, 10, 256, device="cuda")
    g[768:1024] = -0.0
    g[1024:1280] = 3e38
    before = snapshot(s)
    run(s, step=1)
    check_bits(before, s, step=1)
    for step in range(2, 6):
        before = snapshot(s)
        run(s, step=step)
        check_bits(before, s, step=step)


def test_rounding_is_unbiased():
    """Codes stand for their numbers on average over seeds, within their two neighbours always."""
    n, seeds = 256, 400
    base = make([n], F32, F32, 8, seed=11)
    m, r = (O.decode(base[k][0].cpu(), base["scales"][0].cpu(), j) for j, k in enumerate(("exp_avgs", "exp_avg_sqs")))
    _, wm, wv, _, _ = O.step64(base["params"][0].cpu(), base["grads"][0].cpu(), m, r.double() ** 2, **SET)
    sums = [torch.zeros(n, dtype=torch.float64) for _ in range(2)]
    spans = [torch.zeros(n, dtype=torch.float64) for _ in range(2)]
    wants = [wm, wv.sqrt()]
    for seed in range(seeds):
        s = {k: [t.clone() for t in v] for k, v in base.items()}
        run(s, seed=seed)
        for j, k in enumerate(("exp_avgs", "exp_avg_sqs")):
            got = O.decode(s[k][0].cpu(), s["scales"][0].cpu(), j).double()
            sums[j] += got
            spans[j] = torch.maximum(spans[j], (got - wants[j]).abs())
    for j, want in enumerate(wants):
        scale = base["scales"][0][0, j].item()
        # codes are at most an eighth apart, and below 2^-6 scales 2^-9 scales
        step = (want.abs() / 8).clamp(min=2.0 ** -9 * s["scales"][0][0, j].item())
        assert (spans[j] <= 1.001 * step).all() and scale > 0
        inner = want.abs() > 2.0 ** -6 * s["scales"][0][0, j].item()
        # standard deviation of a mean over seeds: at most half a step / sqrt(seeds); six of them
        assert ((sums[j] / seeds - want).abs() <= 6 * step / 2 / math.sqrt(seeds))[inner].all()


def test_two_calls_are_alike():
    a, b = (make(SIZES["units"], BF16, BF16, 8) for _ in range(2))
    for s in (a, b):
        run(s, max_norm=0.1)
    for k in a:
        assert all(same(x, y) for x, y in zip(a[k], b[k]))
    # another seed or step draws other codes, and the same parameters
    c = make(SIZES["units"], BF16, BF16, 8)
    run(c, max_norm=0.1, seed=6)
    assert all(same(x, y) for x, y in zip(a["params"], c["params"]))
    assert not same(a["exp_avgs"][3], c["exp_avgs"][3])


def test_strides():
    """Channels-last parameters; a gradient of other strides, a negated and a sliced one."""
    for bits in (32, 8):
        w = torch.randn(6, 5, 3, 4, device="cuda").to(memory_format=torch.channels_last)
        like = lambda dt: torch.zeros_like(w, dtype=dt)  # noqa: E731
        dt = F32 if bits == 32 else torch.float8_e4m3fn
        wide = torch.randn(6, 5, 3, 8, device="cuda")
        for g in (torch.randn(6, 5, 3, 4, device="cuda"), wide[..., ::2],
                  torch.randn(6, 5, 3, 4, device="cuda", dtype=torch.complex64).conj().imag,
                  torch.randn(1, 5, 1, 1, device="cuda").expand(6, 5, 3, 4)):
            s = {"params": [w.clone(memory_format=torch.preserve_format)], "grads": [g], "exp_avgs": [like(dt)], "exp_avg_sqs": [like(dt)]}
            if bits == 8:
                s["scales"] = [torch.zeros(2, 2, device="cuda")]
            order = lambda t: t.permute(0, 2, 3, 1).reshape(-1).cpu()  # noqa: E731
            want = O.step32(order(w), order(g.resolve_neg()), order(s["exp_avgs"][0]), order(s["exp_avg_sqs"][0]),
                            s["scales"][0].cpu() if bits == 8 else None, seed=5, **dict(SET, step=1))
            norm = run(s, step=1, max_norm=1e9)
            exact = g.double().norm().item()
            assert abs(norm.item() - exact) <= 4 * U * exact
            for k, x in zip(("params", "exp_avgs", "exp_avg_sqs"), want):
                assert same(order(s[k][0]), x)


def test_overlap_is_refused():
    flat = torch.zeros(4096, device="cuda")
    p, g, m, v = flat[:500].clone(), flat[:500].clone(), flat[:500].clone(), flat[:500].clone()
    good = dict(params=[p], grads=[g], exp_avgs=[m], exp_avg_sqs=[v])
    run(good)
    for k in ("grads", "exp_avgs", "exp_avg_sqs"):
        with pytest.raises(ValueError, match="overlap"):
            run(dict(good, **{k: [p]}))
    with pytest.raises(ValueError, match="overlap"):
        run({k: t * 2 for k, t in good.items()})
    a, b = flat[:500], flat[499:999]
    with pytest.raises(ValueError, match="overlap"):
        run(dict(params=[a, b], grads=[g, g], exp_avgs=[m, m.clone()], exp_avg_sqs=[v, v.clone()]))
    # one gradient for two parameters is read twice
    run(dict(params=[p, p.clone()], grads=[g, g], exp_avgs=[m, m.clone()], exp_avg_sqs=[v, v.clone()]))
    with pytest.raises(ValueError, match="overlap"):
        run(good, max_norm=1.0, norm=p[3])


def test_device_numbers():
    """step and lr on the device: the same results as from the host."""
    for bits in (32, 8):
        a, b = (make(SIZES["edges"], F32, F32, bits) for _ in range(2))
        lr = torch.tensor(SET["lr"], device="cuda")
        run(a, step=torch.tensor(7.0, device="cuda"), lr=lr)
        run(b, lr=lr.item())
        for k in a:
            assert all(same(x, y) for x, y in zip(a[k], b[k])), k
    with pytest.raises(ValueError, match="one float32"):
        run(a, step=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="one float32"):
        run(a, lr=torch.ones((), device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError, match="device"):
        run(a, lr=torch.ones(()))


def test_graph():
    """Replays of a captured step, with the count and the rate on the device."""
    for bits in (32, 8):
        s, ref = (make([3000, 5, 70_001], F32, BF16, bits, copy=BF16) for _ in range(2))
        step, lr = torch.zeros((), device="cuda"), torch.tensor(1e-2, device="cuda")

        def body():
            step.add_(1)
            return run(s, step=step, lr=lr, max_norm=0.05)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = body()
        for t in range(1, 4):
            lr.fill_(1e-2 / t)
            for g, r in zip(s["grads"], ref["grads"]):
                g.copy_(torch.randn(g.shape, device="cuda") * 0.01 * t)
                r.copy_(g)
            graph.replay()
            want = run(ref, step=t, lr=lr.item(), max_norm=0.05)
            assert want.item() == norm.item()
            for k in s:
                assert all(same(x, y) for x, y in zip(s[k], ref[k])), (bits, t, k)


def test_other_stream():
    a, b = (make([300_000], F32, F32, 8) for _ in range(2))
    run(a, max_norm=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(b, max_norm=0.1)
    torch.cuda.current_stream().wait_stream(side)
    for k in a:
        assert all(same(x, y) for x, y in zip(a[k], b[k]))


def test_versions_and_empty():
    s = make([10], F32, F32, 32)
    was = [s[k][0]._version for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    run(s)
    now = [s[k][0]._version for k in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    assert [b > a for a, b in zip(was, now)] == [True, False, True, True]
    none = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[])
    assert run(none) is None and run(none, max_norm=1.0).item() == 0.0
    empty = make([0, 0], F32, F32, 8)
    assert run(empty) is None and run(empty, max_norm=1.0).item() == 0.0

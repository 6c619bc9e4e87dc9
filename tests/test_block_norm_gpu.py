"""block_norm, gated_residual and gated_residual_norm, forward and backward, against their
definition in 64 bits.

Tolerances. u = 2^-24. A row's sum of C numbers runs over at most 32 numbers of a thread, five
steps in a warp and 16 warps: k = 60 roundings bound its relative error (of the sum of
magnitudes), a few constants' included. Distances from a number of the row are off by u of
the row's range R, so a mean by E = k u R + u |mean|; the squares, all positive, by k u and their
root by half; a normalised number h = (v - mean) * rstd by

    D(v) = rstd E + |h| (k / 2 + 8) u.

Sums of products whose factors are off add those factors' errors. A vector's gradient is a sum over
rows, in FP32 over at most 256 of them in a thread, five steps in its warp, eight warps and three steps
between CTAs, FP64 beyond: n = min(rows, 256) + 16 roundings of the magnitudes' sum. Each
result adds half a step of its type; z is compared with the norm of the r that was returned.
"""

import itertools

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U, K = 2.0 ** -24, 60
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]
SHAPES = [
    (1, 1, 1), (2, 3, 2), (3, 5, 7), (1, 40, 8), (4, 9, 9), (2, 31, 31), (5, 7, 40), (2, 300, 64), (1, 17, 100),
    (3, 70, 255), (2, 9, 256), (2, 9, 257), (2, 33, 264), (3, 41, 403), (1, 700, 520), (2, 19, 1024), (2, 5, 1152),
    (1, 3, 2047), (1, 4, 4096), (2, 2, 4097), (1, 5, 5000), (2, 3, 8192), (1, 2, 8200), (1, 3, 16384), (1, 2, 16383),
    (40, 1, 48), (2, 3000, 16),
]
EPS = 1e-6


def half_step(t, ref):
    f = torch.finfo(t)
    return (ref.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)


def wide(t):
    return None if t is None else t.detach().double()


def per_row(v, x):
    """A vector of (C,) or (B, C) beside x (B, ..., C)."""
    return v if v.dim() == 1 else v.view(x.shape[0], *[1] * (x.dim() - 2), x.shape[-1])


def normed(v, kind, eps):
    """(h, D, rstd)"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    d = v - mean
    rstd = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = d * rstd
    away = K * U * (v.amax(-1, keepdim=True) - v.amin(-1, keepdim=True)) + U * mean.abs() if kind == "layer" else 0.0
    return h, rstd * away + h.abs() * (K / 2 + 8) * U, rstd


def normed_grad(e, e_off, h, h_off, rstd, kind):
    """The gradient of v for a gradient e (off by e_off) of h, and how far it may be off."""
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    m2 = mean(e * h)
    m2_off = K * U * mean((e * h).abs()) + mean(e_off * h.abs()) + mean(e.abs() * h_off)
    out = e - h * m2
    off = e_off + 4 * U * (e.abs() + (h * m2).abs()) + h.abs() * m2_off + h_off * m2.abs()
    if kind == "layer":
        out = out - mean(e)
        off = off + K * U * mean(e.abs()) + mean(e_off) + 2 * U * mean(e).abs()
    return out * rstd, rstd * off + out.abs() * rstd * (K / 2 + 4) * U


def near(name, got, want, off):
    assert got.shape == want.shape, name
    tol = 1.01 * off + half_step(got.dtype, want) + 1e-44
    bad = ((got.detach().double() - want).abs() - tol).amax().item() if want.numel() else -1.0
    assert not bad > 0 and bool(got.isfinite().all()), f"{name}: {bad:.3g} beyond its tolerance"


def make(b, t, c, xt, yt, gate="none", branch_kind=None, kind="rms", mod=False, form="both", seed=0, wt=None):
    g = torch.Generator().manual_seed(seed + 1000 * c + t)
    randn = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    wt = wt or xt
    d = {"x": (randn(b, t, c) + 0.3 * randn(c)).to(xt)}
    if form != "before":
        d["branch"] = (0.2 + randn(b, t, c)).to(yt)
        if gate != "none":
            d["gate"] = (0.5 * randn(*((c,) if gate == "channel" else (b, c)))).to(wt)
        if branch_kind:
            d["branch_weight"] = (1 + 0.2 * randn(c)).to(wt)
            if branch_kind == "layer":
                d["branch_bias"] = (0.2 * randn(c)).to(wt)
    if form != "after":
        d["weight"] = (1 + 0.2 * randn(c)).to(wt)
        if kind == "layer":
            d["bias"] = (0.2 * randn(c)).to(wt)
        if mod:
            d["scale"], d["shift"] = (0.3 * randn(b, c)).to(wt), (0.3 * randn(b, c)).to(wt)
    return {k: v.cuda() for k, v in d.items()}


def call(d, form, kind="rms", branch_kind=None, s=1.0, eps=EPS, out_dtype=None):
    """(r or None, z or None)"""
    at = d.get
    if form == "before":
        return None, fb.block_norm(d["x"], at("weight"), at("bias"), scale=at("scale"), shift=at("shift"), kind=kind,
                                   eps=eps, out_dtype=out_dtype)
    after = dict(residual_scale=s, branch_kind=branch_kind, branch_weight=at("branch_weight"),
                 branch_bias=at("branch_bias"), eps=eps)
    if form == "after":
        return fb.gated_residual(d["x"], d["branch"], at("gate"), **after), None
    return fb.gated_residual_norm(d["x"], d["branch"], at("gate"), at("weight"), at("bias"), scale=at("scale"),
                                  shift=at("shift"), kind=kind, **after)


def check(d, form, r, z, kind="rms", branch_kind=None, s=1.0, eps=EPS, ups=None, grads=None):
    """Results, and gradients for the given ones of r and z, against the definition."""
    w = {k: wide(v) for k, v in d.items()}
    x = w["x"]
    vec = lambda k, missing: per_row(w[k], x) if k in w else torch.full_like(x[..., :1], missing)  # noqa: E731
    if form != "before":
        y, y_off, y_rstd = w["branch"], torch.zeros_like(w["branch"]), None
        if branch_kind:
            y, y_off, y_rstd = normed(y, branch_kind, eps)
        bw, bb, gate = vec("branch_weight", 1.0), vec("branch_bias", 0.0), s * vec("gate", 1.0)
        t = y * bw + bb
        t_off = bw.abs() * y_off + 3 * U * ((y * bw).abs() + bb.abs())
        want = x + gate * t
        near("r", r, want, gate.abs() * t_off + 3 * U * (gate * t).abs() + U * want.abs())
        base = wide(r)
    else:
        base = x
    if form != "after":
        h, h_off, rstd = normed(base, kind, eps)
        lift = 1 + vec("scale", 0.0)
        a, o = vec("weight", 1.0) * lift, vec("bias", 0.0) * lift + vec("shift", 0.0)
        parts = (vec("bias", 0.0) * lift).abs() + vec("shift", 0.0).abs()
        want = h * a + o
        near("z", z, want, a.abs() * h_off + 5 * U * ((h * a).abs() + parts))
    if grads is None:
        return
    dr, dz = (wide(u) for u in ups)
    rows = tuple(range(x.dim() - 1))
    total = torch.zeros_like(x) if dr is None else dr
    total_off = torch.zeros_like(x)

    def vector(name, terms, off):
        """Sums over the rows that share a vector's numbers."""
        if name not in grads:
            return
        over = rows[1:] if d[name].dim() == 2 else rows
        n = min(x.numel() // x.shape[-1], 256) + 16
        want = terms.sum(over) if over else terms
        off = n * U * terms.abs() + off
        near(name, grads[name], want, off.sum(over) if over else off)

    if dz is not None and form != "after":
        pre = h * vec("weight", 1.0) + vec("bias", 0.0)
        vector("shift", dz, torch.zeros_like(dz))
        vector("scale", dz * pre, dz.abs() * (h_off * vec("weight", 1.0).abs() + 4 * U * (pre.abs() + vec("bias", 0.0).abs())))
        vector("weight", dz * lift * h, (dz * lift).abs() * (h_off + 4 * U * h.abs()))
        vector("bias", dz * lift, 4 * U * (dz * lift).abs())
        e, e_off = normed_grad(dz * a, 4 * U * (dz * a).abs(), h, h_off, rstd, kind)
        total = total + e
        total_off = e_off + 2 * U * total.abs()
    near("x", grads["x"], total, total_off)
    if form == "before":
        return
    vector("gate", s * total * t, (s * t).abs() * total_off + abs(s) * total.abs() * (t_off + 4 * U * (t.abs() + bb.abs())))
    vector("branch_weight", gate * total * y, (gate * y).abs() * total_off + (gate * total).abs() * (y_off + 4 * U * y.abs()))
    vector("branch_bias", gate * total, gate.abs() * total_off + 4 * U * (gate * total).abs())
    e, e_off = total * gate * bw, (gate * bw).abs() * total_off + 4 * U * (total * gate * bw).abs()
    if branch_kind:
        e, e_off = normed_grad(e, e_off, y, y_off, y_rstd, branch_kind)
    near("branch", grads["branch"], e, e_off)


def run(d, form, train=True, ups="both", seed=9, out_dtype=None, **kw):
    """Forward, and backward for random gradients of r and z ("both", "r" or "z" alone)."""
    if train:
        for t in d.values():
            t.requires_grad_(True)
    r, z = call(d, form, out_dtype=out_dtype, **kw)
    if not train:
        check(d, form, r, z, **kw)
        return r, z
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda t: torch.randn(t.shape, generator=g, device="cuda").to(t.dtype)  # noqa: E731
    dr = rand(r) if r is not None and ups != "z" else None
    dz = rand(z) if z is not None and ups != "r" else None
    outs = [(o, u) for o, u in ((r, dr), (z, dz)) if u is not None]
    names = list(d)
    got = torch.autograd.grad([o for o, _ in outs], [d[k] for k in names], [u for _, u in outs])
    grads = dict(zip(names, got))
    for k in names:
        assert grads[k].dtype == d[k].dtype and grads[k].shape == d[k].shape
    check(d, form, r, z, ups=(dr, dz), grads=grads, **kw)
    return r, z, grads


KINDS = [("rms", None, "none", False), ("layer", "rms", "channel", True), ("rms", "layer", "sample", False),
         ("layer", "layer", "none", True), ("layer", None, "sample", True)]


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both(shape, types):
    for kind, branch_kind, gate, mod in KINDS:
        d = make(*shape, *types, gate, branch_kind, kind, mod)
        run(d, "both", kind=kind, branch_kind=branch_kind, s=0.7)


@pytest.mark.parametrize("shape", SHAPES[::3], ids=str)
def test_forward_alone(shape):
    """Without gradients: the same bits as with them."""
    for (kind, branch_kind, gate, mod), types in zip(KINDS, TYPES):
        d = make(*shape, *types, gate, branch_kind, kind, mod)
        kw = dict(kind=kind, branch_kind=branch_kind, s=-1.5)
        r, z = run(d, "both", train=False, **kw)
        r2, z2, _ = run(d, "both", **kw)
        assert torch.equal(r, r2) and torch.equal(z, z2)


@pytest.mark.parametrize("shape", SHAPES[::2], ids=str)
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_before(shape, kind):
    for types in TYPES:
        for mod in (False, True):
            d = make(*shape, *types, kind=kind, mod=mod, form="before")
            run(d, "before", kind=kind, out_dtype=types[1])


@pytest.mark.parametrize("shape", SHAPES[1::2], ids=str)
@pytest.mark.parametrize("branch_kind", [None, "rms", "layer"])
def test_after(shape, branch_kind):
    for types, gate in zip(TYPES, ("none", "channel", "sample", "channel", "sample")):
        run(make(*shape, *types, gate, branch_kind, form="after"), "after", branch_kind=branch_kind, s=0.5)


@pytest.mark.parametrize("ups", ["r", "z"])
def test_one_gradient(ups):
    """r or z alone is used: the other's gradient counts as zero."""
    for kind, branch_kind, gate, mod in KINDS:
        d = make(2, 33, 200, F32, BF16, gate, branch_kind, kind, mod)
        keep = [k for k in d if ups == "z" or k not in ("weight", "bias", "scale", "shift")]
        for t in d.values():
            t.requires_grad_(True)
        r, z = call(d, "both", kind, branch_kind)
        out = r if ups == "r" else z
        up = torch.randn_like(out)
        got = torch.autograd.grad(out, list(d.values()), up, retain_graph=True, allow_unused=True)
        grads = dict(zip(d, got))
        for k in d:
            if k not in keep:
                assert not grads.pop(k).any()
        check(d, "both", r, z, kind, branch_kind, ups=(up, None) if ups == "r" else (None, up), grads=grads)


def test_vector_types():
    """Vectors of other types than the rows'."""
    for wt, types in itertools.product((F32, F16, BF16), TYPES):
        for c in (48, 1000, 1001):
            run(make(2, 5, c, *types, "sample", "layer", "layer", True, wt=wt), "both", kind="layer", branch_kind="layer")


def test_each_gradient_alone():
    """Any one input may be the only one that asks for its gradient."""
    for c in (72, 600):
        kw = dict(kind="layer", branch_kind="layer", s=0.7)
        d = make(3, 20, c, F32, BF16, "sample", "layer", "layer", True)
        r, z, grads = run(d, "both", **kw)
        ups = [torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") for t in (r,)]
        g = torch.Generator(device="cuda").manual_seed(9)
        ups = [torch.randn(t.shape, generator=g, device="cuda").to(t.dtype) for t in (r, z)]
        for k in d:
            one = {n: t.detach().requires_grad_(n == k) for n, t in d.items()}
            (got,) = torch.autograd.grad(call(one, "both", **kw), [one[k]], ups)
            assert torch.equal(got, grads[k]), k


def test_row_values():
    """Rows of equal numbers, of zeros, of one large number, and of magnitudes whose squares leave FP32's range."""
    for xt, c in itertools.product((F32, BF16), (24, 600, 1003)):
        x = torch.randn(7, c, generator=torch.Generator().manual_seed(c))
        x[0] = 3.25
        x[1] = 0.0
        x[2, c // 2] = 1e4
        x[3] *= 1e25
        x[4] *= 1e-25
        x[5] = x[5] * 1e-3 + 1e3
        x = x.to(xt).cuda()
        for kind, eps in itertools.product(("rms", "layer"), (1e-6, 1e-38)):
            z = fb.block_norm(x, kind=kind, eps=eps)
            h, off, _ = normed(x.double(), kind, torch.tensor(eps).double().item())
            rows = [0, 2, 3, 5, 6] + ([4] if eps == 1e-6 else [])
            if kind == "layer":
                assert not z[0].any()
            assert not z[1].any()
            near("z", z[rows], h[rows], off[rows] + 2 * U * h[rows].abs())
            if eps == 1e-38:  # (the rows' mean square is 1e-50: eps is all there is)
                near("z", z[4:5], h[4:5], off[4:5] + 8 * U * h[4:5].abs())


def test_not_finite():
    """An infinite or NaN number spoils its own row alone."""
    for c in (16, 80, 700, 1001):
        for kind in ("rms", "layer"):
            d = make(1, 9, c, F32, F32, "channel", kind, kind)
            clean = call(d, "both", kind, kind)
            for row, v in ((2, float("inf")), (5, float("nan"))):
                for k in ("x", "branch"):
                    e = {n: t.clone() for n, t in d.items()}
                    e[k][0, row, c // 2] = v
                    for a, b in zip(call(e, "both", kind, kind), clean):
                        keep = [i for i in range(9) if i != row]
                        assert torch.equal(a[0, keep], b[0, keep])
                        assert a[0, row].isnan().any() or a[0, row].isinf().any()


def test_zero_eps():
    x = torch.randn(3, 50, device="cuda") * 1e-18
    z = fb.block_norm(x, eps=0.0)
    h, off, _ = normed(x.double(), "rms", 0.0)
    near("z", z, h, off + 2 * U * h.abs())


def test_strides_and_lazy_views():
    """Rows with gaps, permuted images, negated views and expanded gradients."""
    wide_x = torch.randn(4, 6, 96, device="cuda")
    image = torch.randn(2, 40, 5, 7, device="cuda").to(memory_format=torch.channels_last)
    neg = torch.randn(3, 4, 24, device="cuda", dtype=torch.complex64).conj().imag
    for x in (wide_x[:, :, ::2], wide_x[:, ::2], wide_x.transpose(0, 1), image.permute(0, 2, 3, 1), neg,
              torch.randn(1, 1, 32, device="cuda").expand(3, 5, 32), wide_x[0, 0]):
        c = x.shape[-1]
        w = torch.randn(2 * c, device="cuda")[::2]
        got = fb.block_norm(x, w, kind="layer")
        h, off, _ = normed(x.resolve_neg().double(), "layer", EPS)
        near("z", got, h * w.double(), off * w.abs().double() + 2 * U * (h * w.double()).abs())
    leaf = wide_x.clone().requires_grad_(True)
    z = fb.block_norm(leaf[:, :, 1::2], kind="rms")
    z.sum().backward()  # an expanded gradient
    d = {"x": leaf.detach()[:, :, 1::2]}
    check(d, "before", None, z, ups=(None, torch.ones_like(z)), grads={"x": leaf.grad[:, :, 1::2]})
    assert not leaf.grad[:, :, ::2].any()


def test_unaligned_memory():
    """Rows and vectors that begin at no vector's boundary."""
    for c in (64, 520):
        flat = torch.randn(4 * c * 6 + 9, device="cuda", dtype=BF16)
        for at in (1, 3, 8):
            x, y = flat[at:at + 6 * c].view(2, 3, c), flat[6 * c + at:12 * c + at].view(2, 3, c)
            w = torch.randn(c + 1, device="cuda")[1:]
            d = {"x": x.clone(), "branch": y.clone(), "weight": w, "gate": w}
            a = fb.gated_residual_norm(x, y, w, w, kind="layer")
            b = fb.gated_residual_norm(d["x"], d["branch"], w.clone(), w.clone(), kind="layer")
            check(d, "both", *a, kind="layer")
            check(d, "both", *b, kind="layer")


@pytest.mark.parametrize("types", TYPES, ids=str)
@pytest.mark.parametrize("c", [4095, 4099, 6143, 6145, 8191, 8193, 12289, 16381])
def test_long_rows_of_no_whole_vectors(c, types):
    d = make(2, 3, c, *types, gate="sample", branch_kind="layer", kind="layer", mod=True, seed=c)
    run(d, "both", kind="layer", branch_kind="layer")
    d = make(2, 3, c, *types, gate="channel", kind="rms", seed=c)
    run(d, "both", kind="rms")
    d = make(1, 5, c, *types, form="before", kind="rms", seed=c)
    run(d, "before", kind="rms", out_dtype=types[1])


def test_module():
    for kind in ("rms", "layer"):
        m = fb.BlockNorm(80, kind).cuda()
        torch.nn.init.normal_(m.weight)
        x, t = torch.randn(2, 5, 80, device="cuda"), torch.randn(2, 80, device="cuda")
        assert torch.equal(m(x, t, t), fb.block_norm(x, m.weight, m.bias, scale=t, shift=t, kind=kind))
        assert m(x, out_dtype=BF16).dtype == BF16


def test_shapes():
    for shape in ((48,), (5, 48), (2, 3, 48), (2, 3, 4, 48), (2, 1, 3, 2, 48)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        y = torch.randn(shape, device="cuda", requires_grad=True)
        gate = torch.randn((shape[0], 48) if len(shape) > 1 else (48,), device="cuda", requires_grad=True)
        d = {"x": x, "branch": y, "gate": gate}
        run(d, "both", kind="layer", branch_kind="rms")


def test_empty():
    for shape in ((0, 4, 16), (3, 0, 16), (0, 600)):
        x, y = (torch.zeros(shape, device="cuda", requires_grad=True) for _ in range(2))
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        gate = torch.ones(shape[0], shape[-1], device="cuda", requires_grad=True)
        r, z = fb.gated_residual_norm(x, y, gate, w, branch_kind="rms", branch_weight=w)
        assert r.shape == z.shape == shape
        (r.sum() + z.sum()).backward()
        for t in (x, y, w, gate):
            assert t.grad.shape == t.shape and not t.grad.any()


def test_large_rows_in_fp64():
    """Sums over many rows: n in the tolerance stays at 256 rows."""
    d = make(2, 40_000, 24, F32, F32, "channel", "layer", "layer", True)
    run(d, "both", kind="layer", branch_kind="layer")


@pytest.mark.parametrize("shape", [(300, 2, 72), (700, 1, 1000), (1025, 3, 33), (64, 40, 24), (129, 1, 520)], ids=str)
def test_many_samples(shape):
    """More samples than a CTA of the vectors' sums takes: vectors for each beside shared ones."""
    for kind, branch_kind, gate, mod in KINDS:
        d = make(*shape, F32, F32, gate, branch_kind, kind, mod)
        run(d, "both", kind=kind, branch_kind=branch_kind, s=0.7)
    x = torch.randn(shape[0], shape[2], device="cuda", requires_grad=True)  # a row for each sample
    d = {"x": x, "branch": torch.randn_like(x, requires_grad=True),
         "gate": torch.randn_like(x, requires_grad=True), "weight": torch.randn(shape[2], device="cuda", requires_grad=True)}
    run(d, "both", kind="layer", branch_kind="rms")


def test_aliased_results_of_the_c_entry_point():
    """r in x's place and z in branch's, dx in dr's and dbranch in dz's: as in memory of their own."""
    import ctypes

    from tests import test_block_norm_cpu as c

    lib = ctypes.CDLL(c.LIB)
    lib.fssim_block_norm_backward_workspace_bytes.restype = ctypes.c_size_t
    for f in (lib.fssim_block_norm_forward, lib.fssim_block_norm_backward):
        f.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    for rows, cols in ((700, 96), (90, 1001), (60, 2048), (311, 4101), (160, 7001), (11, 9001)):
        x, y, dr, dz = (torch.randn(rows, cols, device="cuda") for _ in range(4))
        results = []
        for alias in (False, True):
            t = [v.clone() for v in (x, y, dr, dz)]
            r, z, dx, dy = t if alias else [torch.empty_like(v) for v in t]
            stats, after = (torch.empty(rows, 2, device="cuda") for _ in range(2))
            a = c.ForwardArgs(kind=2, branch_kind=2, B=1, T=rows, C=cols, eps=1e-6, residual_scale=0.5, x=t[0].data_ptr(),
                              branch=t[1].data_ptr(), r=r.data_ptr(), z=z.data_ptr(), stats=stats.data_ptr(),
                              branch_stats=after.data_ptr())
            stream = torch.cuda.current_stream().cuda_stream
            assert lib.fssim_block_norm_forward(ctypes.byref(a), stream) == 0
            out = [r.clone(), z.clone()]
            weight = torch.empty(cols, device="cuda")
            b = c.BackwardArgs(kind=2, branch_kind=2, B=1, T=rows, C=cols, residual_scale=0.5, r=r.data_ptr(),
                               branch=y.data_ptr(), dr=t[2].data_ptr(), dz=t[3].data_ptr(), stats=stats.data_ptr(),
                               branch_stats=after.data_ptr(), dx=dx.data_ptr(), dbranch=dy.data_ptr(),
                               dweight=c.Channels(weight.data_ptr(), 0, 0))
            size = lib.fssim_block_norm_backward_workspace_bytes(ctypes.byref(b))
            ws = torch.empty(size, dtype=torch.uint8, device="cuda")
            b.workspace, b.workspace_bytes = ws.data_ptr(), size
            assert lib.fssim_block_norm_backward(ctypes.byref(b), stream) == 0
            torch.cuda.synchronize()
            results.append(out + [dx.clone(), dy.clone(), weight])
        assert all(torch.equal(p, q) for p, q in zip(*results))


def test_shared_vectors_and_twice_the_same():
    """One weight for both norms, and the same tensor as x and branch: gradients add up."""
    x = torch.randn(3, 5, 80, device="cuda", dtype=torch.float32, requires_grad=True)
    w = torch.randn(80, device="cuda", requires_grad=True)
    r, z = fb.gated_residual_norm(x, x, w, w, branch_kind="rms", branch_weight=w)
    up = torch.randn_like(r)
    got = torch.autograd.grad((r, z), (x, w), (up, up))
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    h = lambda v: v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt()  # noqa: E731
    rd = xd + wd * (h(xd) * wd)
    want = torch.autograd.grad((rd, h(rd) * wd), (xd, wd), (up.double(), up.double()))
    for g, t in zip(got, want):
        # sums of a few terms of their own size, each within some 100 u
        assert (g.double() - t).abs().max() <= 1e-5 * t.abs().max()


def test_differences():
    """Gradients against differences of the kernel's own results."""
    d = make(2, 3, 40, F32, F32, "sample", "layer", "layer", True, seed=4)
    kw = dict(kind="layer", branch_kind="layer", s=0.7)
    up = [torch.randn(2, 3, 40, device="cuda") for _ in range(2)]
    loss = lambda e: sum((o.double() * u).sum() for o, u in zip(call(e, "both", **kw), up))  # noqa: E731
    for t in d.values():
        t.requires_grad_(True)
    grads = torch.autograd.grad(call(d, "both", **kw), list(d.values()), up)
    h = 2.0 ** -7
    for (k, t), g in zip(d.items(), grads):
        way = torch.randn(t.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        way /= way.norm()
        with torch.no_grad():
            plus, minus = (loss({n: v + sign * h * way if n == k else v for n, v in d.items()}) for sign in (1, -1))
        slope = ((plus - minus) / (2 * h)).item()
        exact = (g.double() * way).sum().item()
        # the cubic term of functions whose scale is 1 (h^2 times it), and rounding of 240 terms / h
        assert abs(slope - exact) <= 20 * h * h * max(1.0, g.norm().item())


def test_refuses_second_derivatives():
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    z = fb.block_norm(x)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(z.sum(), x, create_graph=True)


def test_graph():
    """Forward and backward captured, replayed on new numbers, and two graphs replayed side by side."""
    kw = dict(kind="layer", branch_kind="rms", s=0.7)
    sets = [make(2, 500, 320, F32, BF16, "sample", "rms", "layer", True, seed=i) for i in (1, 2)]
    graphs, results = [], []
    for d in sets:
        for t in d.values():
            t.requires_grad_(True)
        up = (torch.randn(2, 500, 320, device="cuda"), torch.randn(2, 500, 320, device="cuda", dtype=BF16))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = call(d, "both", **kw)
            grads = torch.autograd.grad(outs, list(d.values()), up)
            outs = [o.detach() for o in outs]
        graphs.append(graph)
        results.append((outs, grads, up))
    for d in sets:
        with torch.no_grad():
            for t in d.values():
                t.mul_(0.9)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for d, (outs, grads, up) in zip(sets, results):
        check(d, "both", *outs, ups=up, grads=dict(zip(d, grads)), **kw)


def test_repeats_and_streams():
    d = make(4, 300, 1152, F32, BF16, "sample", "layer", "layer", True)
    kw = dict(kind="layer", branch_kind="layer")
    a = run(d, "both", **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run(d, "both", **kw)
    side.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert all(torch.equal(a[2][k], b[2][k]) for k in d)

"""group_norm_act against its definition in 64 bits: values, gradients, layouts, edge cases.

Tolerances. u = 2^-24. A group's mean is off by at most about 16 u max|x| (sums of eight,
then averages of means), 1/std by as much relatively, so the value before the activation by
    tz = 32 u (max|x| rstd |w| + |xhat w| + |b|).
SiLU and ReLU have slopes below 1.1 and SiLU a second derivative below 0.5; the logistic
function is right to 2^-20 for 16-bit tensors and to 8 u for 32-bit ones. One rounding of the
result adds half a step, finfo.eps / 2 relative.
"""

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t, ref):
    """Half a step of type t at ref (its subnormals' half step at least)."""
    f = torch.finfo(t)
    return (ref.abs() * (f.eps / 2)).clamp_min(f.smallest_normal * f.eps / 2)


def sigmoid_error(dtype):
    return 8 * U if dtype == F32 else 2.0 ** -20


def plain(x, groups, w, b, eps, act, dy=None):
    """Definition in float64 on float64 copies: (y, xhat, z, rstd), and the gradients."""
    n, c, h, wd = x.shape
    v = x.double().reshape(n, groups, -1)
    m = v.shape[2]
    mean = v.mean(2, keepdim=True)
    var = ((v - mean) ** 2).mean(2, keepdim=True)
    rstd = (var + eps) ** -0.5
    xhat = ((v - mean) * rstd).reshape(x.shape)
    wc = (torch.ones(c, device=x.device) if w is None else w).double().view(1, c, 1, 1)
    bc = (torch.zeros(c, device=x.device) if b is None else b).double().view(1, c, 1, 1)
    z = xhat * wc + bc
    s = torch.sigmoid(z)
    y = {"silu": z * s, "relu": torch.where(z < 0, torch.zeros_like(z), z), None: z}[act]
    rs = rstd.expand(-1, -1, c // groups).reshape(n, c, 1, 1)
    if dy is None:
        return y, xhat, z, rs
    slope = {"silu": s * (1 + z * (1 - s)), "relu": (z > 0).double(), None: torch.ones_like(z)}[act]
    dz = dy.double() * slope
    g = (dz * wc).reshape(n, groups, -1)
    xh = xhat.reshape(n, groups, -1)
    dx = rstd * (g - g.sum(2, keepdim=True) / m - xh * ((g * xh).sum(2, keepdim=True) / m))
    return y, xhat, z, rs, dz, dx.reshape(x.shape), (dz * xhat).sum((0, 2, 3)), dz.sum((0, 2, 3))


def z_tolerance(x, xhat, rs, w, b):
    c = x.shape[1]
    wc = 1.0 if w is None else w.double().abs().view(1, c, 1, 1)
    bc = 0.0 if b is None else b.double().abs().view(1, c, 1, 1)
    return 32 * U * (x.double().abs().max() * rs * wc + xhat.abs() * wc + bc)


def check_forward(y, x, groups, w, b, eps, act):
    ref, xhat, z, rs = plain(x, groups, w, b, eps, act)
    tol = 1.1 * z_tolerance(x, xhat, rs, w, b) + sigmoid_error(x.dtype) * ref.abs() + \
        half_step(x.dtype, ref)
    assert y.dtype == x.dtype and y.shape == x.shape
    worst = ((y.double() - ref).abs() / tol).max().item() if ref.numel() else 0.0
    assert worst <= 1.0, f"y is off by {worst:.2f} tolerances"


def check_backward(dx, dw, db, x, groups, w, b, eps, act, dy):
    ref, xhat, z, rs, dz, rdx, rdw, rdb = plain(x, groups, w, b, eps, act, dy)
    n, c = x.shape[:2]
    tz = z_tolerance(x, xhat, rs, w, b)
    dmax = dy.double().abs()
    # ReLU's slope jumps where z is within tz of zero: those pixels are left out of dx, and
    # their dy is an allowance in the sums
    edge = (z.abs() <= tz) if act == "relu" else torch.zeros_like(z, dtype=torch.bool)
    tdz = dmax * (0.5 * tz + sigmoid_error(x.dtype) * 4 + 4 * U) + edge * dmax
    # sums of P*N terms, threads of a few dozen terms each: 128 u of the sum of magnitudes
    txhat = tz / (1.0 if w is None else w.double().abs().view(1, c, 1, 1).clamp_min(1e-3))
    wdt = F32 if w is None else w.dtype
    if db is not None:
        tol = (tdz + 128 * U * dz.abs()).sum((0, 2, 3)) + half_step(wdt, rdb)
        assert db.dtype == wdt and ((db.double() - rdb).abs() / tol).max().item() <= 1.0
    if dw is not None:
        t = tdz * xhat.abs() + dz.abs() * txhat + 128 * U * (dz * xhat).abs()
        tol = t.sum((0, 2, 3)) + half_step(wdt, rdw)
        assert dw.dtype == wdt and ((dw.double() - rdw).abs() / tol).max().item() <= 1.0
    if dx is not None:
        wc = 1.0 if w is None else w.double().abs().view(1, c, 1, 1)

        def mean(t):
            return t.reshape(n, groups, -1).mean(2, keepdim=True).expand(
                -1, -1, t[0].numel() // groups).reshape(t.shape)

        g, tg = dz.abs() * wc, tdz * wc
        tol = rs * (tg + mean(tg) + xhat.abs() * mean(tg * xhat.abs() + g * txhat) +
                    txhat * mean(g * xhat.abs()) +
                    128 * U * (g + mean(g) + xhat.abs() * mean(g * xhat.abs()))) + \
            64 * U * rdx.abs() + half_step(x.dtype, rdx)
        assert dx.dtype == x.dtype
        off = ((dx.double() - rdx).abs() / tol).masked_fill(edge, 0.0).max().item()
        assert off <= 1.0, f"dx is off by {off:.2f} tolerances"


def make(shape, dtype, wdtype, seed, centre=1.0):
    g = torch.Generator().manual_seed(seed)
    n, c, h, w = shape
    x = torch.randn(n, h, w, c, generator=g) * (0.5 + torch.rand(c, generator=g)) + \
        centre * torch.randn(c, generator=g)
    dy = torch.randn(n, h, w, c, generator=g)
    weight = 1 + 0.3 * torch.randn(c, generator=g)
    bias = 0.3 * torch.randn(c, generator=g)
    return (x.to(dtype).cuda().permute(0, 3, 1, 2), dy.to(dtype).cuda().permute(0, 3, 1, 2),
            weight.to(wdtype).cuda(), bias.to(wdtype).cuda())


def grads(x, groups, w, b, eps, act, dy):
    ins = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    it = iter(ins)
    xs, ws, bs = (next(it) if t is not None else None for t in (x, w, b))
    y = fb.group_norm_act(xs, groups, ws, bs, eps=eps, activation=act)
    got = iter(torch.autograd.grad(y, ins, dy))
    return (y.detach(), next(got), next(got) if w is not None else None,
            next(got) if b is not None else None)


SHAPES = [  # (N, C, H, W), groups
    ((1, 1, 1, 1), 1),          # one number: y = act(bias)
    ((2, 3, 1, 1), 3),          # groups of one number
    ((1, 8, 1, 1), 2),
    ((2, 6, 5, 7), 2),          # two channels a vector in 16 bits, one in 32
    ((3, 30, 9, 11), 10),
    ((1, 5, 40, 40), 1),        # odd channels
    ((1, 32, 17, 3), 4),
    ((2, 64, 33, 31), 32),
    ((1, 320, 13, 9), 32),      # groups of ten: vectors across groups
    ((5, 16, 64, 64), 16),      # groups of one channel
    ((1, 2056, 3, 5), 8),       # more channels than one CTA's threads take: two slices
    ((1, 1283, 4, 3), 1),       # one group over several slices, one channel a vector
    ((1, 4096, 2, 2), 4096),
    ((700, 8, 3, 3), 4),        # many samples
    ((1, 16, 300, 301), 4),     # many parts
    ((1, 128, 1, 1000), 32),
    # larger: two passes over tiles and parts, their last ones short
    ((2, 320, 67, 121), 32),
    ((1, 48, 130, 199), 16),    # groups of three
    ((3, 2056, 20, 21), 8),     # two slices
    ((1, 1283, 40, 30), 1),     # a group over six slices
    ((1, 12, 300, 251), 3),
    ((40, 64, 40, 41), 8),
    ((600, 32, 20, 20), 4),     # more samples than a wave of CTAs
    ((1, 1024, 9, 8), 32),
    ((2, 1, 40, 41), 1),        # one channel
    ((1, 1, 300, 301), 1),
    ((1, 65537, 2, 1), 1),      # 257 slices, the last of one channel
    ((1, 40003, 1, 3), 40003),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_values_and_gradients(case, dtype):
    shape, groups = SHAPES[case]
    act = ["silu", None, "relu"][case % 3]
    x, dy, w, b = make(shape, dtype, F32 if case % 2 else dtype, 100 + case)
    y, dx, dw, db = grads(x, groups, w, b, 1e-5, act, dy)
    check_forward(y, x, groups, w, b, 1e-5, act)
    check_backward(dx, dw, db, x, groups, w, b, 1e-5, act, dy)
    assert y.is_contiguous(memory_format=torch.channels_last)
    with torch.no_grad():  # the inference call gives the same bits
        assert torch.equal(fb.group_norm_act(x, groups, w, b, 1e-5, act), y)


# Channels that are no whole vectors: pixels taken together where the samples allow it.
SPANS = [
    ((1, 1, 1, 8), 1),          # one vector in all
    ((1, 3, 2, 4), 1),
    ((1, 3, 2, 4), 3),
    ((2, 3, 2, 2), 1),          # four pixels: 16 bytes in 32 bits only
    ((2, 3, 3, 2), 3),          # two pixels: 4 bytes in 16 bits, elements in 32
    ((2, 3, 3, 3), 1),          # nine: elements in all types
    ((3, 6, 7, 4), 2),
    ((1, 5, 16, 33), 5),
    ((2, 20, 24, 31), 4),
    ((4, 7, 64, 72), 1),
    ((1, 1, 400, 401), 1),      # many parts
    ((1, 3, 304, 301), 3),
    ((300, 3, 20, 20), 1),      # more samples than a wave of CTAs
    ((900, 6, 8, 9), 3),
    ((2, 30, 120, 121), 10),
    ((2, 255, 8, 13), 5),       # most channels of a span
    ((1, 257, 8, 13), 1),       # one too many
    ((1, 2046, 8, 8), 11),
    ((3, 514, 16, 12), 514),    # more groups than an applying pass merges itself
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(SPANS)))
def test_channels_off_the_vector(case, dtype):
    shape, groups = SPANS[case]
    act = ["silu", "relu", None][case % 3]
    x, dy, w, b = make(shape, dtype, dtype if case % 2 else F32, 300 + case)
    for ws, bs in ((w, b), (None, None)):
        y, dx, dw, db = grads(x, groups, ws, bs, 1e-5, act, dy)
        check_forward(y, x, groups, ws, bs, 1e-5, act)
        check_backward(dx, dw, db, x, groups, ws, bs, 1e-5, act, dy)
    with torch.no_grad():
        assert torch.equal(fb.group_norm_act(x, groups, None, None, 1e-5, act), y)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_channels_off_the_vector_at_any_address(offset, dtype):
    shape, groups = (2, 3, 40, 48), 3
    x, dy, w, b = make(shape, dtype, F32, 340)
    n, c, h, wd = shape
    moved = torch.zeros(x.numel() + offset, dtype=dtype, device="cuda")[offset:].view(n, h, wd, c).permute(0, 3, 1, 2)
    moved.copy_(x)
    y, dx, dw, db = grads(moved, groups, w, b, 1e-5, "silu", dy)
    check_forward(y, x, groups, w, b, 1e-5, "silu")
    check_backward(dx, dw, db, x, groups, w, b, 1e-5, "silu", dy)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", ["silu", "relu", None])
def test_activations_and_missing_parameters(act, dtype):
    x, dy, w, b = make((2, 24, 19, 23), dtype, F32, 5)
    for ws, bs in ((w, b), (None, b), (w, None), (None, None)):
        y, dx, dw, db = grads(x, 6, ws, bs, 1e-6, act, dy)
        check_forward(y, x, 6, ws, bs, 1e-6, act)
        check_backward(dx, dw, db, x, 6, ws, bs, 1e-6, act, dy)


@pytest.mark.parametrize("wdtype", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_parameter_types(dtype, wdtype):
    x, dy, w, b = make((2, 16, 12, 15), dtype, wdtype, 6)
    y, dx, dw, db = grads(x, 4, w, b, 1e-5, "silu", dy)
    check_forward(y, x, 4, w, b, 1e-5, "silu")
    check_backward(dx, dw, db, x, 4, w, b, 1e-5, "silu", dy)


@pytest.mark.parametrize("shape", [(2, 16, 12, 15), (1, 16, 12, 15), (2, 16, 200, 201), (1, 16, 300, 301)])
def test_only_the_gradients_asked_for(shape):
    x, dy, w, b = make(shape, F32, F32, 7)
    full = grads(x, 4, w, b, 1e-5, "silu", dy)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        ts = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), need)]
        y = fb.group_norm_act(ts[0], 4, ts[1], ts[2])
        got = iter(torch.autograd.grad(y, [t for t, k in zip(ts, need) if k], dy))
        for k, ref in zip(need, full[1:]):
            if k:
                assert torch.equal(next(got), ref)


def test_gradient_against_differences():
    x, dy, w, b = make((2, 12, 7, 9), F32, F32, 8)
    _, dx, dw, db = grads(x, 3, w, b, 1e-5, "silu", dy)
    g = torch.Generator().manual_seed(1)

    def loss(x, w, b):
        return (plain(x, 3, w, b, 1e-5, "silu")[0] * dy.double()).sum()

    h = 1e-4
    for i, (t, got) in enumerate(((x, dx), (w, dw), (b, db))):
        d = torch.randn(t.shape, generator=g).double().cuda()
        ts = [x.double(), w.double(), b.double()]
        hi, lo = list(ts), list(ts)
        hi[i], lo[i] = ts[i] + h * d, ts[i] - h * d
        want = (loss(*hi) - loss(*lo)) / (2 * h)
        # truncation h^2, and 128 u of the gradient's magnitudes
        tol = 1e-4 * want.abs() + 1e-5 * (got.double().abs() * d.abs()).sum()
        assert ((got.double() * d).sum() - want).abs() <= tol


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layouts(dtype):
    x, dy, w, b = make((3, 24, 10, 14), dtype, F32, 9)
    want = grads(x, 6, w, b, 1e-5, "silu", dy)
    wide = torch.zeros(3, 48, 20, 14, dtype=dtype, device="cuda")
    wide[:, ::2, 5:15] = x
    forms = {
        "nchw": x.contiguous(),
        "strided": wide[:, ::2, 5:15],
        "transposed": x.transpose(2, 3).contiguous().transpose(2, 3),
    }
    # dense channels-last memory that starts off a 16-byte boundary
    for shift in (1, 2, 3):
        store = torch.zeros(x.numel() + shift, dtype=dtype, device="cuda")
        v = store[shift:].view(3, 10, 14, 24).permute(0, 3, 1, 2)
        v.copy_(x)
        forms[f"shift{shift}"] = v
    for name, form in forms.items():
        got = grads(form, 6, w, b, 1e-5, "silu", dy)
        check_forward(got[0], x, 6, w, b, 1e-5, "silu")
        check_backward(*got[1:], x, 6, w, b, 1e-5, "silu", dy)
        if not name.startswith("shift"):
            assert all(torch.equal(p, q) for p, q in zip(got, want)), name
    # gradients of the output in other layouts, a broadcast one among them
    got = grads(x, 6, w, b, 1e-5, "silu", dy.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ones = torch.ones((), dtype=dtype, device="cuda").expand(3, 24, 10, 14)
    got = grads(x, 6, w, b, 1e-5, "silu", ones)
    check_backward(*got[1:], x, 6, w, b, 1e-5, "silu", ones)
    # strided parameters
    ws, bs = torch.stack([w, b], 1).unbind(1)
    assert torch.equal(fb.group_norm_act(x, 6, ws, bs), want[0])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_constant_and_offset_inputs(dtype):
    # equal numbers have no deviation: y is act(bias), exactly up to its rounding
    x = torch.full((2, 12, 30, 31), 1000.25, dtype=dtype, device="cuda")
    _, dy, w, b = make((2, 12, 30, 31), dtype, F32, 10)
    y = fb.group_norm_act(x, 4, w, b, activation=None)
    assert torch.equal(y, b.to(dtype).view(1, 12, 1, 1).expand_as(y))
    _, dx, dw, db = grads(x, 4, w, b, 1e-5, None, dy)
    assert torch.equal(dw, torch.zeros_like(dw)) and torch.isfinite(dx).all()
    # a mean far above the spread
    x = (300.0 + torch.randn(2, 12, 30, 31, device="cuda")).to(dtype)
    got = grads(x, 4, w, b, 1e-5, "silu", dy)
    check_forward(got[0], x, 4, w, b, 1e-5, "silu")
    check_backward(*got[1:], x, 4, w, b, 1e-5, "silu", dy)
    # a border far from the rest
    x[:, :, 0] = 0
    check_forward(fb.group_norm_act(x, 4, w, b), x, 4, w, b, 1e-5, "silu")


@pytest.mark.parametrize("shape", [(2, 12, 8, 9), (2, 12, 300, 301), (9, 12, 130, 131)])
def test_nan_and_inf_stay_in_their_group(shape):
    x, dy, w, b = make(shape, F32, F32, 11)
    for act in ("silu", "relu", None):
        clean = grads(x, 4, w, b, 1e-5, act, dy)
        for bad in (float("nan"), float("inf")):
            xb = x.clone()
            xb[1, 4, 3, 3] = bad  # group 1 of sample 1: channels 3..5
            y, dx, dw, db = grads(xb, 4, w, b, 1e-5, act, dy)
            hit = torch.zeros_like(x, dtype=torch.bool)
            hit[1, 3:6] = True
            assert torch.equal(y[~hit], clean[0][~hit]) and torch.equal(dx[~hit], clean[1][~hit])
            assert y[hit].isnan().all() and dx[hit].isnan().all()
            assert dw[3:6].isnan().all() and dw[:3].isfinite().all() and dw[6:].isfinite().all()


def test_extreme_values():
    for dtype, top in ((F16, 6e4), (BF16, 1e18), (F32, 1e18)):
        x, dy, w, b = make((1, 8, 9, 10), dtype, F32, 12)
        x = (x.float() * (top / 16)).to(dtype)
        check_forward(fb.group_norm_act(x, 2, w, b), x, 2, w, b, 1e-5, "silu")
        x = (x.float() * 1e-30).to(dtype) if dtype != F16 else (x.float() * 1e-10).to(dtype)
        check_forward(fb.group_norm_act(x, 2, w, b), x, 2, w, b, 1e-5, "silu")
    # activations far out on both sides
    x, dy, w, b = make((1, 8, 9, 10), F32, F32, 13)
    y = fb.group_norm_act(x, 2, 1000 * w, b)
    assert y.isfinite().all()
    check_forward(y, x, 2, 1000 * w, b, 1e-5, "silu")


@pytest.mark.parametrize("shape", [(3, 24, 10, 14), (1, 64, 160, 161)])
def test_shared_parameters_accumulate(shape):
    # one layer used twice, and a broadcast gradient: what autograd adds up is each use's own
    x, dy, w, b = make(shape, F32, F32, 18)
    xs, ws, bs = (t.detach().requires_grad_(True) for t in (x, w, b))
    y1 = fb.group_norm_act(xs, 4, ws, bs)
    y2 = fb.group_norm_act(y1, 4, ws, bs)
    y2.sum().backward()
    ones = torch.ones_like(y2)
    _, d1, w2, b2 = grads(y1.detach(), 4, w, b, 1e-5, "silu", ones)
    _, dx, w1, b1 = grads(x, 4, w, b, 1e-5, "silu", d1)
    assert torch.equal(xs.grad, dx)
    assert torch.equal(ws.grad, w1 + w2) and torch.equal(bs.grad, b1 + b2)


def test_empty():
    w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda",
                                                                          requires_grad=True)
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        y = fb.group_norm_act(x, 2, w, b)
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert dx.shape == x.shape and not dw.any() and not db.any()


def test_refusals_on_the_gpu():
    x, dy, w, b = make((1, 8, 9, 10), F32, F32, 14)
    with pytest.raises(RuntimeError, match="x's device"):
        fb.group_norm_act(x, 2, w.cpu(), b)
    with pytest.raises(RuntimeError, match="CUDA device"):
        fb.group_norm_act(x.cpu(), 2)
    xs = x.detach().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(fb.group_norm_act(xs, 2, w, b).sum(), xs, create_graph=True)
    ws = w.detach().requires_grad_(True)
    y = fb.group_norm_act(x, 2, ws, b)
    with torch.no_grad():
        ws.mul_(2)  # the saved weight is no longer the forward's
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_autocast_leaves_the_types_alone():
    x, dy, w, b = make((1, 16, 20, 20), BF16, F32, 15)
    want = fb.group_norm_act(x, 4, w, b)
    with torch.autocast("cuda", dtype=torch.float16):
        got = fb.group_norm_act(x, 4, w, b)
    assert got.dtype == BF16 and torch.equal(got, want)


def test_module_matches_torch():
    torch.manual_seed(0)
    m = fb.GroupNormAct(8, 32, activation="silu").cuda()
    ref = torch.nn.GroupNorm(8, 32).cuda()
    with torch.no_grad():
        ref.weight.normal_()
        ref.bias.normal_()
    m.load_state_dict(ref.state_dict())
    x = torch.randn(2, 32, 21, 22, device="cuda")
    want = torch.nn.functional.silu(ref.double()(x.double()))
    assert (m(x).double() - want).abs().max().item() <= 64 * U * 8


def test_repeats_and_streams():
    x, dy, w, b = make((4, 64, 96, 96), BF16, F32, 16)
    want = grads(x, 16, w, b, 1e-5, "silu", dy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(4):
                results.append(grads(x, 16, w, b, 1e-5, "silu", dy))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_graphs_replay_together():
    shapes = [((2, 32, 40, 41), F32), ((1, 64, 128, 128), BF16)]
    graphs = []
    for k, (shape, dtype) in enumerate(shapes):
        x, dy, w, b = make(shape, dtype, F32, 20 + k)
        leaves = [t.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
                  for t in (x, w, b)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            y = fb.group_norm_act(leaves[0], 8, leaves[1], leaves[2])
            out = (y,) + torch.autograd.grad(y, leaves, dy)
        graphs.append((graph, torch.cuda.Stream(), leaves, dy, out, shape, dtype))
    for round_ in range(3):
        wants = []
        for graph, s, leaves, dy, out, shape, dtype in graphs:
            nx, ndy, nw, nb = make(shape, dtype, F32, 30 + round_)
            with torch.no_grad():
                for t, v in zip(leaves, (nx, nw, nb)):
                    t.copy_(v)
                dy.copy_(ndy)
            wants.append(grads(nx, 8, nw, nb, 1e-5, "silu", ndy))
        torch.cuda.synchronize()
        for _ in range(2):
            for graph, s, *_ in graphs:
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, out, _, _), want in zip(graphs, wants):
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_more_than_two_to_the_31_numbers():
    # 2 x 8 x 11600 x 11600 in 16 bits: 2.15e9 numbers, offsets beyond 32 bits
    n, c, h, w = 2, 8, 11600, 11600
    assert n * c * h * w > 2 ** 31
    x = torch.empty((n, h, w, c), dtype=BF16, device="cuda").permute(0, 3, 1, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in range(n):
        x[i].normal_(generator=g)
        x[i].mul_(1.0 + i)
    weight, bias = torch.rand(c, device="cuda"), torch.rand(c, device="cuda")
    xs = x.requires_grad_(True)
    y = fb.group_norm_act(xs, 4, weight, bias)
    dy = torch.ones((), dtype=BF16, device="cuda").expand_as(y)
    dx, = torch.autograd.grad(y, xs, dy)
    x = x.detach()
    for i in (0, n - 1):
        for k in (0, 3):
            part = x[i, 2 * k:2 * k + 2].float()
            mean = part.mean(dtype=torch.float64)
            std = (part - mean.float()).square_().mean(dtype=torch.float64).add(1e-5).sqrt()
            rows = slice(h - 3, h)
            z = (x[i, 2 * k:2 * k + 2, rows].double() - mean) / std * \
                weight[2 * k:2 * k + 2, None, None] + bias[2 * k:2 * k + 2, None, None]
            want = z * torch.sigmoid(z)
            # the mean of 2.7e8 numbers adds little to half a step
            tol = half_step(BF16, want) + 1e-4
            assert ((y[i, 2 * k:2 * k + 2, rows].double() - want).abs() <= tol).all()
    assert dx.isfinite().all()
    # dx of the last rows follows from the sums over everything: sum dx = 0 in each group
    total = dx[n - 1, 6:8].sum(dtype=torch.float64).abs()
    assert total <= 2.0 ** -9 * dx[n - 1, 6:8].abs().sum(dtype=torch.float64)


def test_a_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x, dy, w, b = make((1, 16, 20, 20), F32, F32, 17)
    want = grads(x, 4, w, b, 1e-5, "silu", dy)
    got = grads(*(t.to("cuda:1") if torch.is_tensor(t) else t for t in (x, 4, w, b, 1e-5, "silu", dy)))
    assert all(torch.equal(p.to("cuda:0"), q) for p, q in zip(got, want))


def test_c_entry_point_in_place():
    """The C call with y == x, a strided batch of two calls on one workspace, and mean and rstd."""
    import ctypes

    from .test_training_cpu import LIB, ForwardArgs

    lib = ctypes.CDLL(LIB)
    lib.fssim_group_norm_forward_workspace_bytes.restype = ctypes.c_size_t
    for shape in ((2, 32, 16, 16), (2, 32, 300, 301)):  # the resident kernel, and the passes
        x, _, w, b = make(shape, F16, F32, 50)
        want = fb.group_norm_act(x, 4, w, b)
        n, c, h, wd = shape
        _, xhat, _, rs = plain(x, 4, w, b, 1e-5, None)
        mean, rstd = torch.empty(2, 4, device="cuda"), torch.empty(2, 4, device="cuda")
        args = ForwardArgs(dtype=1, weight_dtype=0, activation=1, N=n, P=h * wd, C=c, groups=4,
                           eps=1e-5, x=x.data_ptr(), y=x.data_ptr(), weight=w.data_ptr(),
                           bias=b.data_ptr(), mean=mean.data_ptr(), rstd=rstd.data_ptr())
        size = lib.fssim_group_norm_forward_workspace_bytes(ctypes.byref(args))
        ws = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")  # contents arbitrary
        args.workspace, args.workspace_bytes = ws.data_ptr(), size
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        assert lib.fssim_group_norm_forward(ctypes.byref(args), stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(x, want)
        assert (ws[size:] == 255).all()
        ref = rs.view(2, 4, 8)[:, :, 0]
        assert ((rstd.double() - ref).abs() <= 32 * U * 8 * ref).all()

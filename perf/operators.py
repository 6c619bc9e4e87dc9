"""Measured cases of the training operators beside the image losses.

Two operators of a training step whose loss is this package's: the group normalisation with
its activation that the layers of an image network are made of (channels last, forward alone
and with its gradient), and the global gradient norm with clipping that follows the loss's
backward pass. Each is given in its plain form (elementary torch operations in 32 bits) and
as the calls that a user makes of ``fussim_b200``.

Norm cases: x is (n, c, h, w) in the channels-last memory format, normalised over the pixels
and channels of each of ``groups`` groups, scaled and shifted per channel, then activated;
``train`` adds the gradients of x, weight and bias for a given gradient of the output.

Clip cases: a list of gradient tensors, their 2-norm taken together, and each multiplied by
min(1, max_norm / (norm + 1e-6)). ``layout`` gives the tensors' shapes: "gaussians" are the
six parameter tensors of ``count`` splats (59 numbers each), "net" are ``count`` tensors of a
network, two short vectors after each long tensor, ``total`` numbers in the long ones.
``packed`` 0 gives each tensor its own memory; otherwise they are pieces of one flat buffer, as
data-parallel trainers keep them, each starting at a multiple of ``packed`` numbers. ``out`` says where the clipped gradients go: "same" (other buffers of the same type), "f32"
(32-bit buffers that an optimiser keeps) or "inplace".
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------
def _norm(name, train, dtype, n, c, h, w, groups, act, wdtype="f32"):
    return {"name": name, "op": "norm", "train": train, "dtype": dtype, "n": n, "c": c, "h": h,
            "w": w, "groups": groups, "act": act, "wdtype": wdtype}


def _clip(name, layout, dtype, count, total, active, out, packed=0):
    return {"name": name, "op": "clip", "layout": layout, "dtype": dtype, "count": count,
            "total": total, "active": active, "out": out, "packed": packed}


def listed():
    return [
        # the innermost level of a small network on one image: launch latency
        _norm("norm_fwd_16", False, "bf16", 1, 64, 16, 16, 8, "silu", "bf16"),
        # a decoder layer over one 256 x 256 image at inference
        _norm("norm_fwd_256", False, "bf16", 1, 128, 256, 256, 32, "silu"),
        # a full-resolution layer of an image enhancer on one 1080p frame
        _norm("norm_fwd_1080p", False, "f16", 1, 64, 1080, 1920, 16, "silu"),
        # a deep, narrow layer in training: many channels, few pixels
        _norm("norm_train_32", True, "bf16", 4, 512, 32, 32, 32, "silu"),
        # a middle layer of a 256 x 256 training batch
        _norm("norm_train_256", True, "bf16", 8, 128, 256, 256, 32, "silu"),
        # odd image sides and groups of ten channels, no activation (before an attention layer)
        _norm("norm_train_odd_f16", True, "f16", 2, 320, 67, 121, 32, "none"),
        # 32-bit training on odd-sized images, groups of three channels
        _norm("norm_train_517x999", True, "f32", 1, 48, 517, 999, 16, "silu"),
        # the full-resolution layer of a large training batch
        _norm("norm_train_512", True, "bf16", 8, 128, 512, 512, 32, "silu"),
        # a small image network's gradients: latency
        _clip("clip_small", "net", "f32", 24, 60_000, True, "same"),
        # a scene of about a million splats, every step above the limit
        _clip("clip_gaussians", "gaussians", "f32", 1_000_003, 0, True, "same"),
        # a network in 16 bits whose norm stays below the limit, the usual step: in place
        _clip("clip_idle", "net", "bf16", 300, 120_000_000, False, "inplace", 64),
        # 16-bit gradients, packed without gaps, clipped into the 32-bit buffer of a
        # mixed-precision optimiser
        _clip("clip_main_grads", "net", "bf16", 420, 160_000_000, True, "f32", 1),
    ]


def _log_int(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    if rng.random() < 0.6:
        train = rng.random() < 0.5
        groups = rng.choice([1, 4, 8, 16, 32])
        per = rng.choice([1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24])
        n, h, w = _log_int(rng, 1, 16), _log_int(rng, 3, 1100), _log_int(rng, 3, 1100)
        c = groups * per
        while n * c * h * w > 130_000_000:
            if n > 1:
                n = (n + 1) // 2
            elif h > w:
                h = h // 2 + 1
            else:
                w = w // 2 + 1
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        case = _norm("", train, dtype, n, c, h, w, groups, rng.choice(["silu", "silu", "none"]),
                     rng.choice(["f32", dtype]))
    else:
        active = rng.random() < 0.6
        dtype = rng.choice(["f32", "f32", "bf16", "f16"])
        out = rng.choice(["same", "f32"]) if active else "inplace"
        if rng.random() < 0.4:
            case = _clip("", "gaussians", dtype, _log_int(rng, 100, 1_000_000), 0, active, out)
        else:
            count = _log_int(rng, 3, 420)
            packed = rng.choice([1, 64] if count > 60 else [0, 0, 1, 64])
            case = _clip("", "net", dtype, count, _log_int(rng, 10_000, 100_000_000), active, out,
                         packed)
    del case["name"]
    return case


def _shapes(case):
    """Shapes of a clip case's tensors (a function of the case alone)."""
    if case["layout"] == "gaussians":
        n = case["count"]
        return [(n, 3), (n, 1, 3), (n, 15, 3), (n, 1), (n, 3), (n, 4)]
    count, total = case["count"], case["total"]
    r = random.Random(count * 1_000_003 + total)
    longs = (count + 2) // 3
    weights = [math.exp(r.uniform(-2.0, 2.0)) for _ in range(longs)]
    unit = total / sum(weights)
    shapes = []
    for i in range(count):
        if i % 3 == 0:
            shapes.append((max(1, int(unit * weights[i // 3])),))
        else:
            shapes.append((r.randint(1, 1024),))
    return shapes


def _scales(case):
    """Standard deviation of each tensor's gradient: layers differ by orders of magnitude."""
    r = random.Random(case["count"] * 7919 + case["total"])
    # 16-bit IEEE gradients carry a loss scale, the other types none
    base = 8.0 if case["dtype"] == "f16" else 0.05
    return [base * 10.0 ** -r.uniform(0.0, 2.0) for _ in _shapes(case)]


def _limit(case):
    """max_norm: well below the gradients' norm where clipping is active, well above if not."""
    total = sum(s * s * math.prod(shape) for s, shape in zip(_scales(case), _shapes(case)))
    return float((0.3 if case["active"] else 4.0) * math.sqrt(total))


# ------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------
def _buffers(case, dtype):
    """A clip case's tensors (zeros), and what holds them all: a list of the tensors, or of the
    one flat buffer that they are pieces of."""
    shapes, packed = _shapes(case), case["packed"]
    if not packed:
        tensors = [torch.zeros(shape, device="cuda", dtype=dtype) for shape in shapes]
        return tensors, tensors
    starts, end = [], 0
    for shape in shapes:
        starts.append((end + packed - 1) // packed * packed)
        end = starts[-1] + math.prod(shape)
    flat = torch.zeros(end, device="cuda", dtype=dtype)
    return [flat[b:b + math.prod(shape)].view(shape) for b, shape in zip(starts, shapes)], [flat]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    dt = DTYPES[case["dtype"]]
    if case["op"] == "norm":
        n, c, h, w = case["n"], case["c"], case["h"], case["w"]
        wdt = DTYPES[case["wdtype"]]
        spread, centre = 0.5 + randn(c).abs(), randn(c)
        # a convolution's output in the channels-last format: each channel has its own range
        x = randn(n, h, w, c).mul_(spread).add_(centre).to(dt).permute(0, 3, 1, 2)
        state = {"case": case, "x": x, "weight": (1.0 + 0.2 * randn(c)).to(wdt),
                 "bias": (0.2 * randn(c)).to(wdt)}
        if case["train"]:
            state["dy"] = randn(n, h, w, c).to(dt).permute(0, 3, 1, 2)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
        return state
    grads, flat = _buffers(case, dt)
    for t, s in zip(grads, _scales(case)):
        t.copy_(randn(*t.shape).mul_(s))
    state = {"case": case, "grads": grads, "max_norm": _limit(case)}
    if case["out"] == "inplace":
        params = []
        for t in grads:
            p = torch.nn.Parameter(torch.empty_like(t))
            p.grad = t
            params.append(p)
        state["params"] = params
        state["result"] = flat
    else:
        state["out"], state["result"] = _buffers(case, dt if case["out"] == "same" else torch.float32)
    return state


# ------------------------------------------------------------------------------------
# The framework's calls
# ------------------------------------------------------------------------------------
def _own(state):
    import fussim_b200 as fb

    case = state["case"]
    if case["op"] == "norm":
        act = None if case["act"] == "none" else case["act"]
        y = fb.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], eps=EPS,
                              activation=act)
        if not case["train"]:
            return y
        dx, dw, db = torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]),
                                         state["dy"])
        return y.detach(), dx, dw, db
    if case["out"] == "inplace":
        norm = fb.clip_grad_norm_(state["params"], state["max_norm"])
    else:
        _, norm = fb.clip_grad_norm(state["grads"], state["max_norm"], out=state["out"])
    return [norm] + state["result"]


# ------------------------------------------------------------------------------------
# The plain form
# ------------------------------------------------------------------------------------
def _plain_norm(state):
    case = state["case"]
    n, c, h, w, g = (case[k] for k in ("n", "c", "h", "w", "groups"))
    with torch.no_grad():
        x = state["x"].float().view(n, g, c // g, h, w)
        weight = state["weight"].float().view(1, g, c // g, 1, 1)
        bias = state["bias"].float().view(1, g, c // g, 1, 1)
        mean = x.mean(dim=(2, 3, 4), keepdim=True)
        d = x - mean
        rstd = 1.0 / torch.sqrt((d * d).mean(dim=(2, 3, 4), keepdim=True) + EPS)
        xhat = d * rstd
        z = xhat * weight + bias
        if case["act"] == "silu":
            s = 1.0 / (1.0 + torch.exp(-z))
            y = z * s
        else:
            y = z
        dt = state["x"].dtype
        y = y.reshape(n, c, h, w).to(dt)
        if not case["train"]:
            return y
        dz = state["dy"].float().view(n, g, c // g, h, w)
        if case["act"] == "silu":
            dz = dz * (s * (1.0 + z * (1.0 - s)))
        db = dz.sum(dim=(0, 3, 4)).reshape(c)
        dw = (dz * xhat).sum(dim=(0, 3, 4)).reshape(c)
        dxhat = dz * weight
        m1 = dxhat.mean(dim=(2, 3, 4), keepdim=True)
        m2 = (dxhat * xhat).mean(dim=(2, 3, 4), keepdim=True)
        dx = rstd * (dxhat - m1 - xhat * m2)
        return (y, dx.reshape(n, c, h, w).to(dt), dw.to(state["weight"].dtype),
                db.to(state["bias"].dtype))


def _plain_clip(state):
    grads = state["grads"]
    squares = [(t.float() * t.float()).sum(dtype=torch.float64) for t in grads]
    norm = torch.sqrt(torch.stack(squares).sum())
    coef = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    targets = grads if state["case"]["out"] == "inplace" else state["out"]
    for t, o in zip(grads, targets):
        o.copy_(t.float() * coef)
    return [norm.float()] + state["result"]


def run(state):
    if own:
        return _own(state)
    return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_clip(state)


# ------------------------------------------------------------------------------------
# Work and the definition in 64 bits
# ------------------------------------------------------------------------------------
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        elements = case["n"] * case["c"] * case["h"] * case["w"]
        params = case["c"] * DTYPES[case["wdtype"]].itemsize
        silu = case["act"] == "silu"
        # x read, y written; in training also dy read and dx written
        if case["train"]:
            return {"bytes": 4 * elements * size + 4 * params, "flops": elements * (30 if silu else 18)}
        return {"bytes": 2 * elements * size + 2 * params, "flops": elements * (11 if silu else 7)}
    elements = sum(math.prod(s) for s in _shapes(case))
    if not case["active"]:
        # the norm alone: gradients below the limit stay as they are
        return {"bytes": elements * size + 4, "flops": 2 * elements}
    osize = size if case["out"] == "same" else 4
    return {"bytes": elements * (size + osize) + 4, "flops": 3 * elements}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "clip":
            wide, whole = _buffers(case, torch.float64)
            squares = []
            for t, source in zip(wide, state["grads"]):
                t.copy_(source)
                squares.append(float(torch.dot(t.flatten(), t.flatten())))
            total = math.sqrt(math.fsum(squares))
            factor = min(1.0, state["max_norm"] / (total + 1e-6))
            return [torch.tensor(total, dtype=torch.float64, device="cuda")] + \
                [t.mul_(factor) for t in whole]
        n, c, h, w, groups = (case[k] for k in ("n", "c", "h", "w", "groups"))
        per = c // groups
        weight, bias = state["weight"].double(), state["bias"].double()
        y = torch.empty(n, c, h, w, dtype=torch.float64, device="cuda")
        train = case["train"]
        if train:
            dx = torch.empty_like(y)
            dweight, dbias = torch.zeros_like(weight), torch.zeros_like(bias)
        # image by image and group by group, straight from the definition
        for i in range(n):
            for k in range(groups):
                part = slice(k * per, (k + 1) * per)
                v = state["x"][i, part].double().reshape(per, h * w)
                m = h * w * per
                centred = v - v.sum() / m
                inv = (centred.square().sum() / m + EPS) ** -0.5
                normed = centred * inv
                pre = normed * weight[part, None] + bias[part, None]
                sig = torch.sigmoid(pre) if case["act"] == "silu" else None
                y[i, part] = (pre if sig is None else pre * sig).view(per, h, w)
                if train:
                    up = state["dy"][i, part].double().reshape(per, h * w)
                    if sig is not None:
                        up = up * (sig + pre * sig * (1.0 - sig))
                    dbias[part] += up.sum(1)
                    dweight[part] += (up * normed).sum(1)
                    up = up * weight[part, None]
                    up = up - up.sum() / m - normed * ((up * normed).sum() / m)
                    dx[i, part] = (up * inv).view(per, h, w)
        return (y, dx, dweight, dbias) if train else y

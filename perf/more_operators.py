"""Measured cases of the residual-block norms and of the AdamW step.

Two more operators of a training step whose loss is this package's, beside the group norm and
the clipping: the norms that stand before and after a block of an image transformer, fused
with the block's gate, residual scale and modulation (forward alone and with its gradients),
and the AdamW step over many tensors at once, with moments in 32 bits or in 8. Each is given
in its plain form (elementary torch operations in 32 bits) and as the calls that a user makes
of ``fussim_b200``.

Norm cases: x is (b, t, c), b images of t tokens (or pixels), y a block's output of that shape.

    r = x + residual_scale * gate * norm_after(y)       rounded to x's type
    z = norm_before(r) * (1 + scale) + shift            the next block's input, of y's type

A norm is over the c numbers of a token: "rms" or "layer" (with the mean taken off), times a
weight, plus a bias in the "layer" kind. ``form`` "before" is z of x alone, "both" is r and z.
``post`` is the kind of the norm after the block ("none": y as it is); ``gate`` is "none",
"channel" (c numbers, a learned layer scale) or "sample" (b x c numbers, from a conditioning);
``mod`` adds scale and shift (b x c). ``train`` adds all gradients for given gradients of r and z.
``dtype`` is y's and z's, ``xdtype`` that of x, r and of all parameters.

AdamW cases: lists of parameters, gradients and moments, the layouts of the tensors being a
splat scene ("gaussians", ``count`` splats of 59 numbers in six tensors) or a network ("net",
``count`` tensors with ``total`` numbers in the long ones), as pieces of flat buffers that begin
at multiples of ``packed`` numbers. ``pdtype`` and ``gdtype`` are the types of parameters and
gradients; ``copy`` is that of the rounded parameters which a mixed-precision step writes too;
``clip`` multiplies the gradients by min(1, max_norm / (norm + 1e-6)) on the way. ``bits`` 32:
both moments in float32. ``bits`` 8: per block of 256 numbers, float8_e4m3fn codes of the first
moment and of the second one's root, with a float32 scale for each (largest number / 448);
numbers are rounded up or down at random, in proportion, by a hash of seed, step, tensor and
position. The roots of second moments that are not zero are held as at least 2^-6 scales.
"""

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
RESIDUAL_SCALE = 0.7
BETAS = (0.9, 0.99)
ADAM_EPS = 1e-8
DECAY = 0.01
RATE = 1e-4
BLOCK = 256


# ------------------------------------------------------------------------------------
# Cases
# ------------------------------------------------------------------------------------
def _norm(name, form, train, dtype, xdtype, b, t, c, kind, post="none", gate="none", mod=False):
    return {"name": name, "op": "norm", "form": form, "train": train, "dtype": dtype,
            "xdtype": xdtype, "b": b, "t": t, "c": c, "kind": kind, "post": post, "gate": gate,
            "mod": mod}


def _adamw(name, layout, count, total, bits, pdtype, gdtype, copy="none", clip=False, packed=64):
    return {"name": name, "op": "adamw", "layout": layout, "count": count, "total": total,
            "bits": bits, "pdtype": pdtype, "gdtype": gdtype, "copy": copy, "clip": clip,
            "packed": packed}


def listed():
    return [
        # one token in decoding, or one pooled vector: launch latency
        _norm("block_token", "both", False, "bf16", "bf16", 1, 1, 2048, "rms", "rms"),
        # a modulated block of an image transformer at inference: 32 x 32 patches of 8 images
        _norm("block_image", "both", False, "bf16", "bf16", 8, 1024, 1152, "layer", "none",
              "sample", True),
        # the first norm of a wide network over a long sequence of video patches
        _norm("before_long", "before", False, "bf16", "bf16", 1, 16384, 4096, "rms"),
        # a small training step: a few images, norms on both sides, all in 16 bits
        _norm("train_small", "both", True, "bf16", "bf16", 2, 256, 768, "rms", "rms", "channel"),
        # a training batch with its residual stream in 32 bits, modulated
        _norm("train_mod", "both", True, "bf16", "f32", 16, 1024, 1024, "layer", "none", "sample",
              True),
        # odd sizes: rows that begin at no vector's boundary
        _norm("train_odd", "both", True, "f16", "f32", 3, 1771, 403, "layer", "layer", "channel"),
        # narrow layers over the pixels of 128 x 128 images, 32 bits throughout
        _norm("train_pixels", "both", True, "f32", "f32", 8, 16384, 96, "layer", "none", "channel"),
        # a small network's step in 32 bits: latency
        _adamw("adamw_small", "net", 24, 60_000, 32, "f32", "f32"),
        # a scene of about a million splats in 32 bits
        _adamw("adamw_gaussians", "gaussians", 1_000_003, 0, 32, "f32", "f32"),
        # mixed precision: 32-bit parameters, 16-bit gradients and copies, clipped
        _adamw("adamw_mixed", "net", 300, 100_000_000, 32, "f32", "bf16", "bf16", True),
        # moments in 8 bits beside 16-bit parameters: the smallest memory
        _adamw("adamw_8bit", "net", 420, 160_000_000, 8, "bf16", "bf16"),
        # moments in 8 bits, packed without gaps, 32-bit parameters, clipped
        _adamw("adamw_8bit_odd", "net", 90, 20_000_000, 8, "f32", "f32", "none", True, 1),
    ]


def _log_int(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    if rng.random() < 0.55:
        c = _log_int(rng, 8, 8192)
        if rng.random() < 0.6:
            c = (c + 7) // 8 * 8
        b = _log_int(rng, 1, 32)
        t = _log_int(rng, 1, 16384)
        form = rng.choice(["both", "both", "both", "before"])
        train = rng.random() < 0.6
        while b * t * c > 12_000_000:
            if t > b:
                t = t // 2 + 1
            else:
                b = (b + 1) // 2
        kind = rng.choice(["rms", "layer"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        xdtype = rng.choice(["f32", dtype])
        both = form == "both"
        case = _norm("", form, train, dtype, xdtype, b, t, c, kind,
                     rng.choice(["none", "rms", "layer"]) if both else "none",
                     rng.choice(["none", "channel", "sample"]) if both else "none",
                     rng.random() < 0.4)
    else:
        bits = rng.choice([32, 8])
        pdtype, gdtype, copy = rng.choice([("f32", "f32", "none"), ("f32", "f32", "bf16"),
                                           ("f32", "bf16", "bf16"), ("f32", "f16", "f16"),
                                           ("bf16", "bf16", "none"), ("bf16", "f32", "none"),
                                           ("f16", "f16", "none")])
        clip = rng.random() < 0.5
        packed = rng.choice([1, 64, 64])
        if rng.random() < 0.3:
            case = _adamw("", "gaussians", _log_int(rng, 100, 1_000_000), 0, bits, pdtype, gdtype,
                          copy, clip, packed)
        else:
            case = _adamw("", "net", _log_int(rng, 3, 420), _log_int(rng, 10_000, 60_000_000),
                          bits, pdtype, gdtype, copy, clip, packed)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------
def _shapes(case):
    """Shapes of an AdamW case's tensors (a function of the case alone)."""
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


def _spreads(case):
    """Standard deviation of each tensor's gradient: layers differ by orders of magnitude."""
    r = random.Random(case["count"] * 7919 + case["total"])
    # 16-bit IEEE gradients are kept away from the smallest numbers of their type
    base = 1.0 if case["gdtype"] == "f16" else 0.05
    return [base * 10.0 ** -r.uniform(0.0, 2.0) for _ in _shapes(case)]


def _pieces(case, dtype):
    """A flat buffer of zeros, and the tensors that are its pieces."""
    starts, end = [], 0
    for shape in _shapes(case):
        starts.append((end + case["packed"] - 1) // case["packed"] * case["packed"])
        end = starts[-1] + math.prod(shape)
    flat = torch.zeros(end, device="cuda", dtype=dtype)
    return flat, [flat[b:b + math.prod(shape)].view(shape)
                  for b, shape in zip(starts, _shapes(case))]


def _scale_pieces(case):
    """The scales of 8-bit moments, (blocks, 2) for each tensor, in one buffer."""
    blocks = [-(-math.prod(shape) // BLOCK) for shape in _shapes(case)]
    flat = torch.zeros(sum(blocks), 2, device="cuda")
    return flat, list(flat.split(blocks))


def _in_blocks(flat):
    """A tensor's numbers, 256 to a row, the last row filled up with zeros."""
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] == "norm":
        b, t, c = case["b"], case["t"], case["c"]
        xt, yt = DTYPES[case["xdtype"]], DTYPES[case["dtype"]]
        # channels of a residual stream differ in range, and tokens in size
        x = randn(b, t, c).mul_(0.3 + randn(c).abs()).mul_(0.5 + randn(b, t, 1).abs())
        state = {"case": case, "x": x.add_(0.3 * randn(c)).to(xt)}
        del x
        state["weight"] = (1.0 + 0.2 * randn(c)).to(xt)
        if case["kind"] == "layer":
            state["bias"] = (0.2 * randn(c)).to(xt)
        if case["mod"]:
            state["scale"] = (0.3 * randn(b, c)).to(xt)
            state["shift"] = (0.3 * randn(b, c)).to(xt)
        if case["form"] == "both":
            state["y"] = (0.2 + randn(b, t, c) * (0.5 + randn(c).abs())).to(yt)
            if case["gate"] != "none":
                state["gate"] = (0.5 * randn(*((c,) if case["gate"] == "channel" else (b, c)))).to(xt)
            if case["post"] != "none":
                state["post_weight"] = (1.0 + 0.2 * randn(c)).to(xt)
            if case["post"] == "layer":
                state["post_bias"] = (0.2 * randn(c)).to(xt)
        if case["train"]:
            state["leaves"] = [k for k in ("x", "y", "gate", "weight", "bias", "scale", "shift",
                                           "post_weight", "post_bias") if k in state]
            for k in state["leaves"]:
                state[k].requires_grad_(True)
            state["dz"] = randn(b, t, c).to(yt)
            if case["form"] == "both":
                state["dr"] = randn(b, t, c).to(xt)
        return state

    state = {"case": case, "step": 1000}
    kinds = {"params": case["pdtype"], "grads": case["gdtype"]}
    if case["copy"] != "none":
        kinds["copies"] = case["copy"]
    flats = {}
    for k, name in kinds.items():
        flats[k], state[k] = _pieces(case, DTYPES[name])
    moment = torch.float32 if case["bits"] == 32 else torch.float8_e4m3fn
    flats["firsts"], state["firsts"] = _pieces(case, moment)
    flats["seconds"], state["seconds"] = _pieces(case, moment)
    if case["bits"] == 8:
        flats["scales"], state["scales"] = _scale_pieces(case)
    squares = 0.0
    for i, s in enumerate(_spreads(case)):
        shape = state["params"][i].shape
        state["params"][i].copy_(0.05 * randn(*shape))
        grad, first = randn(*shape).mul_(s), randn(*shape).mul_(0.3 * s)
        second = randn(*shape).mul_(s).square_().mul_(0.3).add_(0.5 * s * s)
        if case["layout"] == "gaussians":
            # splats that the views so far have not seen have neither gradient nor moments
            seen = (torch.arange(shape[0], device="cuda") % 16 != 5).float()
            for part in (grad, first, second):
                part.mul_(seen.view(-1, *[1] * (len(shape) - 1)))
        state["grads"][i].copy_(grad)
        squares += s * s * grad.numel()
        if case["bits"] == 32:
            state["firsts"][i].copy_(first)
            state["seconds"][i].copy_(second)
            continue
        for j, (part, codes) in enumerate(((first, state["firsts"][i]), (second.sqrt(), state["seconds"][i]))):
            scales = _in_blocks(part.flatten()).abs().amax(1).clamp(min=2.0 ** -100) / 448.0
            state["scales"][i][:, j] = scales
            codes.view(-1).copy_(part.flatten() / scales.repeat_interleave(BLOCK)[:part.numel()])
    state["max_norm"] = 0.3 * math.sqrt(squares)
    state["result"] = [flats[k] for k in ("params", "copies", "firsts", "seconds", "scales") if k in flats]
    return state


# ------------------------------------------------------------------------------------
# The framework's calls
# ------------------------------------------------------------------------------------
def _own(state):
    import fussim_b200 as fb

    case = state["case"]
    if case["op"] == "norm":
        if case["form"] == "before":
            z = fb.block_norm(state["x"], state["weight"], state.get("bias"), kind=case["kind"],
                              scale=state.get("scale"), shift=state.get("shift"), eps=EPS,
                              out_dtype=DTYPES[case["dtype"]])
            outs, ups = (z,), [state.get("dz")]
        else:
            outs = fb.gated_residual_norm(
                state["x"], state["y"], state.get("gate"), state["weight"], state.get("bias"),
                kind=case["kind"], scale=state.get("scale"), shift=state.get("shift"),
                residual_scale=RESIDUAL_SCALE,
                branch_kind=None if case["post"] == "none" else case["post"],
                branch_weight=state.get("post_weight"), branch_bias=state.get("post_bias"), eps=EPS)
            ups = [state.get("dr"), state.get("dz")]
        if not case["train"]:
            return outs
        grads = torch.autograd.grad(outs, [state[k] for k in state["leaves"]], ups)
        return [o.detach() for o in outs] + list(grads)
    state["step"] += 1
    norm = fb.adamw_step_(
        state["params"], state["grads"], state["firsts"], state["seconds"], state.get("scales"),
        step=state["step"], lr=RATE, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY,
        max_norm=state["max_norm"] if case["clip"] else None, copies=state.get("copies"), seed=7)
    return ([norm] if case["clip"] else []) + state["result"]


# ------------------------------------------------------------------------------------
# The plain form
# ------------------------------------------------------------------------------------
def _normed(v, kind):
    """(v normalised over its last dimension, 1 / its spread)"""
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    inv = 1.0 / torch.sqrt((v * v).mean(dim=-1, keepdim=True) + EPS)
    return v * inv, inv


def _normed_grad(d, vhat, inv, kind):
    """The gradient of v for a gradient d of its normalised form."""
    out = d - vhat * (d * vhat).mean(dim=-1, keepdim=True)
    if kind == "layer":
        out = out - d.mean(dim=-1, keepdim=True)
    return out * inv


def _plain_norm(state):
    case = state["case"]
    b, c = case["b"], case["c"]
    both, kind, post = case["form"] == "both", case["kind"], case["post"]
    xt, yt = DTYPES[case["xdtype"]], DTYPES[case["dtype"]]
    with torch.no_grad():
        p = {k: state[k].float() for k in ("weight", "bias", "post_weight", "post_bias") if k in state}
        for k in ("gate", "scale", "shift"):
            if k in state:
                p[k] = state[k].float().view(-1, 1, c)
        x = state["x"].float()
        r = x
        if both:
            branch = state["y"].float()
            if post != "none":
                yhat, yinv = _normed(branch, post)
                branch = yhat * p["post_weight"]
                if "post_bias" in p:
                    branch = branch + p["post_bias"]
            gate = RESIDUAL_SCALE * p["gate"] if "gate" in p else RESIDUAL_SCALE
            r = (x + gate * branch).to(xt)
        rhat, rinv = _normed(r.float(), kind)
        pre = rhat * p["weight"]
        if "bias" in p:
            pre = pre + p["bias"]
        z = pre * (1.0 + p["scale"]) + p["shift"] if case["mod"] else pre
        outs = [r, z.to(yt)] if both else [z.to(yt)]
        if not case["train"]:
            return outs
        grads = {}
        dpre = state["dz"].float()
        if case["mod"]:
            grads["scale"] = (dpre * pre).sum(dim=1)
            grads["shift"] = dpre.sum(dim=1)
            dpre = dpre * (1.0 + p["scale"])
        grads["weight"] = (dpre * rhat).sum(dim=(0, 1))
        grads["bias"] = dpre.sum(dim=(0, 1))
        dr = _normed_grad(dpre * p["weight"], rhat, rinv, kind)
        if both:
            dr = dr + state["dr"].float()
            per_sample = (RESIDUAL_SCALE * dr * branch).sum(dim=1)
            grads["gate"] = per_sample if case["gate"] == "sample" else per_sample.sum(dim=0)
            dbranch = dr * gate
            if post != "none":
                grads["post_weight"] = (dbranch * yhat).sum(dim=(0, 1))
                grads["post_bias"] = dbranch.sum(dim=(0, 1))
                dbranch = _normed_grad(dbranch * p["post_weight"], yhat, yinv, post)
            grads["y"] = dbranch
        grads["x"] = dr
        return outs + [grads[k].to(state[k].dtype) for k in state["leaves"]]


def _mix(v):
    """A one-to-one scrambling of 32-bit numbers (ints, or int64 tensors)."""
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    v = ((v ^ (v >> 13)) * 0x3C6EF373) & 0xFFFFFFFF
    return v ^ (v >> 16)


def _randoms(seed, step, tensor, blocks):
    """32 random bits for each number of a tensor, (blocks, 256)."""
    key = _mix((_mix((_mix(seed) + step) & 0xFFFFFFFF) + tensor) & 0xFFFFFFFF)
    row = _mix((key + torch.arange(blocks, device="cuda")) & 0xFFFFFFFF)
    v = (row[:, None] + torch.arange(BLOCK, device="cuda") * 0x9E3779B1) & 0xFFFFFFFF
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return v ^ (v >> 15)


def _round_randomly(v, rnd):
    """Numbers in [0, 448] rounded to three bits behind the first, up in as many of the 2^20
    cases of rnd as the distance from the lower neighbour asks for."""
    bits = (v.view(torch.int32) + rnd.int()) & -0x100000
    return bits.view(torch.float32).clamp(max=448.0)


def _plain_adamw(state):
    case = state["case"]
    state["step"] += 1
    t = state["step"]
    with torch.no_grad():
        coef, norm = None, None
        if case["clip"]:
            squares = [(x.float() * x.float()).sum(dtype=torch.float64) for x in state["grads"]]
            norm = torch.sqrt(torch.stack(squares).sum()).float()
            coef = (state["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
        rate = RATE / (1.0 - BETAS[0] ** t)
        lift = 1.0 / math.sqrt(1.0 - BETAS[1] ** t)
        for i, (p, grad) in enumerate(zip(state["params"], state["grads"])):
            first, second = state["firsts"][i], state["seconds"][i]
            g = grad.float().flatten()
            if coef is not None:
                g = g * coef
            if case["bits"] == 8:
                scales = state["scales"][i]
                g = _in_blocks(g)
                m = _in_blocks(first.view(-1).float()) * scales[:, 0:1]
                root = _in_blocks(second.view(-1).float()) * scales[:, 1:2]
                v = root * root
            else:
                m, v = first.view(-1), second.view(-1)
            m = m * BETAS[0] + g * (1.0 - BETAS[0])
            v = v * BETAS[1] + (g * g) * (1.0 - BETAS[1])
            root = torch.sqrt(v)
            change = (m / (root * lift + ADAM_EPS)).view(-1)[:p.numel()]
            new = p.float().view(-1) * (1.0 - RATE * DECAY) - change * rate
            p.copy_(new.view(p.shape))
            if "copies" in state:
                state["copies"][i].copy_(new.view(p.shape))
            if case["bits"] == 32:
                first.view(-1).copy_(m)
                second.view(-1).copy_(v)
                continue
            rnd = _randoms(7, t, i, m.shape[0])
            for j, (codes, part) in enumerate(((first, m), (second, root))):
                top = part.abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
                scales[:, j:j + 1] = top / 448.0
                scaled = part.abs() * (448.0 / top)
                if j:
                    scaled = torch.where(part > 0, scaled.clamp(min=2.0 ** -6), scaled)
                held = _round_randomly(scaled, rnd >> 12 if j else rnd & 0xFFFFF)
                held = torch.where(part < 0, -held, held)
                codes.view(-1).copy_(held.view(-1)[:p.numel()])
    return ([norm] if case["clip"] else []) + state["result"]


def run(state):
    if own:
        return _own(state)
    return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_adamw(state)


# ------------------------------------------------------------------------------------
# Work and the definition in 64 bits
# ------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        b, c = case["b"], case["c"]
        n = b * case["t"] * c
        xs, ys = DTYPES[case["xdtype"]].itemsize, DTYPES[case["dtype"]].itemsize
        both = case["form"] == "both"
        params = c * (1 + (case["kind"] == "layer") + (case["post"] != "none") + (case["post"] == "layer"))
        params += {"none": 0, "channel": c, "sample": b * c}[case["gate"]] + 2 * b * c * case["mod"]
        # x read and z written; with a block's output also y read and r written
        size = n * (xs + ys) * (2 if both else 1) + params * xs
        flops = n * (8 + 4 * both + 6 * (case["post"] != "none"))
        if case["train"]:
            # dz read and dx written (dr read and dy written too), parameters' gradients written
            size += n * (xs + ys) * (2 if both else 1) + params * xs
            flops += n * (14 + 6 * both + 12 * (case["post"] != "none"))
        return {"bytes": size, "flops": flops}
    n = sum(math.prod(s) for s in _shapes(case))
    each = 2 * DTYPES[case["pdtype"]].itemsize + DTYPES[case["gdtype"]].itemsize
    if case["copy"] != "none":
        each += 2
    if case["bits"] == 32:
        each += 16
    else:
        each += 4 + 16 / BLOCK
    return {"bytes": n * each, "flops": n * (14 + 3 * case["clip"] + 14 * (case["bits"] == 8))}


def _exact_norm(state):
    """By torch's differentiation of the definition, image by image."""
    case = state["case"]
    both, b, c = case["form"] == "both", case["b"], case["c"]
    xt = DTYPES[case["xdtype"]]
    names = [k for k in ("gate", "weight", "bias", "scale", "shift", "post_weight", "post_bias") if k in state]
    wide = {k: state[k].detach().double().requires_grad_(case["train"]) for k in names}
    found = {k: [] for k in ("r", "z", "x", "y")}

    def normal(v, kind):
        if kind == "layer":
            v = v - v.sum(-1, keepdim=True) / c
        return v * (v.square().sum(-1, keepdim=True) / c + EPS).rsqrt()

    for i in range(b):
        def of(k):
            v = wide[k]
            return v[i] if v.dim() == 2 else v

        x = state["x"][i].detach().double().requires_grad_(case["train"])
        leaves, r = [x], x
        if both:
            y = state["y"][i].detach().double().requires_grad_(case["train"])
            leaves.append(y)
            out = y
            if case["post"] != "none":
                out = normal(y, case["post"]) * wide["post_weight"]
                if "post_bias" in wide:
                    out = out + wide["post_bias"]
            if "gate" in wide:
                out = out * of("gate")
            r = x + RESIDUAL_SCALE * out
            # r is held in its type, and its gradient passes through that rounding
            r = r + (r.detach().to(xt).double() - r.detach())
        z = normal(r, case["kind"]) * wide["weight"]
        if "bias" in wide:
            z = z + wide["bias"]
        if case["mod"]:
            z = z + z * of("scale") + of("shift")
        found["r"].append(r.detach())
        found["z"].append(z.detach())
        if case["train"]:
            total = (z * state["dz"][i].double()).sum()
            if both:
                total = total + (r * state["dr"][i].double()).sum()
            total.backward()
            for k, leaf in zip(("x", "y"), leaves):
                found[k].append(leaf.grad)
    outs = [torch.stack(found[k]) for k in (("r", "z") if both else ("z",))]
    if case["train"]:
        outs += [wide[k].grad if k in wide else torch.stack(found[k]) for k in state["leaves"]]
    return outs


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(state)
    t = state["step"] + 1
    factor, outs = 1.0, []
    if case["clip"]:
        norm = math.sqrt(math.fsum(float(x.double().flatten().dot(x.double().flatten())) for x in state["grads"]))
        factor = min(1.0, state["max_norm"] / (norm + 1e-6))
        outs.append(torch.tensor(norm, dtype=torch.float64, device="cuda"))
    flat, places = _pieces(case, torch.float64)
    moments = [_pieces(case, torch.float64) for _ in range(2)] if case["bits"] == 32 else None
    scales_flat, scales = _scale_pieces(case)
    scales_flat = scales_flat.double()
    tops = list(scales_flat.split([s.shape[0] for s in scales]))
    for i, place in enumerate(places):
        g = state["grads"][i].double() * factor
        old = [state[k][i].to(torch.float64 if case["bits"] == 32 else torch.float32).double()
               for k in ("firsts", "seconds")]
        if case["bits"] == 8:
            spread = state["scales"][i].double().repeat_interleave(BLOCK, 0)[:g.numel()]
            old = [v * spread[:, j].view(g.shape) for j, v in enumerate(old)]
            old[1] = old[1].square()
        m = old[0] + (1.0 - BETAS[0]) * (g - old[0])
        v = old[1] + (1.0 - BETAS[1]) * (g.square() - old[1])
        mean, spread = m / (1.0 - BETAS[0] ** t), (v / (1.0 - BETAS[1] ** t)).sqrt()
        w = state["params"][i].double()
        place.copy_(w - RATE * (DECAY * w + mean / (spread + ADAM_EPS)))
        if moments:
            moments[0][1][i].copy_(m)
            moments[1][1][i].copy_(v)
        else:
            for j, part in enumerate((m.abs(), v.sqrt())):
                tops[i][:, j] = _in_blocks(part.flatten()).amax(1).clamp(min=2.0 ** -100) / 448.0
    outs.append(flat)
    if case["copy"] != "none":
        outs.append(flat.clone())
    if moments:
        return outs + [moments[0][0], moments[1][0]]
    # a code is drawn by lot, the scales are not
    return outs + [None, None, scales_flat]

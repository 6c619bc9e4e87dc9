"""The AdamW step of one tensor, number by number, on the CPU: in 64 bits, and in the steps of
32 bits that its definition gives (every product, sum, quotient and root rounded by itself)."""

import math

import torch

BLOCK = 256
F8 = torch.float8_e4m3fn
MASK = 0xFFFFFFFF


def mix(v):
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & MASK
    v = ((v ^ (v >> 13)) * 0x3C6EF373) & MASK
    return v ^ (v >> 16)


def random_bits(seed, step, tensor, blocks, first_block=0):
    key = mix((mix((mix(seed) + step) & MASK) + tensor) & MASK)
    row = mix((key + first_block + torch.arange(blocks)) & MASK)[:, None]
    v = (row + torch.arange(BLOCK) * 0x9E3779B1) & MASK
    v = ((v ^ (v >> 15)) * 0xBB67AE85) & MASK
    return v ^ (v >> 15)


def blocks(flat):
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def decode(codes, scales, column):
    """What a moment's codes (in the order of memory) stand for, in FP32."""
    flat = blocks(codes.flatten().float()) * scales[:, column:column + 1]
    return flat.view(-1)[:codes.numel()]


def scale_of(part):
    """A block's largest finite number, in FP32, and the scale."""
    top = torch.where(part.isfinite(), part.abs(), 0.0).amax(1, keepdim=True).clamp(min=2.0 ** -100)
    return top, top * torch.tensor(1.0 / 448.0)


def encode(part, rnd, root):
    """(codes, scales) of blocks of a moment (root: of the second one's root)."""
    top, scales = scale_of(part)
    y = part.abs() * (torch.ones(()) / top * 448.0)
    if root:
        y = torch.where(part > 0, y.clamp(min=2.0 ** -6), y)
    y = ((y.view(torch.int32) + rnd.int()) & -0x100000).view(torch.float32).clamp(max=448.0)
    y = torch.where(part.isfinite(), torch.copysign(y, part), math.nan)
    return y.to(F8), scales


def step32(p, g, m, v, scales=None, *, step, lr, betas, eps, wd, coef=1.0, seed=0, tensor=0, first_block=0):
    """Flat tensors (from a block's first number on); m and v are codes where scales are given. Returns p (FP32, before its own
    rounding), m, v and, of codes, the scales."""
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    n = p.numel()
    p, g = blocks(p.float()), blocks(g.float()) * f(coef)
    if scales is None:
        m, v = blocks(m), blocks(v)
    else:
        m = blocks(m.float()) * scales[:, 0:1]
        root = blocks(v.float()) * scales[:, 1:2]
        v = root * root
    m = m * f(betas[0]) + g * f(1.0 - betas[0])
    v = v * f(betas[1]) + (g * g) * f(1.0 - betas[1])
    root = v.double().sqrt().float()  # (rounded once: 53 bits are enough for that)
    change = m / (root * f(1.0 / math.sqrt(1.0 - betas[1] ** step)) + f(eps))
    p = p * f(1.0 - lr * wd) - change * f(lr / (1.0 - betas[0] ** step))
    flat = lambda t: t.reshape(-1)[:n]  # noqa: E731
    if scales is None:
        return flat(p), flat(m), flat(v)
    rnd = random_bits(seed, step, tensor, p.shape[0], first_block)
    mc, ms = encode(m, rnd & 0xFFFFF, False)
    vc, vs = encode(root, rnd >> 12, True)
    return flat(p), flat(mc), flat(vc), torch.cat([ms, vs], 1)


def step64(p, g, m, v, *, step, lr, betas, eps, wd, coef=1.0):
    """The definition, in 64 bits, of what 32-bit moments (or decoded ones) and gradients hold."""
    p, g, m, v = p.double(), g.double() * coef, m.double(), v.double()
    m = betas[0] * m + (1.0 - betas[0]) * g
    v = betas[1] * v + (1.0 - betas[1]) * g * g
    den = (v / (1.0 - betas[1] ** step)).sqrt() + eps
    change = m / den
    p = (1.0 - lr * wd) * p - lr / (1.0 - betas[0] ** step) * change
    return p, m, v, change, den

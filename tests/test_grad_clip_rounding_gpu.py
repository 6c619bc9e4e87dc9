"""Each clipped number is rounded once: with a norm that is exact (integers, whose squares' sum FP32
and FP64 hold), an FP32 output is the exact product to half a step, and a few 2^-12 of one for the
factor, which is carried to more than 2^-36; 16-bit outputs, rounded from that FP32 number, to
half a step and 2^-24 of themselves."""

import math

import pytest
import torch

import fussim_b200 as fb

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def step(t, ref):
    """The distance of t's numbers at ref."""
    f = torch.finfo(t)
    _, e = torch.frexp(ref)
    return torch.ldexp(torch.full_like(ref, f.eps), e - 1).clamp_min(f.smallest_normal * f.eps)


@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, F32), (F16, F32), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 100, 2.0 ** -70])
def test_rounded_once(dtype, out_dtype, scale):
    if dtype == F16 and scale != 1.0:
        pytest.skip("beyond the type")
    g = torch.Generator().manual_seed(5)
    grads = [(torch.randint(-120, 121, (n,), generator=g).double() * scale).to(dtype).cuda()
             for n in (40_000, 7, 1001)]
    norm = math.sqrt(sum((t.double() / scale).square().sum().item() for t in grads)) * scale
    for k in range(40):
        limit = float(torch.tensor(norm * (0.013 + 0.024 * k), dtype=F32))
        outs = [torch.zeros(t.shape, dtype=out_dtype, device="cuda") for t in grads]
        fb.clip_grad_norm(grads, limit, out=outs)
        coef = min(1.0, limit / (norm + 1e-6))
        for t, o in zip(grads, outs):
            ref = t.double() * coef
            tol = step(out_dtype, ref) * (0.5 + 2.0 ** -10)
            if out_dtype != F32:
                tol = tol + 2.0 ** -24 * ref.abs()
            off = ((o.double() - ref).abs() / tol).max().item()
            assert off <= 1.0, f"{off:.3f} half steps at a factor of {coef}"


def test_a_factor_near_the_smallest_numbers():
    # 3e38 scaled to a norm of 1e-3: a factor of 1e-43, no FP32 number with bits of its own
    g = torch.full((1000,), 3e38, device="cuda")
    out, _ = fb.clip_grad_norm([g], 1e-3)
    limit = float(torch.tensor(1e-3, dtype=F32))
    ref = torch.full((), limit / math.sqrt(1000), dtype=torch.float64)
    # the norm's squares are summed in FP64 there: its own rounding to 2^-53
    assert ((out[0].double().cpu() - ref).abs() <= step(F32, ref) * (0.5 + 2.0 ** -10)).all()

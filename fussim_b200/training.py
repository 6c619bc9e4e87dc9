"""Operators of the training step around the loss.

* ``group_norm_act`` / ``GroupNormAct``: group normalisation with its activation over
  channels-last images, the layer that image networks (whose output goes into ``fused_ssim``
  or ``l1_dssim_loss``) repeat after every convolution; one fused forward and one fused
  backward, statistics in FP32 or wider for every input type.
* ``grad_norm``, ``clip_grad_norm_``, ``clip_grad_norm``: the global 2-norm of many gradient
  tensors and clipping by it, after the loss's backward pass.

Like the losses they run hand-written sm_100a kernels and have no CPU path. The reference
(OpsiClear/fussim) has no counterpart of these; users pair its loss with torch's
``group_norm``, ``silu`` and ``clip_grad_norm_``, whose definitions are kept.
"""

from __future__ import annotations

import math
from typing import Iterable, List, Optional, Sequence, Tuple

import torch

from .functional import _ensure_cuda_extension

ALLOWED_ACTIVATIONS = (None, "silu", "relu")
_ACTIVATION_CODE = {None: 0, "silu": 1, "relu": 2}
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _require_cuda(what: str) -> None:
    if not torch.cuda.is_available():
        raise RuntimeError(f"CUDA is not available. {what} requires a CUDA-capable GPU.")


# ------------------------------------------------------------------------------------
# Group normalisation with an activation
# ------------------------------------------------------------------------------------
def _check_norm(num_groups, num_channels, eps, activation):
    if activation not in ALLOWED_ACTIVATIONS:
        raise ValueError(f"activation must be one of {ALLOWED_ACTIVATIONS}, got {activation!r}")
    if num_groups < 1 or num_channels < 1 or num_channels % num_groups != 0:
        raise ValueError(
            f"the channels must divide into the groups, got {num_channels} channels and "
            f"{num_groups} groups"
        )
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")


def group_norm_act(
    x: torch.Tensor,
    num_groups: int,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    eps: float = 1e-5,
    activation: Optional[str] = "silu",
) -> torch.Tensor:
    """``act(group_norm(x, num_groups, weight, bias, eps))`` over a (B, C, H, W) CUDA tensor.

    Each of ``num_groups`` groups of C / num_groups channels is normalised over its channels
    and pixels (biased variance), scaled by ``weight`` and shifted by ``bias`` (C values each,
    or None), then activated: "silu", "relu" or None. float32, float16 and bfloat16 are read
    natively; statistics, arithmetic and the sums of the gradients are FP32 or wider, and the
    result, of x's type, is rounded once. ``weight`` and ``bias`` share a type, which need not
    be x's (32-bit parameters beside 16-bit images); autocast changes nothing here.

    The kernels work on the channels-last memory format and so is the result; another layout
    of x (or of the incoming gradient) costs one copy. Differentiable once, with respect to x,
    weight and bias. The results repeat bit for bit. Under graph capture follow torch's rule
    for backward passes: the captured leaves must not have live eager graphs.
    """
    if len(x.shape) != 4:
        raise ValueError(
            f"Expected 4D tensor (B, C, H, W), but got {len(x.shape)}D tensor with shape {x.shape}"
        )
    channels = x.shape[1]
    _check_norm(num_groups, channels, eps, activation)
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (channels,):
            raise ValueError(f"{name} must have shape ({channels},), got {tuple(t.shape)}")
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"{name} must be on x's device.\nx: {x.device}, {name}: {t.device}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(
            f"weight and bias must have the same dtype, got {weight.dtype} and {bias.dtype}"
        )
    _require_cuda("group_norm_act")
    if not x.is_cuda:
        raise RuntimeError(f"x must be on a CUDA device, but got device: {x.device}")
    train = torch.is_grad_enabled() and (
        x.requires_grad
        or (weight is not None and weight.requires_grad)
        or (bias is not None and bias.requires_grad)
    )
    return _ensure_cuda_extension().group_norm_act(
        x, num_groups, weight, bias, eps, _ACTIVATION_CODE[activation], train
    )


class GroupNormAct(torch.nn.Module):
    """``group_norm_act`` as a module, with ``torch.nn.GroupNorm``'s arguments, parameter names
    and initial values (its state dicts load here) and the activation."""

    def __init__(
        self,
        num_groups: int,
        num_channels: int,
        eps: float = 1e-5,
        affine: bool = True,
        activation: Optional[str] = "silu",
        device=None,
        dtype=None,
    ):
        super().__init__()
        _check_norm(num_groups, num_channels, eps, activation)
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.eps = eps
        self.affine = affine
        self.activation = activation
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(num_channels, device=device, dtype=dtype))
            self.bias = torch.nn.Parameter(torch.zeros(num_channels, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return group_norm_act(
            x, self.num_groups, self.weight, self.bias, self.eps, self.activation
        )

    def extra_repr(self) -> str:
        return (
            f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, "
            f"activation={self.activation!r}"
        )


# ------------------------------------------------------------------------------------
# Global gradient norm and clipping
# ------------------------------------------------------------------------------------
def _check_grads(grads: Sequence[torch.Tensor], what: str) -> None:
    device = grads[0].device
    for i, g in enumerate(grads):
        if g.layout != torch.strided:
            raise ValueError(f"gradients must be dense tensors, but {i} is {g.layout}")
        if g.dtype not in _DTYPES:
            raise ValueError(f"gradients must be float32, float16 or bfloat16, but {i} is {g.dtype}")
        if g.device != device:
            raise RuntimeError(
                f"gradients must be on one device.\nfirst: {device}, at index {i}: {g.device}"
            )
    _require_cuda(what)
    if device.type != "cuda":
        raise RuntimeError(f"gradients must be on a CUDA device, but got device: {device}")


def _check_max_norm(max_norm) -> float:
    value = float(max_norm)
    if not value >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    return value


def _raise_if_nonfinite(grads) -> None:
    norm = grad_norm(grads)
    if not math.isfinite(norm.item()):
        raise RuntimeError(
            f"the gradients' norm is {norm.item()}; nothing was clipped. Pass "
            "error_if_nonfinite=False to clip all the same"
        )


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all the tensors' numbers taken together: a 0-d float32 CUDA tensor.

    ``grads`` are dense CUDA tensors of one device, float32, float16 or bfloat16 in any mix;
    an empty sequence has norm 0 (on the current device). Squares are summed in FP64 beyond
    eight numbers and FP32's range does not limit them; the result repeats bit for bit. No
    host synchronisation. Not differentiable.
    """
    grads = list(grads)
    if not grads:
        _require_cuda("grad_norm")
        return torch.zeros((), device="cuda")
    _check_grads(grads, "grad_norm")
    return _ensure_cuda_extension().grad_norm(grads)


def clip_grad_norm(
    grads: Iterable[torch.Tensor],
    max_norm: float,
    out: Optional[Sequence[torch.Tensor]] = None,
    error_if_nonfinite: bool = False,
) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """Gradients scaled so that their common 2-norm is at most ``max_norm``, and that norm.

    Every tensor is multiplied by min(1, max_norm / (norm + 1e-6)) and the result rounded once
    into ``out`` (or new tensors of the same types). ``out`` has a tensor for each gradient, of
    its shape, and of its type or float32 (the 32-bit gradients of a mixed-precision
    optimiser); ``out[i]`` may be ``grads[i]``. Otherwise no two of the tensors written, and
    no gradient and another's output, may share memory. A norm that is NaN makes everything
    NaN, an infinite one makes finite numbers 0; ``error_if_nonfinite`` raises instead, before
    anything is written, at the price of a host synchronisation. Tensors whose numbers do not
    fill their memory are copied once more.
    """
    grads = list(grads)
    max_norm = _check_max_norm(max_norm)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"out must have a tensor for each gradient, got {len(out)} for {len(grads)}")
    if not grads:
        _require_cuda("clip_grad_norm")
        return [], torch.zeros((), device="cuda")
    _check_grads(grads, "clip_grad_norm")
    if out is None:
        out = [torch.empty_like(g, requires_grad=False) for g in grads]
    for i, (g, o) in enumerate(zip(grads, out)):
        if o.shape != g.shape:
            raise ValueError(f"out[{i}] must have shape {tuple(g.shape)}, got {tuple(o.shape)}")
        if o.dtype != g.dtype and o.dtype != torch.float32:
            raise ValueError(f"out[{i}] must be {g.dtype} or float32, got {o.dtype}")
        if o.device != g.device or o.layout != torch.strided:
            raise RuntimeError(f"out[{i}] must be a dense tensor on {g.device}")
    if error_if_nonfinite:
        _raise_if_nonfinite(grads)
    return out, _ensure_cuda_extension().clip_grads(grads, out, max_norm)


def clip_grad_norm_(
    parameters,
    max_norm: float,
    error_if_nonfinite: bool = False,
) -> torch.Tensor:
    """Clip the parameters' gradients in place to a common 2-norm of ``max_norm``; returns the
    norm before clipping, a 0-d float32 tensor (``torch.nn.utils.clip_grad_norm_`` for
    ``norm_type=2``). Parameters without a gradient are passed over. Where the norm is within
    the limit the gradients are left untouched (and not read a second time); otherwise as
    ``clip_grad_norm`` with ``out=grads``. A gradient may be given once only.
    """
    max_norm = _check_max_norm(max_norm)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    if not grads:
        _require_cuda("clip_grad_norm_")
        return torch.zeros((), device="cuda")
    _check_grads(grads, "clip_grad_norm_")
    if error_if_nonfinite:
        _raise_if_nonfinite(grads)
    return _ensure_cuda_extension().clip_grads(grads, grads, max_norm)

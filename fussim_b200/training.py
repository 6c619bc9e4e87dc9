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

from typing import Iterable, List, Optional, Sequence, Tuple

import torch

from .functional import _ensure_cuda_extension


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
    of x (or of the incoming gradient) costs one copy. Differentiable once, backwards, with
    respect to x, weight and bias; forward-mode derivatives and tracing (``torch.jit.trace``,
    ``make_fx``) raise RuntimeError. The results repeat bit for bit. Under graph capture follow torch's rule
    for backward passes: the captured leaves must not have live eager graphs.
    """
    # arguments are checked in the extension: the call costs little more than its launches
    return _ensure_cuda_extension().group_norm_act(x, num_groups, weight, bias, eps, activation)


class GroupNormAct(torch.nn.Module):
    """``group_norm_act`` as a module, with ``torch.nn.GroupNorm``'s arguments in their order,
    parameter names and initial values (its state dicts load here), and the activation."""

    def __init__(
        self,
        num_groups: int,
        num_channels: int,
        eps: float = 1e-5,
        affine: bool = True,
        device=None,
        dtype=None,
        activation: Optional[str] = "silu",
    ):
        super().__init__()
        _ensure_cuda_extension().check_norm_settings(num_groups, num_channels, eps, activation)
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


def grad_norm(grads: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all the tensors' numbers taken together: a 0-d float32 CUDA tensor.

    ``grads`` are dense CUDA tensors of one device, float32, float16 or bfloat16 in any mix;
    an empty sequence has norm 0 (on the current device). Squares are summed in FP64 beyond
    32 numbers and FP32's range does not limit them; the result repeats bit for bit. No
    host synchronisation. Not differentiable; tracing raises RuntimeError.
    """
    return _ensure_cuda_extension().grad_norm(list(grads))


def clip_grad_norm(
    grads: Iterable[torch.Tensor],
    max_norm: float,
    out: Optional[Sequence[torch.Tensor]] = None,
    *,
    error_if_nonfinite: bool = False,
) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """Gradients scaled so that their common 2-norm is at most ``max_norm``, and that norm.

    Every tensor is multiplied by min(1, max_norm / (norm + 1e-6)) and the result rounded once
    into ``out`` (or new tensors of the same types). ``out`` has a tensor for each gradient, of
    its shape, and of its type or float32 (the 32-bit gradients of a mixed-precision
    optimiser); ``out[i]`` may be ``grads[i]``. Otherwise no two of the tensors written, and
    no gradient and another's output, may share memory: ValueError (a gradient that does not
    fill its memory is copied before anything is written, and may). A norm that is NaN makes
    everything NaN, an infinite gradient makes finite numbers 0; ``error_if_nonfinite`` raises
    instead, before anything is written, at the price of a host synchronisation. Tensors whose
    numbers do not fill their memory are copied once more. Not differentiable, as ``grad_norm``.
    """
    return _ensure_cuda_extension().clip_grad_norm(
        list(grads), float(max_norm), None if out is None else list(out), error_if_nonfinite
    )


def clip_grad_norm_(
    parameters,
    max_norm: float,
    norm_type: float = 2.0,
    error_if_nonfinite: bool = False,
) -> torch.Tensor:
    """Clip the parameters' gradients in place to a common 2-norm of ``max_norm``; returns the
    norm before clipping, a 0-d float32 tensor (``torch.nn.utils.clip_grad_norm_`` for
    ``norm_type=2``, the only one here: others raise ValueError). Parameters without a gradient
    are passed over. Where the norm is within the limit the gradients are left untouched (and
    not read a second time); otherwise as ``clip_grad_norm`` with ``out=grads``. A gradient may
    be given once only.
    """
    if float(norm_type) != 2.0:
        raise ValueError(f"norm_type must be 2, got {norm_type}")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return _ensure_cuda_extension().clip_grad_norm_(
        list(parameters), float(max_norm), error_if_nonfinite
    )

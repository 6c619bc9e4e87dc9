"""Norms before and after the residual blocks of an image transformer (or any network over rows of
channels), fused with the block's gate, residual scale and modulation.

* ``block_norm`` / ``BlockNorm``: the norm before a block.
* ``gated_residual``: a block's output, normalised, gated and added to the residual stream.
* ``gated_residual_norm``: both in one pass, the end of one block and the start of the next.

The token counterpart of ``group_norm_act`` for networks whose output goes into ``fused_ssim`` or
``l1_dssim_loss``; hand-written sm_100a kernels without a CPU path. The reference
(OpsiClear/fussim) has no counterpart of these.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .functional import _ensure_cuda_extension


def block_norm(
    x: torch.Tensor,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    *,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    kind: str = "rms",
    eps: float = 1e-6,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``(norm(x) * weight + bias) * (1 + scale) + shift`` over the last dimension of a CUDA tensor.

    norm(x) = (x - mean) / sqrt(mean((x - mean)^2) + eps) over the last dimension's C numbers (1 to
    16384); ``kind`` "layer" takes the mean off, "rms" takes it as zero. ``weight`` and ``bias``
    have C values; ``scale`` and ``shift``, a conditioning, C values or (B, C) for x of shape
    (B, ..., C), one row for each sample. Each may be None and have any of the types float32,
    float16 and bfloat16, as x. The result has x's type, or for float32 ``out_dtype``. Statistics
    and arithmetic are FP32 and results are rounded once (gradients of vectors that are summed over
    rows: FP32 over 256 of a thread's rows, FP64 over many CTAs'); autocast changes nothing here.

    Images of shape (B, C, H, W) in the channels-last memory format are normalised over their
    channels as ``x.permute(0, 2, 3, 1)``, without a copy; inputs (and incoming gradients) whose
    last dimension is not dense row behind row cost one. Differentiable once, backwards;
    forward-mode derivatives and tracing raise RuntimeError. The results repeat bit for bit.
    Under graph capture follow torch's rule for backward passes: the captured leaves must not
    have live eager graphs.
    """
    return _ensure_cuda_extension().block_norm(x, weight, bias, scale, shift, kind, eps, out_dtype)


def gated_residual(
    x: torch.Tensor,
    branch: torch.Tensor,
    gate: Optional[torch.Tensor] = None,
    *,
    residual_scale: float = 1.0,
    branch_kind: Optional[str] = None,
    branch_weight: Optional[torch.Tensor] = None,
    branch_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> torch.Tensor:
    """``x + residual_scale * gate * (norm(branch) * branch_weight + branch_bias)``, in x's type.

    ``branch`` is the output of a residual block, of x's shape and of x's type, or 16 bits wide
    beside a float32 residual stream x. ``branch_kind`` is the kind of the norm after the block
    (None: the branch as it is, and then no weight and bias). ``gate`` has C values (a learned
    layer scale) or (B, C) (a conditioning), or is None; ``residual_scale`` is finite in FP32. A
    16-bit result with a normalised branch is formed in FP64 and rounded to FP32 and from that to its
    type. The result may be written in place before the backward pass. Otherwise as ``block_norm``.
    """
    return _ensure_cuda_extension().gated_residual(
        x, branch, gate, residual_scale, branch_kind, branch_weight, branch_bias, eps
    )


def gated_residual_norm(
    x: torch.Tensor,
    branch: torch.Tensor,
    gate: Optional[torch.Tensor] = None,
    weight: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    *,
    scale: Optional[torch.Tensor] = None,
    shift: Optional[torch.Tensor] = None,
    kind: str = "rms",
    residual_scale: float = 1.0,
    branch_kind: Optional[str] = None,
    branch_weight: Optional[torch.Tensor] = None,
    branch_bias: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The end of one block and the start of the next: (r, z) with r as ``gated_residual``'s result
    (rounded to x's type) and z = ``block_norm`` of that r, in the branch's type; one kernel, which
    reads x and branch once, and one pass over rows backwards.
    """
    return _ensure_cuda_extension().gated_residual_norm(
        x, branch, gate, weight, bias, scale, shift, kind, residual_scale, branch_kind,
        branch_weight, branch_bias, eps
    )


class BlockNorm(torch.nn.Module):
    """``block_norm`` as a module, with the parameter names, shapes and initial values of
    ``torch.nn.RMSNorm`` (``kind`` "rms": weight) or ``torch.nn.LayerNorm`` ("layer": weight and
    bias) over ``num_channels``: their state dicts load here."""

    def __init__(
        self,
        num_channels: int,
        kind: str = "rms",
        eps: float = 1e-6,
        affine: bool = True,
        device=None,
        dtype=None,
    ):
        super().__init__()
        if not 1 <= num_channels <= 16384:
            raise ValueError(f"num_channels must be from 1 to 16384, got {num_channels}")
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
        self.num_channels = num_channels
        self.kind = kind
        self.eps = eps
        self.affine = affine
        options = dict(device=device, dtype=dtype)
        if affine:
            self.weight = torch.nn.Parameter(torch.ones(num_channels, **options))
        else:
            self.register_parameter("weight", None)
        if affine and kind == "layer":
            self.bias = torch.nn.Parameter(torch.zeros(num_channels, **options))
        else:
            self.register_parameter("bias", None)

    def forward(
        self,
        x: torch.Tensor,
        scale: Optional[torch.Tensor] = None,
        shift: Optional[torch.Tensor] = None,
        out_dtype: Optional[torch.dtype] = None,
    ) -> torch.Tensor:
        return block_norm(x, self.weight, self.bias, scale=scale, shift=shift, kind=self.kind,
                          eps=self.eps, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        return f"{self.num_channels}, {self.kind!r}, eps={self.eps}, affine={self.affine}"

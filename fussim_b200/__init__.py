"""fussim_b200 — differentiable SSIM for PyTorch on NVIDIA B200 (sm_100a).

Drop-in for the public API of OpsiClear/fussim (``fussim/__init__.py``):

* ``fused_ssim(img1, img2, padding="same", train=True, window_size=11)`` — scalar mean SSIM;
* ``ssim`` / ``SSIM`` — the pytorch-msssim compatible wrappers (``size_average=False``
  returns one value per image);
* ``FusedSSIMMap`` / ``FusedSSIMMapFP16`` — the map-producing autograd Functions;
* ``SUPPORTED_WINDOW_SIZES``, ``get_build_info``, ``check_compatibility``.

Beside the losses, operators of the training step around them: ``group_norm_act`` /
``GroupNormAct`` (group normalisation with its activation, channels last), ``block_norm`` /
``BlockNorm`` / ``gated_residual`` / ``gated_residual_norm`` (the norms before and after a residual block, with its
gate and modulation), ``grad_norm`` / ``clip_grad_norm`` / ``clip_grad_norm_`` (the global gradient
norm and clipping) and ``adamw_step_`` / ``AdamW`` (the AdamW step of many tensors, with moments in
32 or 8 bits).

Gradients of the losses flow to the first image only. Under ``torch.autocast`` the inputs are rounded
to FP16 (whatever the autocast dtype, as the reference does) and the arithmetic stays
FP32. There is no CPU path: every call runs the hand-written sm_100a kernels of
``libfussim_b200.so`` and fails loudly if they are missing.
"""

from .blocks import (  # noqa: F401
    BlockNorm,
    block_norm,
    gated_residual,
    gated_residual_norm,
)
from .functional import (  # noqa: F401
    ALLOWED_PADDING,
    SSIM,
    SUPPORTED_WINDOW_SIZES,
    FusedSSIMMap,
    FusedSSIMMapFP16,
    __version__,
    check_compatibility,
    check_device_errors,
    fused_ssim,
    get_build_info,
    l1_dssim_loss,
    poll_device_error,
    ssim,
)
from .optimizer import AdamW, adamw_moments, adamw_step_  # noqa: F401
from .training import (  # noqa: F401
    GroupNormAct,
    clip_grad_norm,
    clip_grad_norm_,
    grad_norm,
    group_norm_act,
)

__all__ = [
    # Primary API
    "fused_ssim",
    "l1_dssim_loss",
    # pytorch-msssim compatible API
    "ssim",
    "SSIM",
    # Training step around the loss
    "group_norm_act",
    "GroupNormAct",
    "block_norm",
    "BlockNorm",
    "gated_residual",
    "gated_residual_norm",
    "grad_norm",
    "clip_grad_norm",
    "clip_grad_norm_",
    "adamw_step_",
    "adamw_moments",
    "AdamW",
    # Advanced/internal
    "FusedSSIMMap",
    "FusedSSIMMapFP16",
    # Utilities
    "__version__",
    "get_build_info",
    "check_compatibility",
    "check_device_errors",
    "poll_device_error",
    "SUPPORTED_WINDOW_SIZES",
]

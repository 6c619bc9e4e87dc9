"""residual_scale has to be a finite float32: the kernels multiply the gate by it in FP32."""

import ctypes

import pytest
import torch

import fussim_b200 as fb
from tests.test_block_norm_cpu import ARGUMENT, WORKSPACE, X, backward, forward, lib  # noqa: F401

WIDE = [1e39, -1e300, float("inf"), float("-inf"), float("nan")]


@pytest.mark.parametrize("s", WIDE)
def test_refused(lib, s):  # noqa: F811
    for f in (fb.gated_residual, fb.gated_residual_norm):
        with pytest.raises(ValueError, match="residual_scale"):
            f(X, X, residual_scale=s)
    assert lib.fssim_block_norm_forward(ctypes.byref(forward(residual_scale=s)), None) == ARGUMENT
    a = backward(residual_scale=s)
    assert lib.fssim_block_norm_backward(ctypes.byref(a), None) == ARGUMENT
    assert b"residual_scale" in lib.fssim_last_error()


@pytest.mark.parametrize("s", [0.0, -0.5, 3.4e38, 1e-300])
def test_taken(lib, s):  # noqa: F811
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA is not available"):
            fb.gated_residual(X, X, residual_scale=s)
    assert lib.fssim_block_norm_backward(ctypes.byref(backward(residual_scale=s)), None) == WORKSPACE


def test_without_a_branch(lib):  # noqa: F811
    """It is not looked at there."""
    a = backward(residual_scale=float("nan"), branch=None, dbranch=None)
    assert lib.fssim_block_norm_backward(ctypes.byref(a), None) == WORKSPACE

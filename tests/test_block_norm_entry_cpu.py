"""The block norms' C entry points refuse a branch's weight and bias where the branch has no norm, as the
Python functions do: a call that is refused reaches no GPU."""

import ctypes

import pytest

from tests.test_block_norm_cpu import ARGUMENT, SOME, WORKSPACE, Channels, backward, forward, lib  # noqa: F401

VECTOR = Channels(SOME, 0, 0)


@pytest.mark.parametrize("name", ["branch_weight", "branch_bias"])
def test_forward(lib, name):  # noqa: F811
    for kw in (dict(), dict(gate=VECTOR), dict(z=None, kind=0)):
        a = forward(branch_kind=0, **{name: VECTOR}, **kw)
        assert lib.fssim_block_norm_forward(ctypes.byref(a), None) == ARGUMENT
        assert b"branch_kind" in lib.fssim_last_error()
    # without rows nothing is computed, but the arguments are as wrong
    assert lib.fssim_block_norm_forward(ctypes.byref(forward(T=0, branch_kind=0, **{name: VECTOR})), None) == ARGUMENT


@pytest.mark.parametrize("name", ["branch_weight", "branch_bias", "dbranch_weight", "dbranch_bias"])
def test_backward(lib, name):  # noqa: F811
    for kw in (dict(), dict(gate=VECTOR, dgate=VECTOR), dict(dbranch=SOME)):
        a = backward(branch_kind=0, workspace=SOME, workspace_bytes=0, **{name: VECTOR}, **kw)
        assert lib.fssim_block_norm_backward(ctypes.byref(a), None) == ARGUMENT
        assert b"branch_kind" in lib.fssim_last_error()
        assert lib.fssim_block_norm_backward_workspace_bytes(ctypes.byref(a)) == 0


def test_with_a_norm(lib):  # noqa: F811
    """The same vectors go with a norm of the branch (the call is refused later, for its workspace)."""
    a = backward(branch_kind=1, branch_stats=SOME, branch_weight=VECTOR, branch_bias=VECTOR, dbranch_weight=VECTOR)
    assert lib.fssim_block_norm_backward(ctypes.byref(a), None) == WORKSPACE
    assert lib.fssim_block_norm_backward_workspace_bytes(ctypes.byref(a)) > 0

"""Host-side behaviour of the block norms (runs without a GPU): checks of arguments, what cannot be
recorded, and the C entry points' refusals, none of which reaches the GPU."""

import ctypes
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

import fussim_b200 as fb

LIB = os.path.join(os.path.dirname(os.path.abspath(fb.__file__)), "libfussim_b200.so")
X = torch.randn(2, 5, 12)
W = torch.ones(12)


def both(**kw):
    args = dict(x=X, branch=X)
    args.update(kw)
    return fb.gated_residual_norm(**args)


def test_public_names():
    for name in ("block_norm", "BlockNorm", "gated_residual", "gated_residual_norm"):
        assert name in fb.__all__ and hasattr(fb, name)


@pytest.mark.parametrize("kw,match", [
    (dict(kind=None), "kind must be"),
    (dict(kind="group"), "kind must be"),
    (dict(branch_kind="batch"), "branch_kind must be"),
    (dict(eps=-1e-6), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(residual_scale=float("nan")), "residual_scale"),
    (dict(x=torch.tensor(1.0), branch=torch.tensor(1.0)), "at least one dimension"),
    (dict(x=torch.zeros(3, 0), branch=torch.zeros(3, 0)), "at least one dimension"),
    (dict(x=torch.zeros(1, 16385), branch=torch.zeros(1, 16385)), "16384"),
    (dict(x=X.double(), branch=X.double()), "x must be float32"),
    (dict(x=X.to_sparse()), "dense"),
    (dict(branch=X.double()), "branch must be of x's type, float16 or bfloat16"),
    (dict(x=X.half()), "branch must be of x's type, got"),
    (dict(x=X.half(), branch=X.bfloat16()), "branch must be of x's type, got"),
    (dict(branch=X[:1]), "branch must have x's shape"),
    (dict(branch=X.to_sparse()), "branch must be a dense"),
    (dict(gate=torch.ones(2)), "gate must have shape"),
    (dict(gate=torch.ones(5, 12)), "gate must have shape"),
    (dict(gate=torch.ones(2, 1, 12)), "gate must have shape"),
    (dict(gate=W.double()), "gate must be float32"),
    (dict(weight=torch.ones(2, 12)), "weight must have shape"),
    (dict(bias=torch.ones(11)), "bias must have shape"),
    (dict(scale=torch.ones(1, 12)), "scale must have shape"),
    (dict(shift=torch.ones(12, 1)), "shift must have shape"),
    (dict(shift=W.long()), "shift must be float32"),
    (dict(branch_weight=W), "go with branch_kind"),
    (dict(branch_bias=W), "go with branch_kind"),
    (dict(branch_kind="rms", branch_weight=torch.ones(2, 12)), "branch_weight must have shape"),
    (dict(x=X[0, 0], branch=X[0, 0], gate=torch.ones(1, 12)), "gate must have shape"),
])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        both(**kw)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_module(kind):
    m = fb.BlockNorm(12, kind)
    ref = (torch.nn.RMSNorm if kind == "rms" else torch.nn.LayerNorm)(12)
    assert {k: v.shape for k, v in m.state_dict().items()} == {k: v.shape for k, v in ref.state_dict().items()}
    m.load_state_dict(ref.state_dict())
    assert torch.equal(m.weight, ref.weight) and repr(m) == f"BlockNorm(12, {kind!r}, eps=1e-06, affine=True)"
    assert not list(fb.BlockNorm(12, kind, affine=False).parameters())
    assert fb.BlockNorm(12, kind, 1e-5, True, "cpu", torch.bfloat16).weight.dtype == torch.bfloat16
    for args in ((0,), (16385,), (12, "batch")):
        with pytest.raises(ValueError, match="must be"):
            fb.BlockNorm(*args)


def test_out_dtype():
    for x, t in ((X, torch.float64), (X.half(), torch.float32), (X.half(), torch.bfloat16)):
        with pytest.raises(ValueError, match="out_dtype must be of x's type"):
            fb.block_norm(x, out_dtype=t)


def test_devices():
    with pytest.raises(RuntimeError, match="branch must be on x's device"):
        both(branch=X.to("meta"))
    with pytest.raises(RuntimeError, match="gate must be on x's device"):
        both(gate=W.to("meta"))
    if not torch.cuda.is_available():
        for f in (both, lambda: fb.block_norm(X), lambda: fb.gated_residual(X, X)):
            with pytest.raises(RuntimeError, match="CUDA is not available"):
                f()


CALLS = {
    "block_norm": lambda x, w: fb.block_norm(x, w, scale=w),
    "gated_residual": lambda x, w: fb.gated_residual(x, x, w),
    "gated_residual_norm": lambda x, w: fb.gated_residual_norm(x, x, w),
}


@pytest.mark.parametrize("name", CALLS)
def test_recording(name):
    f = CALLS[name]
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        torch.jit.trace(f, (X, W))
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        make_fx(f)(X, W)
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode.*x carries"):
            f(fwAD.make_dual(X.clone(), X), W)
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(X, fwAD.make_dual(W.clone(), W))


# ---- the C entry points ----
P, I64, I32, F, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_double


class Channels(ctypes.Structure):
    _fields_ = [("data", P), ("dtype", I32), ("per_sample", I32)]


class ForwardArgs(ctypes.Structure):
    _fields_ = [("x_dtype", I32), ("y_dtype", I32), ("kind", I32), ("branch_kind", I32), ("B", I64), ("T", I64),
                ("C", I64), ("eps", F), ("residual_scale", F64), ("x", P), ("branch", P), ("r", P), ("z", P)] + \
        [(k, Channels) for k in ("gate", "weight", "bias", "scale", "shift", "branch_weight", "branch_bias")] + \
        [("stats", P), ("branch_stats", P)]


class BackwardArgs(ctypes.Structure):
    _fields_ = [("x_dtype", I32), ("y_dtype", I32), ("kind", I32), ("branch_kind", I32), ("B", I64), ("T", I64),
                ("C", I64), ("residual_scale", F64), ("r", P), ("branch", P), ("dr", P), ("dz", P), ("stats", P),
                ("branch_stats", P)] + \
        [(k, Channels) for k in ("gate", "weight", "bias", "scale", "branch_weight", "branch_bias")] + \
        [("dx", P), ("dbranch", P)] + \
        [(k, Channels) for k in ("dgate", "dweight", "dbias", "dscale", "dshift", "dbranch_weight", "dbranch_bias")] + \
        [("workspace", P), ("workspace_bytes", ctypes.c_size_t)]


SHAPE, DTYPE, NULLPTR, WORKSPACE, ARGUMENT = 2, 3, 4, 5, 7
SOME = 1 << 20  # a pointer that no refused call follows


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.fssim_last_error.restype = ctypes.c_char_p
    lib.fssim_block_norm_backward_workspace_bytes.restype = ctypes.c_size_t
    for f in ("fssim_block_norm_forward", "fssim_block_norm_backward"):
        getattr(lib, f).argtypes = [P, P]
    return lib


def fill(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def forward(**kw):
    return fill(ForwardArgs(kind=1, B=2, T=64, C=32, eps=1e-6, residual_scale=1.0, x=SOME, branch=SOME, r=SOME, z=SOME), kw)


@pytest.mark.parametrize("kw,status", [
    (dict(x_dtype=3), DTYPE), (dict(x_dtype=1), DTYPE), (dict(x_dtype=1, y_dtype=2), DTYPE),
    (dict(kind=0), ARGUMENT), (dict(kind=3), ARGUMENT), (dict(branch_kind=-1), ARGUMENT),
    (dict(B=-1), SHAPE), (dict(T=-1), SHAPE), (dict(C=0), SHAPE), (dict(C=16385), SHAPE),
    (dict(B=1 << 30, T=1 << 30), SHAPE), (dict(B=1 << 41, T=0), SHAPE),
    (dict(B=1 << 33, T=1, gate=Channels(SOME, 0, 1)), SHAPE),
    (dict(eps=-1.0), ARGUMENT), (dict(eps=float("nan")), ARGUMENT),
    (dict(gate=Channels(SOME, 3, 0)), DTYPE), (dict(shift=Channels(SOME + 2, 0, 0)), ARGUMENT),
    (dict(branch_bias=Channels(SOME + 1, 2, 0)), ARGUMENT),
    (dict(x=None), NULLPTR), (dict(r=None), NULLPTR), (dict(z=None, branch=None), NULLPTR),
    (dict(x=SOME + 2), ARGUMENT), (dict(branch=SOME + 1), ARGUMENT), (dict(r=SOME + 2), ARGUMENT),
    (dict(z=SOME + 3), ARGUMENT), (dict(stats=SOME + 4), ARGUMENT), (dict(branch_stats=SOME + 4), ARGUMENT),
    (dict(B=0), 0), (dict(T=0), 0),
])
def test_c_forward_refusals(lib, kw, status):
    assert lib.fssim_block_norm_forward(ctypes.byref(forward(**kw)), None) == status
    assert (lib.fssim_last_error() != b"") == (status != 0)


def backward(**kw):
    return fill(BackwardArgs(kind=1, B=2, T=64, C=32, residual_scale=1.0, r=SOME, branch=SOME, dr=SOME, dz=SOME,
                             stats=SOME, dx=SOME, dweight=Channels(SOME, 0, 0)), kw)


@pytest.mark.parametrize("kw,status", [
    (dict(y_dtype=5), DTYPE), (dict(kind=0), ARGUMENT), (dict(branch_kind=7), ARGUMENT), (dict(C=-5), SHAPE),
    (dict(r=None), NULLPTR), (dict(dz=None, dr=None), NULLPTR), (dict(stats=None), NULLPTR),
    (dict(stats=SOME + 4), ARGUMENT), (dict(branch_kind=1), NULLPTR), (dict(branch=None, dbranch=SOME), NULLPTR),
    (dict(branch=None, dgate=Channels(SOME, 0, 0)), NULLPTR), (dict(dx=SOME + 2), ARGUMENT),
    (dict(dscale=Channels(SOME, 4, 0)), DTYPE), (dict(dgate=Channels(SOME + 2, 0, 0)), ARGUMENT),
    (dict(scale=Channels(SOME + 1, 1, 1)), ARGUMENT),
    (dict(), WORKSPACE), (dict(workspace=SOME, workspace_bytes=8), WORKSPACE),
    (dict(workspace=SOME + 8, workspace_bytes=1 << 30), WORKSPACE),
    (dict(B=0), 0), (dict(dx=None, dweight=Channels()), 0),
])
def test_c_backward_refusals(lib, kw, status):
    assert lib.fssim_block_norm_backward(ctypes.byref(backward(**kw)), None) == status


def test_c_null(lib):
    assert lib.fssim_block_norm_forward(None, None) == NULLPTR
    assert lib.fssim_block_norm_backward(None, None) == NULLPTR
    assert lib.fssim_block_norm_backward_workspace_bytes(None) == 0


def test_c_workspace(lib):
    f = lambda **kw: lib.fssim_block_norm_backward_workspace_bytes(ctypes.byref(backward(**kw)))  # noqa: E731
    assert f() >= 2 * 32 * 4
    assert f(dgate=Channels(SOME, 0, 0)) > f()
    assert f(dweight=Channels()) == 0 and f(B=0) == 0 and f(C=0) == 0
    # sums of bounded numbers of rows: the workspace stays a fraction of the rows themselves
    assert f(T=1 << 24) <= (2 << 24) * 32 * 4 // 16

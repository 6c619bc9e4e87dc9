"""Host-side behaviour of the training-step operators (runs without a GPU): the checks of
arguments, the module, and the C entry points' refusals, none of which reaches the GPU."""

import ctypes
import os

import pytest
import torch

import fussim_b200 as fb

LIB = os.path.join(os.path.dirname(os.path.abspath(fb.__file__)), "libfussim_b200.so")


def test_public_names():
    for name in ("group_norm_act", "GroupNormAct", "grad_norm", "clip_grad_norm", "clip_grad_norm_"):
        assert name in fb.__all__ and hasattr(fb, name)


# ---- group_norm_act ----
X = torch.zeros(2, 12, 4, 5)


@pytest.mark.parametrize("args,kwargs,match", [
    ((torch.zeros(2, 12, 4), 3), {}, "4D"),
    ((X, 5), {}, "divide into the groups"),
    ((X, 0), {}, "divide into the groups"),
    ((X, -3), {}, "divide into the groups"),
    ((torch.zeros(2, 0, 4, 5), 1), {}, "divide into the groups"),
    ((X, 3), dict(activation="tanh"), "activation"),
    ((X, 3), dict(eps=-1e-5), "eps"),
    ((X, 3), dict(eps=float("nan")), "eps"),
    ((X.double(), 3), {}, "float32, float16 or bfloat16"),
    ((X, 3, torch.ones(11)), {}, "weight must have shape"),
    ((X, 3, None, torch.ones(1, 12)), {}, "bias must have shape"),
    ((X, 3, torch.ones(12).long()), {}, "weight must be"),
    ((X, 3, torch.ones(12), torch.ones(12).half()), {}, "same dtype"),
])
def test_group_norm_refusals(args, kwargs, match):
    with pytest.raises(ValueError, match=match):
        fb.group_norm_act(*args, **kwargs)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-CUDA error path")
def test_operators_require_cuda():
    with pytest.raises(RuntimeError, match="CUDA"):
        fb.group_norm_act(X, 3)
    for call in (fb.grad_norm, lambda g: fb.clip_grad_norm(g, 1.0)):
        for grads in ([], [X]):
            with pytest.raises(RuntimeError, match="CUDA"):
                call(grads)
    with pytest.raises(RuntimeError, match="CUDA"):
        fb.clip_grad_norm_([], 1.0)


def test_group_norm_module():
    m = fb.GroupNormAct(4, 12, eps=1e-6, activation="relu")
    ref = torch.nn.GroupNorm(4, 12)
    assert {k: v.shape for k, v in m.state_dict().items()} == \
        {k: v.shape for k, v in ref.state_dict().items()}
    assert torch.equal(m.weight, ref.weight) and torch.equal(m.bias, ref.bias)
    m.load_state_dict(ref.state_dict())
    assert "4, 12, eps=1e-06, affine=True, activation='relu'" in repr(m)
    bare = fb.GroupNormAct(4, 12, affine=False, activation=None)
    assert bare.weight is None and bare.bias is None and not list(bare.parameters())
    with pytest.raises(ValueError, match="divide into the groups"):
        fb.GroupNormAct(5, 12)
    with pytest.raises(ValueError, match="activation"):
        fb.GroupNormAct(4, 12, activation="gelu")


# ---- gradient norm and clipping ----
@pytest.mark.parametrize("value", [-1.0, float("nan")])
def test_max_norm_refusals(value):
    for call in (lambda: fb.clip_grad_norm([X], value), lambda: fb.clip_grad_norm_([X], value)):
        with pytest.raises(ValueError, match="max_norm"):
            call()


def test_signatures_follow_torch():
    with pytest.raises(ValueError, match="norm_type"):
        fb.clip_grad_norm_([X], 1.0, float("inf"))
    with pytest.raises(TypeError):
        fb.clip_grad_norm([X], 1.0, None, True)
    m = fb.GroupNormAct(4, 12, 1e-5, True, "cpu", torch.bfloat16)  # torch.nn.GroupNorm's order
    assert m.weight.dtype == torch.bfloat16 and m.activation == "silu"


def test_gradient_list_refusals():
    with pytest.raises(TypeError, match="must be tensors"):
        fb.grad_norm([X, 1.0])
    with pytest.raises(TypeError, match="must be tensors"):
        fb.clip_grad_norm_([{"params": [X]}], 1.0)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        fb.grad_norm([X, X.double()])
    with pytest.raises(ValueError, match="dense"):
        fb.grad_norm([X[0, 0].to_sparse()])
    with pytest.raises(RuntimeError, match="one device"):
        fb.grad_norm([X, X.to("meta")])
    with pytest.raises(ValueError, match="a tensor for each gradient"):
        fb.clip_grad_norm([X, X], 1.0, out=[X])


# ---- the C entry points ----
class ForwardArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("activation", ctypes.c_int32), ("N", ctypes.c_int64), ("P", ctypes.c_int64),
                ("C", ctypes.c_int64), ("groups", ctypes.c_int64), ("eps", ctypes.c_float),
                ("x", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("y", ctypes.c_void_p), ("mean", ctypes.c_void_p), ("rstd", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


class BackwardArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("activation", ctypes.c_int32), ("N", ctypes.c_int64), ("P", ctypes.c_int64),
                ("C", ctypes.c_int64), ("groups", ctypes.c_int64), ("x", ctypes.c_void_p),
                ("dy", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("mean", ctypes.c_void_p), ("rstd", ctypes.c_void_p), ("dx", ctypes.c_void_p),
                ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


class ClipArgs(ctypes.Structure):
    _fields_ = [("count", ctypes.c_int64), ("grads", ctypes.POINTER(ctypes.c_void_p)),
                ("sizes", ctypes.POINTER(ctypes.c_int64)),
                ("dtypes", ctypes.POINTER(ctypes.c_int32)),
                ("outs", ctypes.POINTER(ctypes.c_void_p)),
                ("out_dtypes", ctypes.POINTER(ctypes.c_int32)), ("max_norm", ctypes.c_float),
                ("norm", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_size_t)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.fssim_last_error.restype = ctypes.c_char_p
    for f in ("fssim_group_norm_forward_workspace_bytes", "fssim_group_norm_backward_workspace_bytes",
              "fssim_grad_clip_workspace_bytes"):
        getattr(lib, f).restype = ctypes.c_size_t
    for f in ("fssim_group_norm_forward", "fssim_group_norm_backward", "fssim_grad_norm",
              "fssim_grad_clip"):
        getattr(lib, f).argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    return lib


SHAPE, DTYPE, NULLPTR, WORKSPACE, ARGUMENT = 2, 3, 4, 5, 7
SOME = 1 << 20  # a pointer that no refused call follows


def _forward(**kw):
    a = ForwardArgs(dtype=0, weight_dtype=0, activation=1, N=2, P=1 << 20, C=32, groups=4, eps=1e-5,
                    x=SOME, y=SOME)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=3), DTYPE), (dict(weight_dtype=-1), DTYPE), (dict(activation=3), ARGUMENT),
    (dict(N=-1), SHAPE), (dict(P=-1), SHAPE), (dict(groups=5), SHAPE), (dict(groups=0), SHAPE),
    (dict(C=0), SHAPE), (dict(C=1 << 24, groups=1), SHAPE), (dict(N=1 << 31), SHAPE),
    (dict(N=1 << 30, P=1 << 40), SHAPE), (dict(eps=-1.0), ARGUMENT),
    (dict(eps=float("nan")), ARGUMENT), (dict(mean=SOME), NULLPTR), (dict(x=None), NULLPTR),
    (dict(y=None), NULLPTR), (dict(x=SOME + 2), ARGUMENT), (dict(), WORKSPACE),
    (dict(workspace=SOME, workspace_bytes=8), WORKSPACE),
    (dict(workspace=SOME + 8, workspace_bytes=1 << 30), WORKSPACE),
    (dict(N=0), 0), (dict(P=0), 0),
])
def test_c_forward_refusals(lib, kw, status):
    assert lib.fssim_group_norm_forward(ctypes.byref(_forward(**kw)), None) == status
    assert (lib.fssim_last_error() != b"") == (status != 0)


def _backward(**kw):
    a = BackwardArgs(dtype=1, weight_dtype=0, activation=1, N=2, P=1 << 20, C=32, groups=4, x=SOME,
                     dy=SOME, mean=SOME, rstd=SOME, dx=SOME)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), DTYPE), (dict(activation=-1), ARGUMENT), (dict(groups=3), SHAPE),
    (dict(x=None), NULLPTR), (dict(dy=None), NULLPTR), (dict(mean=None), NULLPTR),
    (dict(dx=SOME + 1), ARGUMENT), (dict(), WORKSPACE), (dict(N=0), 0), (dict(dx=None), 0),
])
def test_c_backward_refusals(lib, kw, status):
    assert lib.fssim_group_norm_backward(ctypes.byref(_backward(**kw)), None) == status


def test_c_workspace_sizes(lib):
    fwd, bwd = lib.fssim_group_norm_forward_workspace_bytes, lib.fssim_group_norm_backward_workspace_bytes
    assert fwd(ctypes.byref(_forward())) > 0
    assert bwd(ctypes.byref(_backward())) >= 2 * 32 * 8
    for f, make in ((fwd, _forward), (bwd, _backward)):
        for kw in (dict(N=0), dict(P=0), dict(groups=0), dict(groups=5), dict(N=-1)):
            assert f(ctypes.byref(make(**kw))) == 0
        assert f(None) == 0


def _clip(sizes, n=None, dtypes=None, out_dtypes=None, grads=None, outs=None, **kw):
    n = len(sizes) if n is None else n
    a = ClipArgs(count=n, max_norm=1.0, norm=SOME, workspace=SOME, workspace_bytes=1 << 30)
    k = max(1, len(sizes))
    a.sizes = (ctypes.c_int64 * k)(*sizes)
    a.dtypes = (ctypes.c_int32 * k)(*(dtypes or [0] * len(sizes)))
    a.out_dtypes = (ctypes.c_int32 * k)(*(out_dtypes or dtypes or [0] * len(sizes)))
    a.grads = (ctypes.c_void_p * k)(*(grads or [SOME] * len(sizes)))
    a.outs = (ctypes.c_void_p * k)(*(outs or [SOME] * len(sizes)))
    for key, v in kw.items():
        setattr(a, key, v)
    return a


@pytest.mark.parametrize("make,status", [
    (lambda: _clip([4], n=-1), SHAPE), (lambda: _clip([-4]), SHAPE),
    (lambda: _clip([1 << 61]), SHAPE), (lambda: _clip([4], dtypes=[5]), DTYPE),
    (lambda: _clip([4], dtypes=[1], out_dtypes=[2]), DTYPE),
    (lambda: _clip([4], dtypes=[0], out_dtypes=[1]), DTYPE),
    (lambda: _clip([4], grads=[None]), NULLPTR), (lambda: _clip([4], outs=[None]), NULLPTR),
    (lambda: _clip([4], grads=[SOME + 2]), ARGUMENT), (lambda: _clip([4], norm=None), NULLPTR),
    (lambda: _clip([4], max_norm=-1.0), ARGUMENT),
    (lambda: _clip([4], dtypes=[1], out_dtypes=[0]), ARGUMENT),  # in place with another type
    (lambda: _clip([4], max_norm=float("nan")), ARGUMENT),
    (lambda: _clip([4], workspace=None), WORKSPACE),
    (lambda: _clip([4], workspace_bytes=4), WORKSPACE),
    (lambda: _clip([4], workspace=SOME + 4), WORKSPACE),
])
def test_c_clip_refusals(lib, make, status):
    assert lib.fssim_grad_clip(ctypes.byref(make()), None) == status


def test_c_clip_workspace(lib):
    f = lib.fssim_grad_clip_workspace_bytes
    assert f(ctypes.byref(_clip([]))) == 0 and f(None) == 0
    assert f(ctypes.byref(_clip([0, 0]))) == 0
    # a partial sum for each CTA, a bounded number for any size, and their sum
    assert f(ctypes.byref(_clip([1, 0, 2049]))) == 4 * 8
    most = f(ctypes.byref(_clip([1 << 40])))
    assert 148 * 8 <= most <= 1 << 16
    assert most < f(ctypes.byref(_clip([1 << 30] * 2000))) <= 3 * most  # three tables

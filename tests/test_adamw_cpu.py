"""Host-side behaviour of the AdamW step (runs without a GPU): checks of arguments, and the C
entry point's refusals, none of which reaches the GPU."""

import ctypes
import os

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import fussim_b200 as fb

LIB = os.path.join(os.path.dirname(os.path.abspath(fb.__file__)), "libfussim_b200.so")
F8 = torch.float8_e4m3fn


def call(n=1, shape=(3, 5), dtype=torch.float32, gdtype=None, moment=torch.float32, **kw):
    """adamw_step_ of n tensors of a kind; keyword arguments replace what is passed."""
    args = dict(params=[torch.zeros(shape, dtype=dtype) for _ in range(n)],
                grads=[torch.zeros(shape, dtype=gdtype or dtype) for _ in range(n)],
                exp_avgs=[torch.zeros(shape, dtype=moment) for _ in range(n)],
                exp_avg_sqs=[torch.zeros(shape, dtype=moment) for _ in range(n)], step=1, lr=1e-3)
    args.update(kw)
    return fb.adamw_step_(**args)


Z = torch.zeros(3, 5)


def test_public_name():
    assert "adamw_step_" in fb.__all__


@pytest.mark.parametrize("kw,match", [
    (dict(grads=[]), "a tensor for each parameter"),
    (dict(exp_avgs=[Z, Z]), "a tensor for each parameter"),
    (dict(exp_avg_sqs=[]), "a tensor for each parameter"),
    (dict(copies=[]), "a tensor for each parameter"),
    (dict(betas=(1.0, 0.9)), "betas"),
    (dict(betas=(0.9, -0.1)), "betas"),
    (dict(betas=(float("nan"), 0.9)), "betas"),
    (dict(eps=-1e-8), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(weight_decay=-1.0), "weight_decay"),
    (dict(lr=-1.0), "lr"),
    (dict(lr=float("nan")), "lr"),
    (dict(step=0), "step"),
    (dict(step=-3), "step"),
    (dict(step=1.5), "step"),
    (dict(step=float("nan")), "step"),
    (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=float("nan")), "max_norm"),
    (dict(norm=torch.zeros(())), "norm goes with max_norm"),
    (dict(seed=-1), "seed"),
    (dict(seed=1 << 32), "seed"),
    (dict(dtype=torch.float64), "float32, float16 or bfloat16"),
    (dict(dtype=torch.bfloat16, gdtype=torch.float16), "parameter's type or float32"),
    (dict(gdtype=torch.float64), "parameter's type or float32"),
    (dict(params=[torch.zeros(3, 10)[:, ::2]]), "fill its memory"),
    (dict(params=[torch.zeros(1, 5).expand(3, 5)]), "fill its memory"),
    (dict(params=[torch.zeros(3, 5, dtype=torch.complex64).conj().imag]), "fill its memory"),
    (dict(grads=[Z.to_sparse()]), "dense"),
    (dict(grads=[torch.zeros(5, 3)]), "must have shape"),
    (dict(moment=torch.bfloat16), "float32"),
    (dict(exp_avg_sqs=[Z.half()]), "float32"),
    (dict(exp_avgs=[torch.zeros(15)]), "must have shape"),
    (dict(exp_avgs=[torch.zeros(5, 3).t()]), "parameter's strides"),
    (dict(moment=F8), "need their scales"),
    (dict(scales=[torch.zeros(1, 2)]), "scales go with moments"),
    (dict(moment=F8, scales=[torch.zeros(2, 2)]), r"\(1, 2\)"),
    (dict(moment=F8, scales=[torch.zeros(1, 2).half()]), r"\(1, 2\)"),
    (dict(moment=F8, scales=[torch.zeros(2, 1).t()], shape=(300,)), r"\(2, 2\)"),
    (dict(moment=F8, scales=[torch.zeros(2, 2).t()], shape=(300,)), "contiguous"),
    (dict(n=2, moment=F8, exp_avgs=[Z, Z.to(F8)], scales=[torch.zeros(1, 2)] * 2), "scales go with"),
    (dict(n=2, moment=F8, exp_avgs=[Z.to(F8), Z], scales=[torch.zeros(1, 2)] * 2), "as the first"),
    (dict(copies=[Z]), "of a float32 parameter"),
    (dict(dtype=torch.bfloat16, copies=[Z.bfloat16()]), "of a float32 parameter"),
    (dict(copies=[torch.zeros(5, 3).half().t()]), "parameter's strides"),
])
def test_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(params=[Z, 1.0]), "must be tensors"),
    (dict(step=None), "adamw_step_"),
    (dict(lr="fast"), "adamw_step_"),
])
def test_type_refusals(kw, match):
    with pytest.raises(TypeError, match=match):
        call(**({"n": 2} if "params" in kw else {}), **kw)


def test_devices():
    with pytest.raises(RuntimeError, match="device"):
        call(grads=[Z.to("meta")])
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA is not available"):
            call()
        with pytest.raises(RuntimeError, match="CUDA is not available"):
            call(n=0)


def test_tracing():
    f = lambda p: call(params=[p], max_norm=1.0)  # noqa: E731
    with pytest.raises(RuntimeError, match="adamw_step_ cannot be traced"):
        torch.jit.trace(f, Z.clone())
    with pytest.raises(RuntimeError, match="adamw_step_ cannot be traced"):
        make_fx(f)(Z.clone())


# ---- the C entry point ----
P, I64, I32, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_double


class Args(ctypes.Structure):
    _fields_ = [("count", I64), ("params", P), ("grads", P), ("exp_avgs", P), ("exp_avg_sqs", P),
                ("scales", P), ("copies", P), ("sizes", P), ("dtypes", P), ("grad_dtypes", P),
                ("copy_dtypes", P), ("state_bits", I32), ("maximize", I32), ("seed", ctypes.c_uint32),
                ("step", I64), ("step_at", P), ("lr", F64), ("lr_at", P), ("beta1", F64),
                ("beta2", F64), ("eps", F64), ("weight_decay", F64), ("norm", P), ("max_norm", F64)]


SHAPE, DTYPE, NULLPTR, ARGUMENT = 2, 3, 4, 7
SOME = 1 << 20  # a pointer that no refused call follows


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(LIB)
    lib.fssim_last_error.restype = ctypes.c_char_p
    lib.fssim_adamw_step.argtypes = [P, P]
    return lib


def make(sizes=(4,), keep=[], **kw):
    """Arguments; those of the tensors' arrays are given by one value for all tensors."""
    n = len(sizes)
    a = Args(count=n, state_bits=32, step=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8)

    def array(kind, values):
        keep.append((kind * max(1, n))(*values))
        return ctypes.cast(keep[-1], P)

    a.sizes = array(I64, sizes)
    for k in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
        setattr(a, k, array(P, [kw.pop(k, SOME)] * n))
    for k in ("dtypes", "grad_dtypes"):
        setattr(a, k, array(I32, [kw.pop(k, 0)] * n))
    for k, kind in (("scales", P), ("copies", P), ("copy_dtypes", I32)):
        if k in kw:
            setattr(a, k, array(kind, [kw.pop(k)] * n))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(count=-1), SHAPE), (dict(sizes=(-4,)), SHAPE), (dict(sizes=(1 << 61,)), SHAPE),
    (dict(state_bits=16), ARGUMENT), (dict(beta1=1.0), ARGUMENT), (dict(beta2=-0.5), ARGUMENT),
    (dict(beta2=float("nan")), ARGUMENT), (dict(eps=-1.0), ARGUMENT), (dict(lr=-1.0), ARGUMENT),
    (dict(lr=float("inf")), ARGUMENT), (dict(weight_decay=float("nan")), ARGUMENT),
    (dict(step=0), ARGUMENT), (dict(norm=SOME, max_norm=-1.0), ARGUMENT),
    (dict(norm=SOME + 2), ARGUMENT), (dict(step_at=SOME + 1), ARGUMENT), (dict(lr_at=SOME + 3), ARGUMENT),
    (dict(dtypes=3), DTYPE), (dict(dtypes=1, grad_dtypes=2), DTYPE), (dict(grad_dtypes=-1), DTYPE),
    (dict(copies=SOME, copy_dtypes=0), DTYPE),
    (dict(dtypes=2, grad_dtypes=2, copies=SOME, copy_dtypes=2), DTYPE),
    (dict(state_bits=8), NULLPTR), (dict(state_bits=8, scales=None), NULLPTR),
    (dict(state_bits=8, scales=SOME + 2), ARGUMENT),
    (dict(copies=SOME), NULLPTR), (dict(copies=None, copy_dtypes=1), NULLPTR),
    (dict(copies=SOME + 1, copy_dtypes=1), ARGUMENT),
    (dict(params=None), NULLPTR), (dict(grads=None), NULLPTR), (dict(exp_avgs=None), NULLPTR),
    (dict(exp_avg_sqs=None), NULLPTR), (dict(params=SOME + 2), ARGUMENT), (dict(grads=SOME + 1), ARGUMENT),
    (dict(exp_avgs=SOME + 2), ARGUMENT), (dict(exp_avg_sqs=SOME + 1), ARGUMENT),
    (dict(sizes=()), 0), (dict(sizes=(0, 0), params=None), 0),
])
def test_c_refusals(lib, kw, status):
    assert lib.fssim_adamw_step(ctypes.byref(make(**kw)), None) == status
    assert (lib.fssim_last_error() != b"") == (status != 0)


def test_c_null(lib):
    assert lib.fssim_adamw_step(None, None) == NULLPTR
    a = make()
    a.sizes = None
    assert lib.fssim_adamw_step(ctypes.byref(a), None) == NULLPTR


# ---- the class ----
@pytest.mark.parametrize("kw,match", [
    (dict(state_bits=16), "state_bits"), (dict(lr=-1.0), "lr"), (dict(lr=float("nan")), "lr"),
    (dict(lr=torch.tensor(1e-3)), "capturable"), (dict(betas=(1.0, 0.9)), "first of betas"),
    (dict(betas=(0.9, 1.5)), "second of betas"), (dict(eps=-1.0), "eps"), (dict(weight_decay=-0.1), "weight_decay"),
    (dict(max_norm=-1.0), "max_norm"), (dict(max_norm=float("nan")), "max_norm"), (dict(seed=-1), "seed"),
    (dict(seed=1 << 32), "seed"),
])
def test_optimizer_refusals(kw, match):
    with pytest.raises(ValueError, match=match):
        fb.AdamW([torch.nn.Parameter(Z.clone())], **kw)


def test_moments():
    p = torch.zeros(3, 100, 2, 2).to(memory_format=torch.channels_last)
    for bits, dtype in ((32, torch.float32), (8, F8)):
        first, second, scales = fb.adamw_moments(p.half(), bits)
        for t in (first, second):
            assert t.dtype == dtype and t.shape == p.shape and t.stride() == p.stride() and not t.float().any()
        assert scales is None if bits == 32 else scales.shape == (5, 2)
    with pytest.raises(ValueError, match="bits"):
        fb.adamw_moments(p, 4)

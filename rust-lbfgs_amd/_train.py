"""ctypes declarations of include/lbfgs_train.h, and what losses.py and directions.py share: the loaders of
liblbfgs_train.so and of the extension that makes their ordinary calls, and the checks of torch tensors.

The operators take tensors of the GPU and enqueue HIP kernels on the tensors' device and its current stream, as torch's own
operators do.  There is no CPU fallback: without the built library, or with tensors elsewhere, they raise.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import operator
import os

import torch  # before the library: it has to bind to torch's HIP runtime
from torch.autograd import forward_ad

from . import _build, _ffi
from .api import _raise

ABI_VERSION = 1  # LBFGS_TRAIN_ABI_VERSION of the header these declarations were written against
DTYPES = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
WIDE_GRAD = 256  # LBFGS_TRAIN_WIDE_GRAD


class Rows(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("targets", C.c_void_p), ("dtype", C.c_int32), ("_pad", C.c_int32), ("outer", C.c_int64),
                ("inner", C.c_int64), ("vocab", C.c_int64), ("outer_stride", C.c_int64), ("inner_stride", C.c_int64),
                ("ignore_index", C.c_int64)]


class Sequences(C.Structure):
    _fields_ = [("offsets", C.c_void_p), ("mask", C.c_void_p), ("offset_bits", C.c_int32), ("dtype", C.c_int32), ("tokens", C.c_int64),
                ("count", C.c_int64)]


_vp, _i, _i64, _u64, _d = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_double
SIGNATURES = {  # every symbol the header declares
    "lbfgs_train_abi_version": (C.c_int, []),
    "lbfgs_train_build_id": (C.c_char_p, []),
    "lbfgs_train_last_error": (C.c_char_p, []),
    "lbfgs_train_token_logprobs_workspace": (_u64, [_i, _i64, _i64]),
    "lbfgs_train_token_logprobs": (C.c_int, [C.POINTER(Rows), _d, _vp, _vp, _vp, _u64, _vp]),
    "lbfgs_train_token_logprobs_grad": (C.c_int, [C.POINTER(Rows), _d, _vp, _vp, _vp, _vp]),
    "lbfgs_train_sequences_workspace": (_u64, [_i64, _i64]),
    "lbfgs_train_preference": (C.c_int, [C.POINTER(Sequences), _vp, _vp, _d, _d, _i, _i, _vp, _vp, _vp, _vp, _u64, _vp]),
    "lbfgs_train_policy": (C.c_int, [C.POINTER(Sequences), _vp, _vp, _vp, _vp, _i, _d, _d, _d, _i, _vp, _vp, _vp, _vp, _vp, _u64, _vp]),
    "lbfgs_train_orthogonalize_workspace": (_u64, [_i, _i64, _i64, _i64]),
    "lbfgs_train_orthogonalize": (C.c_int, [_i, _i64, _i64, _i64, _vp, _vp, _i, _d, _d, _d, _vp, _u64, _vp]),
}

_LIB = None


def load():
    """Load liblbfgs_train.so.  Raises if it is not built, or built from other sources than the checked-out ones."""
    global _LIB
    if _LIB is not None:
        return _LIB
    libdir = os.environ.get("LBFGS_HIP_LIB_DIR", _ffi.HERE)
    path = os.path.join(libdir, os.path.basename(_build.TRAIN_LIB))
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: the HIP extension is not built (python -c 'import rust_lbfgs_amd as r; r.build()'); "
                          "this package has no CPU fallback")
    if os.path.realpath(libdir) == os.path.realpath(_ffi.HERE) and os.environ.get("LBFGS_HIP_ALLOW_STALE") != "1":
        have, want = _build.embedded_id(path, "LBFGS_TRAIN_BUILD_ID"), _build.train_build_id()
        if have != want:
            raise ImportError(f"{path} carries build id {have}, the checked-out sources hash to {want}: rebuild "
                              "(python -c 'import rust_lbfgs_amd as r; r.build()'), or set LBFGS_HIP_ALLOW_STALE=1 to load it anyway")
    lib = C.CDLL(path, mode=C.RTLD_LOCAL)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    if lib.lbfgs_train_abi_version() != ABI_VERSION:
        raise ImportError(f"{path} has ABI version {lib.lbfgs_train_abi_version()}, this package was written against {ABI_VERSION}: rebuild")
    _LIB = lib
    return lib


_CALLS = None


def calls():
    """The extension liblbfgs_train_calls.so: a function for each operator that does the whole of an ordinary call -- tensors that are dense,
    of the right types and shapes and on the current device -- and returns its results, or the status of a refused one, or None: it has done
    nothing, and the operator's own checks follow.  Raises if it is not built, or built from other sources or for another torch."""
    global _CALLS
    if _CALLS is not None:
        return _CALLS
    lib, path = load(), _build.CALLS_LIB
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: the extension is not built (python -c 'import rust_lbfgs_amd as r; r.build()')")
    have, want = _build.embedded_id(path, "LBFGS_TRAIN_CALLS_BUILD_ID"), _build.calls_build_id()
    if have != want and os.environ.get("LBFGS_HIP_ALLOW_STALE") != "1":
        raise ImportError(f"{path} carries build id {have}, the checked-out sources and this torch hash to {want}: rebuild "
                          "(python -c 'import rust_lbfgs_amd as r; r.build()'), or set LBFGS_HIP_ALLOW_STALE=1 to load it anyway")
    loader = importlib.machinery.ExtensionFileLoader("liblbfgs_train_calls", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(loader.name, loader))
    loader.exec_module(module)
    functions = [C.cast(getattr(lib, "lbfgs_train_" + name), C.c_void_p).value for name in (
        "token_logprobs_workspace", "token_logprobs", "token_logprobs_grad", "sequences_workspace", "preference", "policy", "orthogonalize_workspace", "orthogonalize")]
    # (the current stream of a device, as a number; on a build of torch without a GPU there is none to ask for, nor a tensor that would need it)
    module.bind(*functions, getattr(torch._C, "_cuda_getCurrentRawStream", None))
    _CALLS = module
    return module


def check(rc):
    if rc != 0:
        _raise(rc, load().lbfgs_train_last_error().decode())


def results(done):
    """What a native call left: its results, or the status of a refused one."""
    if type(done) is not tuple:
        check(done)
    return done


def wide(dtype):
    """What sums and losses of this element type come out in."""
    return torch.float64 if dtype == torch.float64 else torch.float32


def floating(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be float64, float32, bfloat16 or float16, not {t.dtype}")
    plain(name, t)


def plain(name, t):
    """`t` is what its memory holds, and nothing else: the kernels see no more of it."""
    if t.is_neg():
        raise TypeError(f"{name} is a view whose sign is still to be applied: resolve_neg() first")
    if forward_ad.unpack_dual(t).tangent is not None:
        raise TypeError(f"{name} carries a forward-mode derivative, which the operators do not have: the result's would be lost")


def on_gpu(name, t, others=()):
    """The one device of these tensors, (name, tensor or None) each."""
    dev = t.device
    if dev.type != "cuda":
        raise TypeError(f"{name} is on {dev}: the operators run on the GPU, there is no CPU fallback")
    for other, o in others:
        if o is not None and o.device != dev:
            raise ValueError(f"{other} is on {o.device}, {name} on {dev}")
    return dev


def like(name, t, what, dtype, shape):
    """`t` has this element type and shape."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} as {what} asks for, not {t.dtype}")
    plain(name, t)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)} as {what} asks for, not {tuple(t.shape)}")


def whole(name, v, bits):
    """`v` as a number that the C-ABI's signed integer of so many bits holds: ctypes would keep the low bits of any other."""
    v = operator.index(v)
    if not -(1 << bits - 1) <= v < 1 << bits - 1:
        raise ValueError(f"{name} must fit {bits} bits, {v} does not")
    return v


def ptr(t):
    return None if t is None else t.data_ptr()


def enqueue(function, device, *arguments):
    """`function(*arguments, stream)` with the tensors' device as the current one, on its current stream."""
    if torch._C._cuda_getDevice() == device.index:  # (what torch.cuda.current_device() asks, once torch has started)
        rc = function(*arguments, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = function(*arguments, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != 0:
        check(rc)


def refuse_capture(what, instead):
    """Autograd inside a stream capture goes through the leaf's accumulation node, and where an eager graph of the same leaf keeps
    that node alive on another stream, torch ends the process.  The call cannot see that, so it is refused."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} with a gradient to come cannot be captured into a graph: capture {instead}, which need no autograd")

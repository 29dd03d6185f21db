"""ctypes binding of libf16acc_ops.so (the C ABI in include/f16acc_ops.h).

There is no fallback: if the library is missing, importing this module raises.
"""

import ctypes
import os

import torch

from .build import LIB_OPS

if not os.path.exists(LIB_OPS):
    raise ImportError(f"{LIB_OPS} is not built; run `python f16acc_amd/build.py` (needs hipcc for gfx950)")

_dll = ctypes.CDLL(LIB_OPS)

_i64, _vp, _int, _f32, _size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t

# name -> argument types; every function but the last three returns an error code
_SIGNATURES = {
    "f16acc_quant_rows": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64, _vp],
    "f16acc_quant_both": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64] * 2 + [_vp],
    "f16acc_quant_weight": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64, _vp, _i64, _vp],
    "f16acc_pack8": [_vp, _vp] + [_i64] * 5 + [_vp],
    "f16acc_mm_fp8": [_vp, _i64, _vp, _i64, _i64] * 2 + [_int, _vp, _vp] + [_i64] * 5 + [_int] * 3 + [_vp, _size, _vp],
    "f16acc_linear_fp8": [_vp, _int, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp] + [_i64] * 3 + [_vp, _size, _vp],
    "f16acc_route": [_vp, _int] + [_i64] * 3 + [_int] * 3 + [_vp] + [_int] * 3 + [_f32, _vp, _vp, _vp],
    "f16acc_route_grad": [_vp, _int] + [_i64] * 3 + [_int] * 4 + [_f32, _vp, _vp, _i64, _i64, _vp, _vp],
    "f16acc_experts": [_vp, _int] + [_i64] * 3 + [_vp, _i64, _i64, _vp, _int, _int] + [_i64] * 2
                      + [_vp] + [_i64] * 3 + [_vp] + [_i64] * 4 + [_vp] + [_i64] * 2 + [_vp] + [_i64] * 3
                      + [_vp, _vp, _size, _vp],
    "f16acc_mm_fp8_workspace": [_i64] * 3 + [_int] * 3,
    "f16acc_linear_fp8_workspace": [_i64] * 3,
    "f16acc_experts_workspace": [_i64, _int, _int, _i64, _i64],
    "f16acc_ops_strerror": [_int],
    "f16acc_ops_abi_version": [],
}
EXPORTS = tuple(_SIGNATURES)  # the symbols include/f16acc_ops.h declares
ABI_VERSION = 1


def _bind(name):
    f = getattr(_dll, name)
    f.argtypes = _SIGNATURES[name]
    f.restype = _size if name.endswith("_workspace") else ctypes.c_char_p if name.endswith("strerror") else _int
    return f


(quant_rows, quant_both, quant_weight, pack8, mm_fp8, linear_fp8, route, route_grad, experts, mm_fp8_workspace,
 linear_fp8_workspace, experts_workspace, strerror, abi_version) = map(_bind, EXPORTS)

E_ARG, E_UNSUPPORTED, E_WORKSPACE = -1, -2, -3
TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
FP8 = torch.float8_e4m3fn
BLOCK = 128

if abi_version() != ABI_VERSION:
    raise ImportError(f"{LIB_OPS} has ABI version {abi_version()}, this package needs {ABI_VERSION}: rebuild it")


def call(f, dev, *args):
    """f(*args, stream) on `dev`'s current torch stream; raises RuntimeError for a failure."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return call(f, dev, *args)
    rc = f(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc != 0:
        raise RuntimeError(strerror(rc).decode())


def ptr(t):
    return None if t is None else t.data_ptr()


def up(v, m):
    return -(-v // m) * m


def blocks(v):
    return -(-v // BLOCK)


def on_gpu(name, *tensors):
    """The one GPU the given tensors (None: skipped) are on; ValueError otherwise."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda or (dev is not None and t.device != dev):
            raise ValueError(f"{name} needs tensors on one GPU")
        dev = t.device
    return dev

"""Binding of libf16acc_ops.so: its C ABI (include/f16acc_ops.h) through ctypes,
and `host`, the torch side of the operators (csrc/ops/torch_ops.cpp), which
fp4.py, fp8.py and moe.py call.

There is no fallback: if a library is missing, importing this module raises.
"""

import ctypes
import importlib.util
import os

import torch

from .build import LIB_OPS, OPS_TORCH

for _f in (LIB_OPS, OPS_TORCH):
    if not os.path.exists(_f):
        raise ImportError(f"{_f} is not built; run `python f16acc_amd/build.py` (needs hipcc for gfx950)")

_dll = ctypes.CDLL(LIB_OPS)

_i64, _vp, _int, _f32, _size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t

# name -> argument types
_SIGNATURES = {
    "f16acc_quant_rows": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64, _vp],
    "f16acc_quant_both": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64] * 2 + [_vp],
    "f16acc_quant_weight": [_vp, _int] + [_i64] * 4 + [_vp, _i64, _vp, _i64, _vp, _i64, _vp],
    "f16acc_pack8": [_vp, _vp] + [_i64] * 5 + [_vp],
    "f16acc_column_sums": [_vp, _int] + [_i64] * 4 + [_vp, _vp, _size, _vp],
    "f16acc_mm_fp8": [_vp, _i64, _vp, _i64, _i64] * 2 + [_int, _vp, _vp] + [_i64] * 5 + [_int] * 3 + [_vp, _size, _vp],
    "f16acc_linear_fp8": [_vp, _int, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp] + [_i64] * 3 + [_vp, _size, _vp],
    "f16acc_route": [_vp, _int] + [_i64] * 3 + [_int] * 3 + [_vp] + [_int] * 3 + [_f32, _vp, _vp, _vp],
    "f16acc_route_grad": [_vp, _int] + [_i64] * 3 + [_int] * 4 + [_f32, _vp, _vp, _i64, _i64, _vp, _vp],
    "f16acc_experts_any_rows": [_vp, _int] + [_i64] * 3 + [_int],
    "f16acc_experts": [_vp, _int] + [_i64] * 3 + [_vp, _i64, _i64, _vp, _int, _int] + [_i64] * 2
                      + [_vp] + [_i64] * 3 + [_vp] + [_i64] * 4 + [_vp] + [_i64] * 2 + [_vp] + [_i64] * 3
                      + [_vp, _vp, _size, _vp],
    "f16acc_column_sums_workspace": [_i64, _i64],
    "f16acc_mm_fp8_workspace": [_i64] * 3 + [_int] * 3,
    "f16acc_linear_fp8_workspace": [_i64] * 3 + [_vp, _i64],
    "f16acc_experts_workspace": [_i64, _int, _int, _i64, _i64],
    "f16acc_layer_any_rows": [_i64, _int, _i64, _i64],
    "f16acc_layer": [_vp, _int] + [_i64] * 3 + [_vp, _int, _i64, _i64] + [_int] * 3 + [_vp] + [_int] * 3 + [_f32]
                    + [_i64] * 2 + [_vp] + [_i64] * 3 + [_vp] + [_i64] * 4 + [_vp] + [_i64] * 2 + [_vp] + [_i64] * 3
                    + [_vp, _vp, _size, _vp],
    "f16acc_layer_workspace": [_i64, _int, _int, _i64, _i64],
    "f16acc_fp4_quant": [_vp, _vp, _int, _vp],
    "f16acc_fp4_transpose": [_vp, _i64, _i64] * 2 + [_i64] * 2 + [_vp, _i64, _vp, _i64, _i64, _vp],
    "f16acc_fp4_values": [_vp, _i64, _i64] * 2 + [_i64] * 2 + [_vp, _int, _vp],
    "f16acc_mm_fp4": ([_vp, _i64, _i64, _vp] + [_i64] * 3) * 2 + [_vp, _vp] + [_i64] * 5 + [_int] * 3 + [_vp, _size, _vp],
    "f16acc_linear_fp4": [_vp, _int, _i64, _i64, _vp, _i64, _vp, _i64, _i64, _vp, _vp] + [_i64] * 3 + [_vp, _size, _vp],
    "f16acc_linear_fp4_few": [_i64] * 4,
    "f16acc_mm_fp4_workspace": [_vp, _i64, _i64, _i64] * 2 + [_i64] * 3 + [_int] * 2,
    "f16acc_linear_fp4_workspace": [_i64] * 3 + [_vp, _i64],
    "f16acc_ops_strerror": [_int],
    "f16acc_ops_abi_version": [],
}


class Fp4Matrix(ctypes.Structure):
    """f16acc_fp4_matrix."""
    _fields_ = [("x", _vp), ("rows", _i64), ("cols", _i64), ("sr", _i64), ("sc", _i64), ("q", _vp), ("ldq", _i64), ("s", _vp),
                ("s_row", _i64), ("s_quad", _i64), ("qt", _vp), ("ldqt", _i64), ("st", _vp), ("st_row", _i64),
                ("st_quad", _i64)]


EXPORTS = tuple(_SIGNATURES)  # the symbols include/f16acc_ops.h declares
ABI_VERSION = 1
E_ARG, E_UNSUPPORTED, E_WORKSPACE = -1, -2, -3


def _bind(name):
    f = getattr(_dll, name)
    f.argtypes = _SIGNATURES[name]
    f.restype = _size if name.endswith("_workspace") else ctypes.c_char_p if name.endswith("strerror") else _int
    return f


(quant_rows, quant_both, quant_weight, pack8, column_sums, mm_fp8, linear_fp8, route, route_grad, experts_any_rows,
 experts, column_sums_workspace, mm_fp8_workspace, linear_fp8_workspace, experts_workspace,
 layer_any_rows, layer, layer_workspace, fp4_quant, fp4_transpose, fp4_values, mm_fp4, linear_fp4, linear_fp4_few,
 mm_fp4_workspace, linear_fp4_workspace, strerror, abi_version) = map(_bind, EXPORTS)

if abi_version() != ABI_VERSION:
    raise ImportError(f"{LIB_OPS} has ABI version {abi_version()}, this package needs {ABI_VERSION}: rebuild it")


def _load_host(path=OPS_TORCH):
    spec = importlib.util.spec_from_file_location("f16acc_ops_torch", path)
    try:
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
    except ImportError as e:
        raise ImportError(f"{path} does not load with torch {torch.__version__} (built for another?): rebuild it") from e
    if mod.torch_version != torch.__version__.split("+")[0] or mod.abi_version != ABI_VERSION:
        raise ImportError(f"{path} was built for torch {mod.torch_version}, ABI {mod.abi_version}: rebuild it")
    return mod


host = _load_host()

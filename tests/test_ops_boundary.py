"""The operators' C ABI without a GPU: what the library exports, and what it
refuses before it launches anything."""

import ctypes
import os
import re

import pytest
import torch

from f16acc_amd import _ops, fp8, moe
from f16acc_amd.build import LIB_OPS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    src = open(os.path.join(ROOT, "include", "f16acc_ops.h")).read()
    names = sorted(set(re.findall(r"\b(f16acc_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", src, flags=re.S))))
    dll = ctypes.CDLL(LIB_OPS)
    assert names and all(hasattr(dll, n) for n in names)
    assert sorted(_ops.EXPORTS) == names
    assert _ops.abi_version() == _ops.ABI_VERSION


def test_every_argument_is_bound_with_its_c_type():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "f16acc_ops.h")).read(), flags=re.S)
    kinds = {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "size_t": ctypes.c_size_t}
    for name, args in re.findall(r"\b(f16acc_\w+)\s*\(([^)]*)\)", src):
        want = [] if args.strip() == "void" else [
            ctypes.c_void_p if "*" in a else kinds[a.split()[0]] for a in args.replace("const ", "").split(",")]
        assert _ops._SIGNATURES[name] == want, name


def test_mm_checks():
    def call(x=256, ldx=256, sx=256, sxm=1, sxk=1, w=256, ldw=256, sw=256, swn=1, swk=1, rows=0, c=256, M=4, N=4, K=256, t=0, tile=-1,
             splits=0):
        return _ops.mm_fp8(x, ldx, sx, sxm, sxk, w, ldw, sw, swn, swk, rows, None, c, N, 1, M, N, K, t, tile, splits, None, 0, None)

    assert call(M=-1) == call(K=-1) == call(t=3) == call(rows=2) == call(c=None) == call(x=None) == _ops.E_ARG
    assert call(sx=None) == call(swn=-1) == call(sxk=-1) == _ops.E_ARG
    assert call(ldx=250) == call(ldw=128) == call(x=8) == call(w=264) == _ops.E_UNSUPPORTED
    assert call(K=1 << 23, ldx=1 << 23, ldw=1 << 23) == _ops.E_UNSUPPORTED
    assert call(tile=6) == call(tile=-2) == call(splits=-1) == _ops.E_ARG
    assert call(splits=2) == _ops.E_WORKSPACE and _ops.mm_fp8_workspace(4, 4, 256, 0, -1, 2) >= 2 * 4 * 4 * 4
    assert call(M=0) == call(N=0) == 0


def test_quantisation_checks():
    assert _ops.quant_rows(None, 0, 2, 2, 2, 1, 256, 128, 256, 2, None) == _ops.E_ARG
    assert _ops.quant_rows(256, 5, 2, 2, 2, 1, 256, 128, 256, 2, None) == _ops.E_ARG
    assert _ops.quant_rows(256, 0, 2, 2, 2, 1, None, 128, 256, 2, None) == _ops.E_ARG
    assert _ops.quant_rows(256, 0, 2, 200, 200, 1, 256, 128, 256, 2, None) == _ops.E_UNSUPPORTED
    assert _ops.quant_rows(256, 0, 2, 2, 2, 1, 256, 100, 256, 2, None) == _ops.E_UNSUPPORTED
    assert _ops.quant_rows(256, 0, 0, 2, 2, 1, None, 0, None, 0, None) == 0
    assert _ops.quant_both(256, 0, 2, 2, 2, 1, None, 0, None, 0, None, 0, None, 0, None) == _ops.E_ARG
    assert _ops.quant_weight(256, 0, 2, 2, 2, 1, 256, 128, 256, 1, 264, 128, None) == _ops.E_UNSUPPORTED
    assert _ops.pack8(256, 256, 2, 20, 20, 1, 16, None) == _ops.E_ARG
    assert _ops.pack8(256, 256, 2, 20, 20, 1, 24, None) == _ops.E_UNSUPPORTED


def test_linear_and_workspace_checks():
    need = _ops.linear_fp8_workspace(100, 64, 300, 256, 304)
    assert need >= 100 * 384 + 100 * 3 * 4 and _ops.linear_fp8_workspace(0, 64, 300, 256, 304) == 0
    # K is no multiple of 16, or the rows are not aligned: room for a copy of the weight
    assert need >= _ops.linear_fp8_workspace(100, 64, 304, 256, 304) + 64 * 304
    assert _ops.linear_fp8_workspace(100, 64, 304, 264, 304) >= _ops.linear_fp8_workspace(100, 64, 304, 256, 304) + 64 * 304

    def call(ws=256, n=need, M=100, t=0, ldw=304, K=300, w=256):
        return _ops.linear_fp8(256, t, 300, 1, w, ldw, 256, 3, 1, None, 256, M, 64, K, ws, n, None)

    assert call(ws=None) == call(n=need - 1) == call(ws=128) == _ops.E_WORKSPACE
    assert call(t=4) == call(M=-2) == call(K=0) == call(w=None) == _ops.E_ARG
    assert call(ldw=299) == _ops.E_UNSUPPORTED and call(M=0) == 0


def test_route_checks():
    def call(T=4, E=16, k=2, groups=1, top=1, x=256, w=256, t=0):
        return _ops.route(x, t, T, E, 1, E, k, 0, None, groups, top, 1, 1.0, w, 256, None)

    assert call(T=-1) == call(k=0) == call(k=17) == call(groups=3) == call(groups=4, top=5) == _ops.E_ARG
    assert call(groups=4, top=1, k=5) == call(x=None) == call(w=None) == call(t=9) == call(groups=0) == _ops.E_ARG
    assert call(E=1025) == call(E=130, groups=65, k=1) == call(E=200, k=65) == _ops.E_UNSUPPORTED
    assert call(T=0) == 0
    assert _ops.route_grad(256, 0, 4, 16, 1, 16, 2, 0, 1, 1.0, 256, None, 2, 1, 256, None) == _ops.E_ARG
    assert _ops.route_grad(256, 0, 4, 16, 1, 16, 2, 0, 1, 1.0, 256, 256, 2, 1, 264, None) == _ops.E_UNSUPPORTED


def test_experts_checks():
    T, k, E, D, I = 8, 2, 4, 256, 128
    need = _ops.experts_workspace(T, k, E, D, I)

    def call(T=T, E=E, ld1=D, ws=256, n=need, w1=256, k=k, t=0, w1e=2 * I * D):
        return _ops.experts(256, t, T, D, 1, 256, k, 1, 256, k, E, D, I, w1, w1e, I * D, ld1, 256, 4, 2, 2, 1, 256,
                            I * D, I, 256, 2, 1, 1, 256, ws, n, None)

    assert call(ws=None) == call(n=need - 1) == call(ws=64) == _ops.E_WORKSPACE
    assert call(E=0) == call(k=0) == call(w1=None) == call(t=7) == call(T=-1) == call(w1e=-16) == _ops.E_ARG
    assert call(E=1025) == call(ld1=128) == call(ld1=264) == call(w1=264) == call(T=1 << 40) == _ops.E_UNSUPPORTED
    assert call(T=0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 128)
    for f in (lambda: fp8.quantize(x), lambda: fp8.quantize_weight(x), lambda: fp8.linear(x, x), lambda: moe.route(x, 2)):
        with pytest.raises(ValueError):
            f()

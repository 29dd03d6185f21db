"""The 4-bit operators without a GPU: what the C ABI and the Python functions refuse, and that a call
neither records into a trace nor holds the interpreter."""

import ctypes
import functools
import sys
import threading

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from f16acc_amd import _ops, fp4
from tests.test_ops_tracing import Wrapper

F4, E8 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def test_quantisation_checks():
    def call(x=256, t=0, rows=4, cols=200, q=256, ldq=128, s=256, sr=8, sq=4, qt=None, ldqt=0, st=None, str_=4, stq=4, second=False):
        m = _ops.Fp4Matrix(x, rows, cols, cols, 1, q, ldq, s, sr, sq, qt, ldqt, st, str_, stq)
        none = _ops.Fp4Matrix(None, 0, 0, 0, 1, None, 0, None, 0, 0, None, 0, None, 0, 0)
        a, b = (none, m) if second else (m, None)
        return _ops.fp4_quant(ctypes.byref(a), ctypes.byref(b) if b else None, t, None)

    for second in (False, True):
        f = functools.partial(call, second=second)
        assert f(x=None) == f(t=3) == f(t=-1) == f(rows=-1) == f(cols=-1) == f(q=None) == _ops.E_ARG
        assert f(s=None) == f(sr=-4) == f(sq=-4) == f(qt=256, ldqt=64) == _ops.E_ARG
        assert f(ldq=100) == f(ldq=192) == f(ldq=64) == f(q=264) == f(s=258) == f(sr=6) == _ops.E_UNSUPPORTED
        assert f(qt=256, ldqt=128, st=256) == f(qt=260, ldqt=64, st=256) == f(rows=1 << 41) == _ops.E_UNSUPPORTED
        assert f(qt=256, ldqt=64 << 30, st=256, rows=128 << 30, q=None) == _ops.E_UNSUPPORTED
        big = dict(q=None, qt=256, st=256, ldqt=64 << 14, rows=1 << 21)  # more tiles than a launch holds
        assert f(cols=1 << 17, **big) == _ops.E_UNSUPPORTED
        assert f(rows=0) == f(cols=0) == 0
    assert _ops.fp4_quant(None, None, 0, None) == _ops.E_ARG

    def back(x=256, s=256, qt=256, ldqt=64, st=256, rows=4):
        return _ops.fp4_transpose(x, 100, 1, s, 7, 1, rows, 200, qt, ldqt, st, 4, 800, None)

    assert back(x=None) == back(s=None) == back(qt=None) == back(st=None) == back(rows=-2) == _ops.E_ARG
    assert back(ldqt=128) == back(qt=8) == back(st=257) == _ops.E_UNSUPPORTED and back(rows=0) == 0

    def values(q=256, s=256, out=256, t=0, rows=4):
        return _ops.fp4_values(q, 100, 1, s, 7, 1, rows, 200, out, t, None)

    assert values(q=None) == values(s=None) == values(out=None) == values(t=3) == values(rows=-1) == _ops.E_ARG
    assert values(out=264) == _ops.E_UNSUPPORTED and values(rows=0) == 0


def test_mm_checks():
    def workspace(x=256, xr=128, xc=1, sxq=0, w=256, wr=128, swq=0, M=4, N=4, K=256, tile=-1, splits=0):
        return _ops.mm_fp4_workspace(x, xr, xc, sxq, w, wr, 1, swq, M, N, K, tile, splits)

    need = workspace()

    def call(x=256, xr=128, xc=1, sx=256, sxm=8, sxb=1, sxq=0, w=256, wr=128, sw=256, swn=8, swq=0, c=256, M=4, N=4, K=256, t=0,
             tile=-1, splits=0, ws=256, n=need):
        return _ops.mm_fp4(x, xr, xc, sx, sxm, sxb, sxq, w, wr, 1, sw, swn, 1, swq, None, c, N, 1, M, N, K, t, tile, splits, ws,
                           n, None)

    assert call(M=-1) == call(K=-1) == call(N=-1) == call(t=3) == call(c=None) == call(x=None) == call(w=None) == _ops.E_ARG
    assert call(sx=None) == call(sw=None) == call(swn=-1) == call(sxb=-1) == call(sxq=-4) == call(K=0) == _ops.E_ARG
    assert call(xr=-128) == call(wr=-1) == call(xc=-1) == _ops.E_ARG
    assert call(K=1 << 24, xr=1 << 23, wr=1 << 23) == call(M=1 << 31) == call(N=1 << 31) == _ops.E_UNSUPPORTED
    assert call(sxq=6) == call(sxq=4, sxm=6) == call(swq=4, sw=258) == call(sxq=4, sxm=1 << 23) == _ops.E_UNSUPPORTED
    assert call(sxq=4, x=264) == call(sxq=4, xr=120) == call(swq=4, wr=1 << 23) == call(sxq=4, xc=2) == _ops.E_UNSUPPORTED
    assert call(M=1 << 20, N=1 << 16, tile=5, ws=None) == call(M=1 << 30, N=1 << 14) == _ops.E_UNSUPPORTED
    assert call(M=1 << 20, N=(1 << 16) - 64, tile=5, ws=None) == _ops.E_WORKSPACE
    assert call(tile=6) == call(tile=-2) == call(splits=-1) == _ops.E_ARG
    assert call(ws=None) == call(ws=128) == call(n=need - 1) == _ops.E_WORKSPACE
    # single scale bytes are reordered; rows that are not aligned, or do not end with a block, are copied; parts of K
    assert need >= 2 * 4 * 2 * 4 and workspace(sxq=4, swq=4) == 0
    for other in (dict(x=264), dict(xr=130), dict(xc=2), dict(K=254), dict(w=257), dict(wr=1 << 23)):
        assert workspace(**other) >= need + 4 * 128
        assert call(**other) == _ops.E_WORKSPACE
    assert workspace(M=1, xr=1) == workspace(M=1)  # the stride of a single row addresses nothing
    assert workspace(sxq=4, swq=4, K=1024, xr=512, wr=512, tile=2, splits=2) >= 2 * 4 * 4 * 4
    assert call(M=0) == call(N=0) == 0 == workspace(M=0) == workspace(tile=6) == workspace(splits=-1)


def test_linear_checks():
    need = _ops.linear_fp4_workspace(100, 64, 288, 256, 144)
    assert need >= 100 * 192 + 100 * 3 * 4 + 64 * 3 * 4 and _ops.linear_fp4_workspace(0, 64, 288, 256, 144) == 0
    # K is no multiple of 32, or the rows are not aligned: room for a copy of the weight
    for other in ((280, 256, 144), (288, 264, 144), (288, 256, 145)):
        assert _ops.linear_fp4_workspace(100, 64, *other) >= need + 64 * 144

    def call(ws=256, n=need, M=100, N=64, t=0, ldw=144, K=288, w=256, sw=256, swn=9, y=256):
        return _ops.linear_fp4(256, t, K, 1, w, ldw, sw, swn, 1, None, y, M, N, K, ws, n, None)

    assert call(ws=None) == call(n=need - 1) == call(ws=128) == _ops.E_WORKSPACE
    assert call(t=4) == call(M=-2) == call(N=-1) == call(K=0) == call(w=None) == call(sw=None) == call(swn=-1) == _ops.E_ARG
    assert call(M=1 << 30, N=1 << 14) == _ops.E_UNSUPPORTED and call(M=1, N=1 << 27, K=2, ws=None) == _ops.E_WORKSPACE
    assert call(y=None) == _ops.E_ARG and call(ldw=143) == _ops.E_UNSUPPORTED and call(M=0) == call(N=0) == 0


def test_the_stride_of_a_single_weight_row_is_not_looked_at():
    for M, K, w in ((1, 288, 256), (100, 288, 256), (100, 250, 256), (100, 288, 257)):
        sizes = {_ops.linear_fp4_workspace(M, 1, K, w, ldw) for ldw in (0, 1, 16, 143, 144, 1 << 23, -16)}
        assert len(sizes) == 1 and sizes.pop() > 0
    assert _ops.linear_fp4(256, 0, 288, 1, 256, 0, 256, 9, 1, None, 256, 100, 1, 288, None, 0, None) == _ops.E_WORKSPACE


def test_few_tokens_need_no_workspace():
    few = _ops.linear_fp4_few
    assert few(1, 8960, 1536, 1) == few(16, 64, 288, 1) == few(1, 28672, 7169, 1) == few(1, 64, 1, 9) == 1
    assert few(17, 64, 288, 1) == few(1, 64, 288, 2) == few(8, 28672, 7168, 1) == few(1, 64, 1 << 16, 1) == 0
    assert few(0, 64, 288, 1) == few(1, 0, 288, 1) == few(1, 64, 0, 1) == few(-1, 64, 288, 1) == 0
    for M in (1, 16):  # a column stride that the kernel does not take: the tiles, and their workspace
        assert _ops.linear_fp4(256, 0, 600, 2, 256, 144, 256, 9, 1, None, 256, M, 64, 288, None, 0, None) == _ops.E_WORKSPACE


CPU = torch.zeros(4, 64)
Q, S = torch.zeros(4, 32, dtype=torch.uint8).view(F4), torch.zeros(4, 2, dtype=torch.uint8).view(E8)
CALLS = {
    "quantize": lambda x: fp4.quantize(x)[0].view(torch.uint8), "dequantize": lambda x: fp4.dequantize(Q, S) + x,
    "mm": lambda x: fp4.mm(Q, S, Q.t(), S.t()) + x[:, :4], "linear": lambda x: fp4.linear(x, x),
    "linear_stored": lambda x: fp4.linear(x, Q, S),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_cpu_tensors_traces_and_tangents_are_refused(name):
    f = CALLS[name]
    with pytest.raises(ValueError, match="GPU"):
        f(CPU)
    for kw in (dict(), dict(pre_dispatch=True)):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(f, **kw)(CPU)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(f, CPU)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError, match="traced"):
        f(torch.zeros(4, 64))
    for transform in (torch.func.vmap(f), torch.func.grad(lambda x: f(x).float().sum())):
        with pytest.raises(NotImplementedError, match="traced"):
            transform(CPU)
    if name in ("quantize", "linear", "linear_stored"):
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(CPU, CPU.clone()))


@pytest.mark.parametrize("name", sorted(CALLS))
def test_the_interpreter_is_free_during_a_call(name):
    """The waiting thread never asks for the interpreter: it gets it only where a call gives it up."""
    lock, passed = threading.Lock(), threading.Event()
    lock.acquire()

    def wait():
        with lock:
            passed.set()

    waiting = threading.Thread(target=wait)
    waiting.start()
    before = sys.getswitchinterval()
    sys.setswitchinterval(1000.0)
    try:
        lock.release()
        for _ in range(3000):
            with pytest.raises(ValueError):
                CALLS[name](CPU)
            if passed.is_set():
                break
        assert passed.is_set()
    finally:
        sys.setswitchinterval(before)
        waiting.join()


@pytest.mark.gpu
def test_tensors_that_are_not_plain_and_batched_gradients_are_refused():
    x = torch.randn(64, 64, device="cuda", requires_grad=True)
    q, s = fp4.quantize(x.detach())
    for f in (fp4.quantize, lambda x: fp4.linear(x, x), lambda x: fp4.linear(x, q, s)):
        for bad in (torch.complex(x, x).conj().imag, Wrapper(x.detach()), x.detach().to_sparse()):
            with pytest.raises(ValueError, match="plain"):
                f(bad)
    for y in (fp4.linear(x, x), fp4.linear(x, q, s)):
        dy = torch.ones_like(y)
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(dy)
        with pytest.raises(ValueError, match="plain"):
            torch.autograd.grad(y, x, torch.stack([dy, dy]), is_grads_batched=True, retain_graph=True)
        want, = torch.autograd.grad(y, x, -2 * dy, retain_graph=True)
        negated = torch.complex(dy, 2 * dy).conj().imag
        assert torch.equal(torch.autograd.grad(y, x, negated)[0], want)

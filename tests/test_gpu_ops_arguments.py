"""Arguments of the operators at the edges of what they take, and what mm_tile refuses."""

import pytest
import torch

from f16acc_amd import _ops, fp8, moe
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, F8, normal, weight

pytestmark = pytest.mark.gpu


def test_mm_tile_refuses_what_does_not_fit():
    M, N, K = 40, 72, 256
    a, sa = fp8.quantize(normal(M, K))
    w, ws = weight(N, K)
    f = lambda out, bias=None, tile=4, splits=1: fp8.mm_tile(a, sa, w.t(), ws.t(), out, tile, splits, bias)
    out = torch.empty(M, N, device=DEV)
    short, pair = torch.zeros(N - 1, device=DEV), torch.zeros(1, N, device=DEV)
    bad = [lambda: f(torch.empty(M + 1, N, device=DEV)), lambda: f(torch.empty(M, N + 200, device=DEV)),
           lambda: f(torch.empty(M, device=DEV)), lambda: f(out.int()), lambda: f(out.double()), lambda: f(out.cpu()),
           lambda: f(out[:1].expand(M, N)), lambda: f(out, short), lambda: f(out, pair), lambda: f(out, pair[0].half()),
           lambda: f(out, pair[0].cpu()), lambda: f(out, tile=6), lambda: f(out, tile=-2), lambda: f(out, splits=-1),
           lambda: fp8.mm_tile(a, sa, w.t(), ws.t().repeat_interleave(128, 1)[:, :N], out, 1, 1)]
    for g in bad:
        with pytest.raises(ValueError):
            g()
    bias = normal(3 * N, dtype=torch.float32)[::3]
    f(out, bias)
    ref.check_product(out, ref.values(a, sa), ref.values(w, ws, 128), bias)


def test_mm_tile_without_a_product_is_the_bias():
    M, N = 5, 7
    z = lambda *s: torch.zeros(*s, device=DEV)
    out, bias = torch.full((M, N), 3.0, device=DEV), normal(N, dtype=torch.float32)
    a, b = z(M, 0).to(torch.float8_e4m3fn), z(0, N).to(torch.float8_e4m3fn)
    fp8.mm_tile(a, z(M, 0), b, z(0, 1), out, -1, 0)
    assert bool((out == 0).all())
    fp8.mm_tile(a, z(M, 0), b, z(0, 1), out, -1, 0, bias)
    assert torch.equal(out, bias.expand(M, N))


def test_rows_more_than_4_mib_apart():
    M, N, K, far = 20, 24, 256, (1 << 22) + 64
    a, sa = fp8.quantize(normal(M, K))
    w, ws = weight(N, K)
    want = fp8.mm(a, sa, w.t(), ws.t(), torch.float32)
    pool = torch.zeros(N * far, dtype=torch.uint8, device=DEV).view(F8)
    apart = lambda t: pool[:t.shape[0] * far].view(t.shape[0], far)[:, :K].copy_(t)
    assert torch.equal(fp8.mm(apart(a), sa, w.t(), ws.t(), torch.float32), want)
    assert torch.equal(fp8.mm(a, sa, apart(w).t(), ws.t(), torch.float32), want)
    x = normal(M, K)
    assert torch.equal(fp8.linear(x, apart(w), ws), fp8.linear(x, w, ws))
    args = torch.ones(M, 1, device=DEV), torch.zeros(M, 1, dtype=torch.int32, device=DEV)
    w2 = torch.zeros(2, 3, far, dtype=torch.uint8, device=DEV).view(F8)[:, :, :128]
    small = fp8.quantize_weight(normal(2, 2, 128, 3)), fp8.quantize_weight(normal(2, 3, 128))
    w2.copy_(small[1][0])
    x3 = normal(M, 3)
    assert torch.equal(moe.experts(x3, *args, *small[0], w2, small[1][1]), moe.experts(x3, *args, *small[0], *small[1]))


def test_scales_more_than_4_mib_apart():
    M, N, K, far = 20, 200, 256, (1 << 20) + 16
    x = normal(M, K)
    a, sa = fp8.quantize(x)
    w, ws = weight(N, K)
    b, sb = fp8.quantize(normal(N, K, seed=5))
    pool = torch.zeros(N * far, device=DEV)
    apart = lambda t: pool[:t.shape[0] * far].view(t.shape[0], far)[:, :t.shape[1]].copy_(t)
    want = fp8.mm(a, sa, w.t(), ws.t())
    assert torch.equal(fp8.mm(a, apart(sa), w.t(), ws.t()), want)
    assert torch.equal(fp8.mm(a[:1], apart(sa[:1]), w.t(), ws.t()), fp8.mm(a[:1], sa[:1], w.t(), ws.t()))
    assert torch.equal(fp8.mm(a, sa, w.t(), apart(ws).t()), want)
    assert torch.equal(fp8.mm(a, sa, b.t(), apart(sb).t()), fp8.mm(a, sa, b.t(), sb.t()))
    assert torch.equal(fp8.linear(x, w, apart(ws)), fp8.linear(x, w, ws))
    grad = lambda s: torch.autograd.grad(fp8.linear(x.requires_grad_(), w, s), x, normal(M, N, seed=3))[0]
    assert torch.equal(grad(apart(ws)), grad(ws))


@pytest.mark.parametrize("shape", [(0, 0), (0, 5), (5, 0), (3, 0, 40), (3, 40, 0), (0, 4, 4), (2, 0, 130, 7), (2, 2, 0, 7)])
def test_empty_weights(shape):
    for dtype in (torch.float16, torch.float32):
        q, s = fp8.quantize_weight(torch.zeros(shape, dtype=dtype, device=DEV))
        assert q.shape == shape and q.dtype == F8 and s.dtype == torch.float32
        assert s.shape == (*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128))


@pytest.mark.parametrize("rows,cols,ldq", [(5, 200, 256), (5, 200, 640), (70, 1, 256), (3, 128, 1280)])
def test_rows_wider_than_their_blocks(rows, cols, ldq):
    """The C ABI's rows may be padded by whole blocks: zeros, and no scale past the last block with a column."""
    x = normal(rows, cols)
    q = torch.full((rows, ldq), 7, dtype=torch.uint8, device=DEV)
    blocks = -(-cols // 128)
    s = torch.full((ldq // 128 + 2, rows), 7.0, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    assert _ops.quant_rows(x.data_ptr(), 0, rows, cols, cols, 1, q.data_ptr(), ldq, s.data_ptr(), rows, stream) == 0
    want = fp8.quantize(x)
    assert torch.equal(q[:, :cols], want[0].view(torch.uint8)) and bool((q[:, cols:] == 0).all())
    assert torch.equal(s[:blocks].t(), want[1]) and bool((s[blocks:] == 7.0).all())


def test_experts_refuses_every_operand_that_requires_a_gradient():
    x, w = normal(4, 128), torch.ones(4, 1, device=DEV)
    ids = torch.zeros(4, 1, dtype=torch.int32, device=DEV)
    args = [x, w, ids, *fp8.quantize_weight(normal(2, 2, 128, 128)), *fp8.quantize_weight(normal(2, 128, 128))]
    want = moe.experts(*args)
    for i in (0, 1, 3, 4, 5, 6):
        grown = list(args)
        grown[i] = args[i].detach().clone().requires_grad_()
        with pytest.raises(ValueError, match="backward"):
            moe.experts(*grown)
        with torch.no_grad():
            assert torch.equal(moe.experts(*grown), want)

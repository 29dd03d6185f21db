"""8-bit block-scaled products on the GPU against plain 64-bit statements."""

import pytest
import torch

from f16acc_amd import fp8
from tests import ops_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = torch.float8_e4m3fn


def normal(*shape, dtype=torch.float16, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def weight(*shape, seed=1):
    """A stored weight: (q, scales)."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(*shape, generator=g) * 120).clamp(-448, 448).to(F8)
    s = torch.rand(*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128), generator=g) * 1e-3 + 1e-4
    return q.to(DEV), s.to(DEV)


def same_quantised(q, s, want_q, want_s):
    assert q.dtype == F8 and s.dtype == torch.float32
    assert torch.equal(s.cpu(), want_s)
    assert torch.equal(q.cpu().float().double(), want_q)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (5, 129), (130, 1000), (257, 1536)])
def test_quantize_rows_exactly(shape, dtype):
    x = normal(*shape, dtype=dtype)
    same_quantised(*fp8.quantize(x), *ref.quantize(x))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (127, 3), (129, 5), (300, 250)])
def test_quantize_columns_and_squares_exactly(shape, dtype):
    x = normal(*shape, dtype=dtype)
    same_quantised(*fp8.quantize(x, transposed=True), *ref.quantize(x.t()))
    same_quantised(*fp8.quantize_weight(x), *ref.quantize(x, 128, 128))


def test_quantize_strides_and_leading_dimensions():
    x = normal(6, 40, 300)
    for v in (x[:, ::2, ::3], x.transpose(0, 1), x[:, :, 7:], x[0].t(), x.transpose(1, 2), x[:, :1].expand(6, 5, 300)):
        q, s = fp8.quantize(v)
        assert q.shape == v.shape
        want = ref.quantize(v.reshape(-1, v.shape[-1]))
        same_quantised(q.reshape(-1, v.shape[-1]), s.reshape(-1, s.shape[-1]), *want)
    w = normal(3, 140, 200)
    q, s = fp8.quantize_weight(w.transpose(1, 2))
    for i in range(3):
        same_quantised(q[i], s[i], *ref.quantize(w[i].t(), 128, 128))
    q, s = fp8.quantize(normal(0, 40))
    assert q.shape == (0, 40) and s.shape == (0, 1)


def test_quantize_every_e4m3_tie_and_the_extremes():
    # blocks whose largest value is 448 have scale 1 and reciprocal 1: values pass unscaled
    mids = torch.cat([(torch.arange(2 ** 11).float() / 2.0 ** 11 + 1) * 2.0 ** e for e in range(-12, 9)])
    x = torch.cat([mids, -mids, torch.tensor([0.0, -0.0, 2.0 ** -10, 2.0 ** -11, 3 * 2.0 ** -10])])
    x = x[x.abs() <= 448]
    x = torch.nn.functional.pad(x, (0, -len(x) % 127)).view(-1, 127)
    x = torch.cat([x, torch.full((len(x), 1), 448.0)], 1).to(DEV)
    q, s = fp8.quantize(x)
    assert bool((s == 1).all())
    same_quantised(q, s, *ref.quantize(x))
    # zeros, a subnormal block, the largest finite values
    x = torch.zeros(3, 128, device=DEV)
    x[1] = 1e-38
    x[2] = torch.finfo(torch.float32).max
    q, s = fp8.quantize(x)
    same_quantised(q, s, *ref.quantize(x))
    assert bool((q[0].float() == 0).all()) and bool((q[2].float() == 448).all())


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_block_with_a_non_finite_value_spoils_its_own_row_only(bad):
    w, ws = weight(192, 256)
    for M in (4, 40, 300):  # the small kernel, the tiles
        x = normal(M, 256)
        good = fp8.linear(x, w, ws)
        x[3, 200] = bad
        y = fp8.linear(x, w, ws)
        rows = [i for i in range(M) if i != 3]
        assert torch.equal(y[rows], good[rows]) and bool(torch.isnan(y[3]).all())
    s = fp8.quantize(x)[1]
    assert bool(torch.isnan(s[3, 1])) and bool(torch.isfinite(s[3, 0]))


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 128, 128), (2, 16, 400), (16, 100, 1000), (17, 130, 129), (33, 64, 256),
                                   (64, 200, 384), (100, 300, 500), (129, 257, 640), (500, 700, 200), (1030, 520, 300)])
def test_mm(M, N, K, out):
    a, sa = fp8.quantize(normal(M, K, std=0.5))
    w, ws = weight(N, K)
    c = fp8.mm(a, sa, w.t(), ws.t(), out)
    assert c.dtype == out and c.shape == (M, N)
    ref.check_product(c, ref.values(a, sa), ref.values(w, ws, 128))


@pytest.mark.parametrize("M,N,K", [(1, 2, 1), (20, 130, 100), (70, 66, 384), (300, 257, 500), (1100, 1300, 130)])
def test_mm_with_a_scale_for_each_column(M, N, K):
    a, sa = fp8.quantize(normal(M, K))
    b, sb = fp8.quantize(normal(N, K, seed=5, std=3.0))
    ref.check_product(fp8.mm(a, sa, b.t(), sb.t(), torch.float32), ref.values(a, sa), ref.values(b, sb))


def test_mm_large_tiles_in_every_k_order():
    """Operands of small integers with power-of-two scales: every sum is exact, so every tile must be."""
    g = torch.Generator().manual_seed(3)
    for M, N, K in ((4096, 4096, 256), (2048, 1537, 1000), (640, 4000, 384), (200, 8192, 640)):
        a = torch.randint(-3, 4, (M, K), generator=g).float().to(F8).to(DEV)
        b = torch.randint(-3, 4, (N, K), generator=g).float().to(F8).to(DEV)
        sa = torch.exp2(torch.randint(-2, 3, (M, -(-K // 128)), generator=g).float()).to(DEV)
        sb = torch.exp2(torch.randint(-2, 3, (-(-N // 128), -(-K // 128)), generator=g).float()).to(DEV)
        want = (a.float() * sa.repeat_interleave(128, 1)[:, :K]).double() @ (
            b.float() * sb.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).double().t().contiguous()
        assert torch.equal(fp8.mm(a, sa, b.t(), sb.t(), torch.float32).double(), want)
        sr = torch.exp2(torch.randint(-2, 3, (N, -(-K // 128)), generator=g).float()).to(DEV)
        want = (a.float() * sa.repeat_interleave(128, 1)[:, :K]).double() @ (
            b.float() * sr.repeat_interleave(128, 1)[:, :K]).double().t().contiguous()
        assert torch.equal(fp8.mm(a, sa, b.t(), sr.t(), torch.float32).double(), want)


@pytest.mark.parametrize("tile,splits", [(t, s) for t in range(6) for s in (1, 3)])
def test_mm_every_tile_and_split(tile, splits):
    """The same product in every tile, whole and in parts of K: exact sums, ragged edges, both kinds of scales."""
    g = torch.Generator().manual_seed(7)
    for M, N, K in ((1, 1, 300), (300, 333, 1000), (513, 580, 640)):
        a = torch.randint(-3, 4, (M, K), generator=g).float().to(F8).to(DEV)
        b = torch.randint(-3, 4, (N, K), generator=g).float().to(F8).to(DEV)
        sa = torch.exp2(torch.randint(-2, 3, (M, -(-K // 128)), generator=g).float()).to(DEV)
        bias = torch.randint(-9, 9, (N,), generator=g).float().to(DEV)
        for rows in (False, True):
            if rows and tile not in (0, 2, 4):
                continue
            sb = torch.exp2(torch.randint(-2, 3, (N if rows else -(-N // 128), -(-K // 128)), generator=g).float()).to(DEV)
            want = ref.values(a, sa) @ ref.values(b, sb, 1 if rows else 128).t() + bias.cpu().double()
            for out in (torch.empty(M, N, device=DEV), torch.empty(N, M, device=DEV).t(),
                        torch.zeros(M, N + 5, device=DEV)[:, 3:N + 3]):
                fp8.mm_tile(a, sa, b.t(), sb.t(), out, tile, splits, bias)
                assert torch.equal(out.cpu().double(), want)


def test_mm_layouts():
    M, N, K = 90, 150, 272
    a, sa = fp8.quantize(normal(M, K))
    w, ws = weight(N, K)
    want = fp8.mm(a, sa, w.t(), ws.t(), torch.float32)
    wide = torch.zeros(2 * M, K + 48, dtype=torch.uint8, device=DEV).view(F8)
    wide[::2, 16:K + 16] = a
    wide[::2, K + 16:] = torch.full((), float("nan")).to(F8)  # what lies past K is not read
    views = [wide[::2, 16:K + 16], a.t().contiguous().t(), torch.cat([a[:, :1], a], 1)[:, 1:]]
    for v in views:
        assert torch.equal(v.float(), a.float())
        assert torch.equal(fp8.mm(v, sa, w.t(), ws.t(), torch.float32), want)
    assert torch.equal(fp8.mm(a, sa.contiguous(), w.t().contiguous(), ws.t().contiguous(), torch.float32), want)
    one = torch.ones(1, 1, device=DEV)
    b = fp8.mm(a, one.expand(M, 3), w.t(), one.expand(3, 2), torch.float32)
    ref.check_product(b, a.cpu().double(), w.cpu().double())


def test_mm_reads_past_neither_k_nor_n():
    """NaN bytes all around an operand's rows."""
    for M, N, K in ((40, 72, 144), (300, 200, 400), (5, 40, 208)):
        nan = torch.full((), float("nan")).to(F8)
        hold = [torch.zeros(n + 300, 1024, dtype=torch.uint8, device=DEV).view(F8) for n in (M, N)]
        for h in hold:
            h[:] = nan
        a, b = hold[0][:M, :K], hold[1][:N, :K]
        qa, sa = fp8.quantize(normal(M, K))
        w, ws = weight(N, K)
        a.copy_(qa), b.copy_(w)
        assert torch.equal(fp8.mm(a, sa, b.t(), ws.t()), fp8.mm(qa, sa, w.t(), ws.t()))


def test_mm_offsets_past_32_bits():
    M, N, K = 330000, 24, 16384
    q = torch.zeros(M, K, dtype=torch.uint8, device=DEV)
    q[-300:] = normal(300, K).to(F8).view(torch.uint8)
    s = torch.ones(M, K // 128, device=DEV)
    w, ws = weight(N, K)
    f32 = lambda q, s: fp8.mm_tile(q, s, w.t(), ws.t(), torch.empty(len(q), N, device=DEV), 4, 1)
    c = f32(q.view(F8), s)  # (one tile and no split for both: the same sums in the same order)
    assert torch.equal(c[-300:], f32(q.view(F8)[-300:].clone(), s[-300:]))
    ref.check_product(c[-20:], q.view(F8)[-20:].cpu().double(), ref.values(w, ws, 128))
    assert bool((c[:M - 300] == 0).all())


def test_mm_empty():
    f = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=DEV).view(F8)
    z = lambda *s: torch.zeros(*s, device=DEV)
    assert fp8.mm(f(0, 8), z(0, 1), f(8, 3), z(1, 1)).shape == (0, 3)
    assert fp8.mm(f(3, 8), z(3, 1), f(8, 0), z(1, 0)).shape == (3, 0)
    assert bool((fp8.mm(f(3, 0), z(3, 0), f(0, 4), z(0, 1)) == 0).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K,bias", [(1, 1, 1, True), (1, 300, 1536, False), (3, 1537, 250, True), (8, 64, 16, True),
                                        (15, 130, 2000, False), (16, 128, 1040, True), (17, 128, 1040, True),
                                        (77, 257, 897, True), (150, 400, 512, False)])
def test_linear_stored_weight(M, N, K, bias, dtype):
    x = normal(M, K, dtype=dtype)
    w, ws = weight(N, K)
    b = normal(N, dtype=dtype, seed=9) if bias else None
    y = fp8.linear(x, w, ws, b)
    assert y.dtype == dtype
    ref.check_product(y, ref.rounded(x), ref.values(w, ws, 128), b)


@pytest.mark.parametrize("M", [1, 7, 12, 40, 200])
def test_linear_weight_rows_at_any_address(M):
    """Rows that start anywhere and end anywhere, NaN bytes around them; a row-major [K, N] weight."""
    K, N = 403, 70
    w, ws = weight(N, K)
    x = normal(M, K)
    want = fp8.linear(x, w, ws)
    ref.check_product(want, ref.rounded(x), ref.values(w, ws, 128))
    for pad, off in ((5, 3), (13, 0), (45, 16), (16, 8)):
        hold = torch.full((N * (K + pad) + 64,), float("nan")).to(F8).to(DEV)
        v = hold[off:off + N * (K + pad)].view(N, K + pad)[:, :K]
        v.copy_(w)
        assert torch.equal(fp8.linear(x, v, ws), want)
    assert torch.equal(fp8.linear(x, w.t().contiguous().t(), ws), want)
    assert torch.equal(fp8.linear(x, w[:1], ws[:1]), fp8.linear(x, w[:1].clone(), ws[:1]))


def test_linear_views_and_leading_dimensions():
    w, ws = weight(96, 256)
    x = normal(4, 6, 512)
    for v in (x[:, :, ::2], x[:, :, :256], x[:2, 1:3, 3:259], x[0, 0, :256], x[:, :1, :256].expand(4, 3, 256)):
        y = fp8.linear(v, w, ws)
        assert y.shape == (*v.shape[:-1], 96)
        ref.check_product(y.reshape(-1, 96), ref.rounded(v.reshape(-1, 256)), ref.values(w, ws, 128))
    assert fp8.linear(x[:0, :, :256], w, ws).shape == (0, 6, 96)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 130, 200), (130, 1, 70), (50, 260, 129), (300, 128, 256), (257, 300, 520)])
def test_linear_gradients_against_the_formula(M, N, K, dtype):
    x = normal(M, K, dtype=dtype).requires_grad_()
    w = normal(N, K, dtype=dtype, seed=2, std=0.1).requires_grad_()
    dy = normal(M, N, dtype=dtype, seed=3)
    y = fp8.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    wq = ref.rounded(w, 128, 128)
    ref.check_product(y, ref.rounded(x), wq)
    ref.check_product(dx, ref.rounded(dy), wq.t())
    ref.check_product(dw, ref.rounded(dy.t()), ref.rounded(x.t()))
    only, = torch.autograd.grad(fp8.linear(x.detach(), w), w, dy)
    assert torch.equal(only, dw)
    only, = torch.autograd.grad(fp8.linear(x, w.detach()), x, dy)
    assert torch.equal(only, dx)
    assert torch.equal(fp8.linear(x.detach(), w.detach()), y)


def test_linear_gradients_against_differences():
    """Values that e4m3 holds with scale 1 in both directions, so the layer is bilinear and its differences exact."""
    g = torch.Generator().manual_seed(4)
    M, N, K = 128, 128, 256

    def exact(r, c):
        t = torch.randint(-4, 5, (r, c), generator=g).float()
        t[torch.arange(r), torch.arange(r) % c] = 448.0  # every row, column and square block has its 448
        for i in range(128, c):
            t[i % r, i] = 448.0
        return t.to(DEV)

    x, w, dy = exact(M, K), exact(N, K), exact(M, N)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fp8.linear(xg, wg), (xg, wg), dy)
    f = lambda x, w: (fp8.linear(x, w).double() * dy.double()).sum()
    scale = 448.0 ** 2 * 8
    for (i, j) in ((0, 5), (77, 200), (127, 130)):
        e = torch.zeros_like(x)
        e[i, j] = 1.0
        assert abs(((f(x + e, w) - f(x - e, w)) / 2 - dx[i, j]).item()) <= ref.MFMA * scale * N
        assert abs(((f(x, w + e) - f(x, w - e)) / 2 - dw[i, j]).item()) <= ref.MFMA * scale * M


def test_linear_bias_and_stored_weight_gradients():
    x, w, b = normal(40, 200).requires_grad_(), normal(60, 200, seed=2).requires_grad_(), normal(60).requires_grad_()
    dy = normal(40, 60, seed=3)
    dx, dw, db = torch.autograd.grad(fp8.linear(x, w, bias=b), (x, w, b), dy)
    assert torch.equal(db, dy.sum(0)) and dx.shape == x.shape and dw.shape == w.shape
    q, s = weight(60, 200)
    dx, db = torch.autograd.grad(fp8.linear(x, q, s, b), (x, b), dy)
    ref.check_product(dx, ref.rounded(dy), ref.values(q, s, 128).t())
    assert torch.equal(db, dy.sum(0))


def test_linear_gradients_from_expanded_and_strided_grads():
    x, w = normal(30, 40, dtype=torch.float32).requires_grad_(), normal(20, 40, dtype=torch.float32, seed=2).requires_grad_()
    for dy in (torch.ones((), device=DEV).expand(30, 20), normal(20, 30, dtype=torch.float32, seed=3).t()):
        got = torch.autograd.grad(fp8.linear(x, w), (x, w), dy)
        want = torch.autograd.grad(fp8.linear(x, w), (x, w), dy.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):  # there is no second derivative
        dx, = torch.autograd.grad(fp8.linear(x, w).sum(), x, create_graph=True)
        torch.autograd.grad(dx.sum(), w)
    a = normal(6, 5, 40, dtype=torch.float32)
    view = a.transpose(0, 1).requires_grad_()
    dx, = torch.autograd.grad(fp8.linear(view, w).square().sum(), view)
    assert dx.shape == view.shape


def test_linear_empty_gradients():
    x, w = torch.zeros(0, 32, device=DEV, requires_grad=True), normal(8, 32, dtype=torch.float32).requires_grad_()
    dx, dw = torch.autograd.grad(fp8.linear(x, w).sum(), (x, w))
    assert dx.shape == (0, 32) and bool((dw == 0).all())


def test_same_bits_every_time_and_on_any_stream():
    x, (w, ws) = normal(200, 1000), weight(400, 1000)
    want = fp8.linear(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [fp8.linear(x, w, ws) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_graph_replays_match_eager():
    w, ws = weight(300, 512)
    for M in (3, 100):
        x = normal(M, 512)
        fp8.linear(x, w, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp8.linear(x, w, ws)
        for i in range(3):
            x.copy_(normal(M, 512, seed=20 + i))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, fp8.linear(x, w, ws))


def test_refusals():
    x, (w, ws) = normal(4, 256), weight(64, 256)
    q, s = fp8.quantize(x)
    bad = [lambda: fp8.quantize(x.double()), lambda: fp8.quantize(x.cpu()), lambda: fp8.quantize(normal(2, 3, 4), True),
           lambda: fp8.quantize_weight(x[0]), lambda: fp8.quantize(q), lambda: fp8.linear(x, w), lambda: fp8.linear(x, w, ws[:, :1]),
           lambda: fp8.linear(x, w, ws.double()), lambda: fp8.linear(x[:, :128], w, ws), lambda: fp8.linear(x, w.cpu(), ws),
           lambda: fp8.linear(x, w, ws, normal(63)), lambda: fp8.linear(x, w, ws, normal(64, dtype=torch.float32)),
           lambda: fp8.linear(x, x[:, :256], ws), lambda: fp8.linear(x.to(F8), w, ws), lambda: fp8.mm(q, s, w, ws),
           lambda: fp8.mm(q, s[:, :1], w.t(), ws.t()), lambda: fp8.mm(q, s, w.t(), ws), lambda: fp8.mm(x, s, w.t(), ws.t()),
           lambda: fp8.mm(q, s, w.t(), ws.t(), torch.int8), lambda: fp8.mm(q, s.half(), w.t(), ws.t()),
           lambda: fp8.mm(q[0], s, w.t(), ws.t())]
    for f in bad:
        with pytest.raises(ValueError):
            f()

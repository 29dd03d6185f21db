"""Microscaled 4-bit products on the GPU against plain 64-bit statements."""

import pytest
import torch

from f16acc_amd import _ops, fp4
from tests import fp4_reference as ref
from tests.fp4_reference import E8, F4

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def normal(*shape, dtype=torch.float16, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(DEV)


def stored(N, K, seed=1, low=-4, high=2):
    """A stored operand [N, ceil(K / 2)] of any codes and its scales; an odd last value stands alone."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (N, -(-K // 2)), generator=g, dtype=torch.uint8)
    if K % 2:
        q[:, -1] &= 15
    s = torch.randint(127 + low, 128 + high, (N, -(-K // 32)), generator=g).to(torch.uint8)
    return q.view(F4).to(DEV), s.view(E8).to(DEV)


def u8(t):
    return t.view(torch.uint8)


def same_quantised(q, s, x):
    want_q, want_e = ref.quantize(x)
    assert q.dtype == F4 and s.dtype == E8
    assert q.shape == (x.shape[0], -(-x.shape[1] // 2)) and s.shape == want_e.shape
    assert torch.equal(u8(s).cpu().long(), want_e + 127)
    got, finite = ref.unpack(q, x.shape[1]), (want_e != 128).repeat_interleave(32, 1)[:, :x.shape[1]]
    assert torch.equal(torch.where(finite, got, 0.0), torch.where(finite, want_q, 0.0))
    if x.shape[1] % 2:
        assert bool((u8(q)[:, -1] < 16).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (130, 1000), (257, 1536), (2, 127), (7, 129)])
def test_quantize_exactly_in_both_directions(shape, dtype):
    x = normal(*shape, dtype=dtype)
    same_quantised(*fp4.quantize(x), x)
    same_quantised(*fp4.quantize(x, transposed=True), x.t())


def test_quantize_strides_and_leading_dimensions():
    x = normal(6, 40, 300)
    for v in (x[:, ::2, ::3], x.transpose(0, 1), x[:, :, 7:], x[0].t(), x.transpose(1, 2), x[:, :1].expand(6, 5, 300), x[0, 0]):
        q, s = fp4.quantize(v)
        assert q.shape == (*v.shape[:-1], -(-v.shape[-1] // 2)) and s.shape == (*v.shape[:-1], -(-v.shape[-1] // 32))
        flat = v.reshape(-1, v.shape[-1])
        same_quantised(u8(q).reshape(len(flat), -1).view(F4), u8(s).reshape(len(flat), -1).view(E8), flat)
    for v in (x[0], x[0].t(), x[1, ::3, 5:]):
        same_quantised(*fp4.quantize(v, transposed=True), v.t())
    for shape, want in (((0, 40), (0, 20)), ((3, 0), (3, 0)), ((2, 0, 7), (2, 0, 4))):
        q, s = fp4.quantize(torch.zeros(shape, device=DEV))
        assert q.shape == want and s.shape == (*shape[:-1], -(-shape[-1] // 32))
    q, s = fp4.quantize(torch.zeros(0, 40, device=DEV), transposed=True)
    assert q.shape == (40, 0) and s.shape == (40, 0)


def test_quantize_every_tie_and_the_extremes():
    """Blocks whose largest value is 4 have scale 1: the values pass unscaled; all quarters and sixteenths up to 7."""
    v = torch.arange(-111, 112).float() / 16
    x = torch.nn.functional.pad(v, (0, -len(v) % 31)).view(-1, 31)
    x = torch.cat([x, torch.full((len(x), 1), 4.0)], 1)
    for scale in (2.0 ** -90, 2.0 ** -3, 1.0, 2.0 ** 100):
        y = (x * scale).to(DEV)
        q, s = fp4.quantize(y)
        same_quantised(q, s, y)
        assert bool((ref.scales(s) == scale).all())
    for dtype, scales in ((torch.float16, (2.0 ** -12, 2.0 ** -3, 2.0 ** 12)), (torch.bfloat16, (2.0 ** -90, 1.0, 2.0 ** 100))):
        for scale in scales:
            y = (x * scale).to(dtype).to(DEV)
            assert torch.equal(y.float().cpu(), x * scale)
            same_quantised(*fp4.quantize(y), y)
            same_quantised(*fp4.quantize(y.t(), transposed=True), y)
    y = (torch.arange(-96, 96).view(6, 32) * 2.0 ** -24).half().to(DEV)  # binary16's subnormal values
    same_quantised(*fp4.quantize(y), y)
    same_quantised(*fp4.quantize(y.t(), transposed=True), y)
    for dtype in TYPES:  # magnitudes of every size beside each other, zeros of both signs
        g = torch.Generator().manual_seed(8)
        big = 15 if dtype == torch.float16 else 120
        y = torch.ldexp(torch.randn(40, 160, generator=g), torch.randint(-big, big - 4, (40, 160), generator=g)).to(dtype).to(DEV)
        y[3, :40], y[5, 7] = -0.0, 0.0
        same_quantised(*fp4.quantize(y), y)
        same_quantised(*fp4.quantize(y, transposed=True), y.t())
    # the border between two scales: 7 is the next power of two's; zeros, tiny blocks, the largest finite values
    big = torch.finfo(torch.float32).max
    edge = torch.tensor([7.0, 6.9999995, 3.5, 3.4999998, 0.0, 2.0 ** -100, 2.0 ** -101, 1e-40, big, 1.0], device=DEV)
    y = edge[:, None] * torch.linspace(-1, 1, 32, device=DEV)
    q, s = fp4.quantize(y)
    same_quantised(q, s, y)
    same_quantised(*fp4.quantize(y.t(), transposed=True), y)
    assert bool((ref.unpack(q)[4] == 0).all()) and ref.scales(s)[0, 0] == 2.0 and ref.scales(s)[1, 0] == 1.0


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_block_with_a_non_finite_value_spoils_its_own_row_only(bad):
    w, ws = stored(192, 256)
    for M in (4, 40, 300):  # the small kernel, the tiles
        x = normal(M, 256)
        good = fp4.linear(x, w, ws)
        x[3, 200] = bad
        y = fp4.linear(x, w, ws)
        rows = [i for i in range(M) if i != 3]
        assert torch.equal(y[rows], good[rows]) and bool(torch.isnan(y[3]).all())
    q, s = fp4.quantize(x)
    same_quantised(q, s, x)
    qt, st = fp4.quantize(x, transposed=True)
    assert u8(st)[200, 0] == 255 and int((u8(st) == 255).sum()) == 1 and int((u8(s) == 255).sum()) == 1
    v = fp4.dequantize(q, s)
    assert bool(torch.isnan(v[3, 192:224]).all()) and int(torch.isnan(v).sum()) == 32
    # a weight's block: its output channel
    u8(ws)[5, 7] = 255
    for M in (4, 40, 300):
        y = fp4.linear(normal(M, 256), w, ws)
        assert bool(torch.isnan(y[:, 5]).all()) and int(torch.isnan(y).sum()) == M


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 16), (3, 5), (70, 33), (130, 100), (2, 3, 40)])
def test_dequantize_is_exact(shape, dtype):
    """Every code at scales whose products each type holds or rounds once."""
    g = torch.Generator().manual_seed(3)
    q = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).view(F4).to(DEV)
    sizes = (*shape[:-1], -(-shape[-1] // 16))
    for low, high in ((120, 135), (0, 256), (100, 145)):
        s = torch.randint(low, high, sizes, generator=g).to(torch.uint8).view(E8).to(DEV)
        v = fp4.dequantize(q, s, dtype)
        want = ref.values(q, s).to(dtype)
        assert v.dtype == dtype and v.shape == (*shape[:-1], 2 * shape[-1])
        assert torch.equal(torch.isnan(v).cpu(), torch.isnan(want))
        assert torch.equal(v.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(fp4.dequantize(q.transpose(0, -1).contiguous().transpose(0, -1), s, dtype).nan_to_num(), v.nan_to_num())


def test_dequantize_of_quantize_and_empty():
    x = normal(50, 77, dtype=torch.bfloat16)
    q, s = fp4.quantize(x)
    assert torch.equal(fp4.dequantize(q, s, torch.bfloat16)[:, :77].cpu().double(), ref.rounded(x))
    assert bool((fp4.dequantize(q, s)[:, 77] == 0).all())
    for shape in ((0, 8), (3, 0)):
        q, s = fp4.quantize(torch.zeros(shape, device=DEV))
        assert fp4.dequantize(q, s).shape == shape


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 2), (1, 128, 32), (2, 16, 400), (16, 100, 1000), (17, 130, 130), (33, 64, 256),
                                   (64, 200, 384), (100, 300, 500), (129, 257, 640), (500, 700, 200), (1030, 520, 300)])
def test_mm(M, N, K, out):
    a, sa = stored(M, K, seed=2)
    w, ws = stored(N, K)
    c = fp4.mm(a, sa, w.t(), ws.t(), out)
    assert c.dtype == out and c.shape == (M, N)
    ref.check_product(c, ref.values(a, sa), ref.values(w, ws))


def test_mm_scales_of_every_size():
    """Scales from 2^-60 to 2^60 in one sum: every block is multiplied by its own two."""
    a, sa = stored(70, 640, seed=2, low=-60, high=60)
    w, ws = stored(90, 640, low=-60, high=60)
    ref.check_product(fp4.mm(a, sa, w.t(), ws.t(), torch.float32), ref.values(a, sa), ref.values(w, ws))


@pytest.mark.parametrize("tile,splits", [(t, s) for t in range(6) for s in (1, 3)])
def test_mm_every_tile_and_split(tile, splits):
    """The same product in every tile, whole and in parts of K: sums of few bits, so exact; ragged edges."""
    g = torch.Generator().manual_seed(7)
    for M, N, K in ((1, 1, 300), (300, 333, 1000), (513, 580, 640), (200, 300, 4000)):
        a, sa = stored(M, K, seed=2, low=-1, high=2)
        w, ws = stored(N, K, low=-1, high=2)
        bias = torch.randint(-9, 9, (N,), generator=g).float().to(DEV)
        want = ref.values(a, sa) @ ref.values(w, ws).t() + bias.cpu().double()
        for out in (torch.empty(M, N, device=DEV), torch.empty(N, M, device=DEV).t(),
                    torch.zeros(M, N + 5, device=DEV)[:, 3:N + 3]):
            fp4.mm_tile(a, sa, w.t(), ws.t(), out, tile, splits, bias)
            assert torch.equal(out.cpu().double(), want)
        wide = torch.full((M + 2, N + 6), 5.0, device=DEV, dtype=torch.float16)
        fp4.mm_tile(a, sa, w.t(), ws.t(), wide[1:-1, 3:-3], tile, splits)
        wide[1:-1, 3:-3] = 5.0
        assert bool((wide == 5.0).all())  # nothing around the result is written


def test_mm_large():
    for M, N, K in ((4096, 4096, 256), (2048, 1537, 1000), (640, 4000, 384), (200, 8192, 640)):
        a, sa = stored(M, K, seed=2, low=-1, high=2)
        w, ws = stored(N, K, low=-1, high=2)
        want = ref.values(a, sa).to(DEV) @ ref.values(w, ws).to(DEV).t().contiguous()
        assert torch.equal(fp4.mm(a, sa, w.t(), ws.t(), torch.float32).double(), want)


def test_mm_layouts():
    M, N, K = 90, 150, 288
    a, sa = stored(M, K, seed=2)
    w, ws = stored(N, K)
    want = fp4.mm(a, sa, w.t(), ws.t(), torch.float32)
    wide = torch.full((2 * M, K // 2 + 48), 0x77, dtype=torch.uint8, device=DEV)
    wide[::2, 16:K // 2 + 16] = u8(a)
    views = [wide[::2, 16:K // 2 + 16].view(F4), u8(a).t().contiguous().t().view(F4),
             torch.cat([u8(a)[:, :1], u8(a)], 1)[:, 1:].view(F4)]
    for v in views:
        assert torch.equal(u8(v), u8(a))
        assert torch.equal(fp4.mm(v, sa, w.t(), ws.t(), torch.float32), want)
    back = lambda t, d: u8(t).t().contiguous().t().view(d)
    assert torch.equal(fp4.mm(a, back(sa, E8), back(w, F4).t(), back(ws, E8).t(), torch.float32), want)
    every = u8(ws).repeat_interleave(3, 1)[:, ::3].view(E8)
    assert torch.equal(fp4.mm(a, sa, w.t(), every.t(), torch.float32), want)
    one = torch.full((1, 1), 127, dtype=torch.uint8, device=DEV).view(E8)
    c = fp4.mm(a, u8(one).expand(M, 9).view(E8), w.t(), u8(one).expand(9, N).view(E8), torch.float32)
    ref.check_product(c, ref.unpack(a), ref.unpack(w))


def test_mm_reads_past_neither_k_nor_n():
    """Other codes and NaN scales all around an operand's rows."""
    for M, N, K in ((40, 72, 160), (300, 200, 400), (5, 40, 224), (130, 260, 1000)):
        a, sa = stored(M, K, seed=2)
        w, ws = stored(N, K)
        want = fp4.mm(a, sa, w.t(), ws.t())

        def hold(t, d, fill):
            h = torch.full((t.shape[0] + 300, 1024), fill, dtype=torch.uint8, device=DEV)
            v = h[:t.shape[0], :t.shape[1]]
            v.copy_(u8(t))
            return v.view(d)

        got = fp4.mm(hold(a, F4, 0x77), hold(sa, E8, 255), hold(w, F4, 0x77).t(), hold(ws, E8, 255).t())
        assert torch.equal(got, want)


def test_mm_offsets_past_32_bits():
    M, N, K = 600000, 24, 16384
    q = torch.zeros(M, K // 2, dtype=torch.uint8, device=DEV)
    s = torch.full((M, K // 32), 127, dtype=torch.uint8, device=DEV)
    a, sa = stored(300, K, seed=2)
    q[-300:], s[-300:] = u8(a), u8(sa)
    w, ws = stored(N, K)
    f32 = lambda q, s: fp4.mm_tile(q, s, w.t(), ws.t(), torch.empty(len(q), N, device=DEV), 4, 1)
    c = f32(q.view(F4), s.view(E8))  # (one tile and no split for both: the same sums in the same order)
    assert torch.equal(c[-300:], f32(a, sa)) and bool((c[:-300] == 0).all())
    ref.check_product(c[-20:], ref.values(a[-20:], sa[-20:]), ref.values(w, ws))


def test_mm_empty():
    f = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=DEV).view(F4)
    z = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=DEV).view(E8)
    assert fp4.mm(f(0, 8), z(0, 1), f(8, 3), z(1, 3)).shape == (0, 3)
    assert fp4.mm(f(3, 8), z(3, 1), f(8, 0), z(1, 0)).shape == (3, 0)
    assert bool((fp4.mm(f(3, 0), z(3, 0), f(0, 4), z(0, 4)) == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,bias", [(1, 1, 1, True), (1, 300, 1536, False), (3, 1537, 250, True), (8, 64, 16, True),
                                        (15, 130, 2000, False), (16, 128, 1040, True), (17, 128, 1040, True),
                                        (77, 257, 897, True), (150, 400, 512, False), (2, 40, 4500, False), (8, 20, 12288, True),
                                        (1, 20, 65535, True), (1, 20, 120000, False), (8, 24, 15000, True), (7, 20, 40000, False)])
def test_linear_stored_weight(M, N, K, bias, dtype):
    x = normal(M, K, dtype=dtype)
    w, ws = stored(N, K)
    b = normal(N, dtype=dtype, seed=9) if bias else None
    y = fp4.linear(x, w, ws, b)
    assert y.dtype == dtype
    ref.check_product(y, ref.rounded(x), ref.values(w, ws, K), b)


@pytest.mark.parametrize("N,K", [(40, 100), (530, 3000), (520, 3200), (4112, 2048), (4096, 4000), (4100, 4097)])
def test_linear_where_few_tokens_become_many(N, K):
    """Up to 16 tokens are one kernel's, of 8 or 16 waves, fewer where the weight is large; there a token's result is the same
    whatever is beside it."""
    x, (w, ws) = normal(17, K, dtype=torch.bfloat16), stored(N, K)
    bias = normal(N, dtype=torch.bfloat16, seed=3)
    values, wv = ref.values(*fp4.quantize(x), K), ref.values(w, ws, K)
    one = fp4.linear(x[:1], w, ws, bias)
    for M in (1, 2, 7, 8, 9, 15, 16, 17):
        y = fp4.linear(x[:M], w, ws, bias)
        ref.check_product(y, values[:M], wv, bias)
        assert M > 7 or torch.equal(y[:1], one)


@pytest.mark.parametrize("M", [1, 7, 12, 40, 200])
def test_linear_weight_rows_at_any_address(M):
    """Rows that start anywhere and end anywhere, other codes around them; a row-major [K / 2, N] weight; an odd
    last value whose high half is not zero."""
    K, N = 403, 70
    w, ws = stored(N, K)
    x = normal(M, K)
    want = fp4.linear(x, w, ws)
    ref.check_product(want, ref.rounded(x), ref.values(w, ws, K))
    P = w.shape[1]
    for pad, off in ((5, 3), (13, 0), (45, 16), (16, 8)):
        hold = torch.full((N * (P + pad) + 64,), 0x77, dtype=torch.uint8, device=DEV)
        v = hold[off:off + N * (P + pad)].view(N, P + pad)[:, :P]
        v.copy_(u8(w))
        v[:, -1] += 0x50
        assert torch.equal(fp4.linear(x, v.view(F4), ws), want)
    assert torch.equal(fp4.linear(x, u8(w).t().contiguous().t().view(F4), u8(ws).t().contiguous().t().view(E8)), want)
    assert torch.equal(fp4.linear(x, w[:1], ws[:1]), fp4.linear(x, u8(w)[:1].clone().view(F4), ws[:1]))


def test_linear_views_and_leading_dimensions():
    w, ws = stored(96, 256)
    x = normal(4, 6, 512)
    for v in (x[:, :, ::2], x[:, :, :256], x[:2, 1:3, 3:259], x[0, 0, :256], x[:, :1, :256].expand(4, 3, 256)):
        y = fp4.linear(v, w, ws)
        assert y.shape == (*v.shape[:-1], 96)
        ref.check_product(y.reshape(-1, 96), ref.rounded(v.reshape(-1, 256)), ref.values(w, ws))
    assert fp4.linear(x[:0, :, :256], w, ws).shape == (0, 6, 96)
    assert bool((fp4.linear(x[..., :0], w[:, :0], ws[:, :0], normal(96)) == normal(96)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 130, 200), (130, 1, 70), (50, 260, 129), (300, 128, 256), (257, 300, 520)])
def test_linear_gradients_against_the_formula(M, N, K, dtype):
    x = normal(M, K, dtype=dtype).requires_grad_()
    w = normal(N, K, dtype=dtype, seed=2, std=0.1).requires_grad_()
    dy = normal(M, N, dtype=dtype, seed=3)
    y = fp4.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref.check_product(y, ref.rounded(x), ref.rounded(w))
    ref.check_product(dx, ref.rounded(dy), ref.rounded(w.t()))
    ref.check_product(dw, ref.rounded(dy.t()), ref.rounded(x.t()))
    only, = torch.autograd.grad(fp4.linear(x.detach(), w), w, dy)
    assert torch.equal(only, dw)
    only, = torch.autograd.grad(fp4.linear(x, w.detach()), x, dy)
    assert torch.equal(only, dx)
    assert torch.equal(fp4.linear(x.detach(), w.detach()), y)


@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
def test_weights_of_another_type(dtype, wtype):
    x, w = normal(70, 200, dtype=dtype).requires_grad_(), normal(90, 200, dtype=wtype, seed=2).requires_grad_()
    dy = normal(70, 90, dtype=dtype, seed=3)
    y = fp4.linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == wtype
    ref.check_product(y, ref.rounded(x), ref.rounded(w))
    ref.check_product(dx, ref.rounded(dy), ref.rounded(w.t()))
    ref.check_product(dw, ref.rounded(dy.t()), ref.rounded(x.t()))


def test_a_training_step_in_a_graph():
    """Forward and backward recorded while eager steps of the same leaves come and go; every replay like eager."""
    x, w, b = normal(64, 160).requires_grad_(), normal(96, 160, seed=2, std=0.1).requires_grad_(), normal(96).requires_grad_()
    dy = normal(64, 96, seed=3)
    step = lambda: torch.autograd.grad(fp4.linear(x, w, bias=b), (x, w, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(normal(64, 160, seed=10 + i))
            dy.copy_(normal(64, 96, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, step()))


def test_several_calls_at_once():
    """Streams beside each other, every call with its own workspace."""
    w, ws = stored(700, 1000)
    xs = [normal(n, 1000, seed=n) for n in (3, 60, 300)]
    want = [fp4.linear(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    outs = []
    for x in xs:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            outs.append([fp4.linear(x, w, ws) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, y) for y, out in zip(want, outs) for o in out)


def test_linear_gradients_against_differences():
    """Values that 4 bits hold with scale 1 in both directions, so the layer is bilinear and its differences exact."""
    g = torch.Generator().manual_seed(4)
    M, N, K = 64, 96, 160

    def held(r, c):
        t = torch.randint(-2, 3, (r, c), generator=g).float()
        for i in range(0, r, 32):
            for j in range(0, c, 32):
                t[i:i + 32, j:j + 32].fill_diagonal_(6.0)  # every row and column of a block has its 6
        return t.to(DEV)

    x, w, dy = held(M, K), held(N, K), held(M, N)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(fp4.linear(xg, wg), (xg, wg), dy)
    f = lambda x, w: (fp4.linear(x, w).double() * dy.double()).sum()
    for (i, j) in ((0, 5), (37, 100), (63, 130)):
        e = torch.zeros_like(x)
        e[i, j] = 1.0
        assert ((f(x + e, w) - f(x - e, w)) / 2).item() == dx[i, j].item()
        e = torch.zeros_like(w)
        e[i, j] = 1.0
        assert ((f(x, w + e) - f(x, w - e)) / 2).item() == dw[i, j].item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 40, 31), (40, 60, 200), (130, 257, 333), (20, 128, 512)])
def test_stored_weight_gradients(M, N, K, dtype):
    """dx takes the weight's values quantised along N."""
    x, b = normal(M, K, dtype=dtype).requires_grad_(), normal(N, dtype=dtype).requires_grad_()
    dy = normal(M, N, dtype=dtype, seed=3)
    q, s = stored(N, K)
    dx, db = torch.autograd.grad(fp4.linear(x, q, s, b), (x, b), dy)
    ref.check_product(dx, ref.rounded(dy), ref.rounded(ref.values(q, s, K).t()))
    exact = dy.double().sum(0)
    bound = M * 2.0 ** -23 * dy.double().abs().sum(0) + ref.ROUND[dtype] * exact.abs() + 2.0 ** -25
    assert bool(((db.double() - exact).abs() <= bound).all())
    far = torch.zeros(2 * N, 3 * q.shape[1], dtype=torch.uint8, device=DEV)[::2, ::3].copy_(u8(q)).view(F4)
    wide = torch.zeros(s.shape[1], N, dtype=torch.uint8, device=DEV).t().copy_(u8(s)).view(E8)
    assert torch.equal(torch.autograd.grad(fp4.linear(x, far, wide), x, dy)[0], dx)


def test_linear_gradients_from_expanded_and_strided_grads():
    x, w = normal(30, 40, dtype=torch.float32).requires_grad_(), normal(20, 40, dtype=torch.float32, seed=2).requires_grad_()
    for dy in (torch.ones((), device=DEV).expand(30, 20), normal(20, 30, dtype=torch.float32, seed=3).t()):
        got = torch.autograd.grad(fp4.linear(x, w), (x, w), dy)
        want = torch.autograd.grad(fp4.linear(x, w), (x, w), dy.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    q, s = stored(20, 40)
    for layer in ((w,), (q, s)):
        with pytest.raises(RuntimeError):  # there is no second derivative
            dx, = torch.autograd.grad(fp4.linear(x, *layer).sum(), x, create_graph=True)
            torch.autograd.grad(dx.sum(), w)
    view = normal(6, 5, 40, dtype=torch.float32).transpose(0, 1).requires_grad_()
    dx, = torch.autograd.grad(fp4.linear(view, w).square().sum(), view)
    assert dx.shape == view.shape


def test_linear_empty_gradients():
    x, w = torch.zeros(0, 32, device=DEV, requires_grad=True), normal(8, 32, dtype=torch.float32).requires_grad_()
    dx, dw = torch.autograd.grad(fp4.linear(x, w).sum(), (x, w))
    assert dx.shape == (0, 32) and bool((dw == 0).all())
    q, s = stored(8, 32)
    y = fp4.linear(x, q, s)
    assert y.shape == (0, 8) and torch.autograd.grad(y.sum(), x)[0].shape == (0, 32)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3)])
def test_results_can_be_changed_in_place(lead):
    x, w = normal(*lead, 40).requires_grad_(), normal(30, 40, seed=2).requires_grad_()
    b, (q, s) = normal(30, seed=3).requires_grad_(), stored(30, 40)
    for f in (lambda: fp4.linear(x, w), lambda: fp4.linear(x, w, bias=b), lambda: fp4.linear(x, q, s, b)):
        y = f()
        y += 1.0
        got, want = (torch.autograd.grad(v.float().square().sum(), (x, w, b), allow_unused=True) for v in (y, f() + 1.0))
        assert [g is None for g in got] == [g is None for g in want]
        assert all(torch.equal(a, c) for a, c in zip(got, want) if a is not None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 30, 40), (12, 130, 200), (300, 257, 384), (64, 256, 1500)])
def test_a_bias_is_added_before_the_one_rounding(M, N, K, dtype):
    x, w = normal(M, K, dtype=dtype), normal(N, K, dtype=dtype, seed=2)
    b = normal(2 * N, dtype=dtype, seed=3, std=30.0)[::2]  # (strided)
    y = fp4.linear(x, w, bias=b)
    ref.check_product(y, ref.rounded(x), ref.rounded(w), b)
    grown = [t.detach().requires_grad_() for t in (x, w, b)]
    z = fp4.linear(*grown[:2], bias=grown[2])
    assert torch.equal(z, y)
    assert torch.equal(torch.autograd.grad(z.float().sum(), grown[2])[0], torch.full_like(b, M))


def test_same_bits_every_time_and_on_any_stream():
    x, (w, ws) = normal(200, 1000), stored(400, 1000)
    want = fp4.linear(x, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [fp4.linear(x, w, ws) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_graph_replays_match_eager():
    w, ws = stored(300, 512)
    for M in (3, 100):
        x = normal(M, 512)
        fp4.linear(x, w, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fp4.linear(x, w, ws)
            v = fp4.dequantize(*fp4.quantize(x))
        for i in range(3):
            x.copy_(normal(M, 512, seed=20 + i))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, fp4.linear(x, w, ws)) and torch.equal(v, fp4.dequantize(*fp4.quantize(x)))


def test_a_layer_quantised_served_and_tuned():
    """The operators as they are used together: a weight quantised once, then read by every form of the product."""
    x, w = normal(40, 320, dtype=torch.bfloat16), normal(160, 320, dtype=torch.bfloat16, seed=2, std=0.05)
    wq, ws = fp4.quantize(w)
    y = fp4.linear(x, wq, ws)
    q, s = fp4.quantize(x)
    assert torch.equal(y, fp4.mm(q, s, wq.t(), ws.t(), torch.bfloat16)) and torch.equal(y, fp4.linear(x, w))
    assert all(torch.equal(fp4.linear(x[i:i + 1], wq, ws).float(), f) for i, f in enumerate(
        fp4.linear(x[:8], wq, ws).float().split(1)))  # few tokens: a token's result whatever is beside it
    ref.check_product(y, ref.values(q, s), ref.values(wq, ws))
    v = fp4.dequantize(wq, ws, torch.bfloat16)
    again = fp4.quantize(v)  # what 4 bits hold they hold again
    assert torch.equal(fp4.dequantize(*again, torch.bfloat16), v)


def test_refusals():
    x, (w, ws) = normal(4, 256), stored(64, 256)
    q, s = fp4.quantize(x)
    bad = [lambda: fp4.quantize(x.double()), lambda: fp4.quantize(x.cpu()), lambda: fp4.quantize(normal(2, 3, 4), True),
           lambda: fp4.quantize(q), lambda: fp4.linear(x, w), lambda: fp4.linear(x, w, ws[:, :1]),
           lambda: fp4.linear(x, w, u8(ws)), lambda: fp4.linear(x[:, :128], w, ws), lambda: fp4.linear(x, w.cpu(), ws),
           lambda: fp4.linear(x, w, ws, normal(63)), lambda: fp4.linear(x, w, ws, normal(64, dtype=torch.float32)),
           lambda: fp4.linear(x, x[:, :128], ws), lambda: fp4.linear(x, u8(w), ws), lambda: fp4.linear(q, w, ws),
           lambda: fp4.mm(q, s, w, ws), lambda: fp4.mm(q, s[:, :1], w.t(), ws.t()), lambda: fp4.mm(q, s, w.t(), ws),
           lambda: fp4.mm(x, s, w.t(), ws.t()), lambda: fp4.mm(q, s, w.t(), ws.t(), torch.int8),
           lambda: fp4.mm(q, u8(s), w.t(), ws.t()), lambda: fp4.mm(q[0], s, w.t(), ws.t()),
           lambda: fp4.dequantize(q, s[:, :2]), lambda: fp4.dequantize(u8(q), s), lambda: fp4.dequantize(q, u8(s)),
           lambda: fp4.dequantize(q, s, torch.float64), lambda: fp4.dequantize(q, s.cpu())]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_mm_tile_refuses_what_does_not_fit():
    M, N, K = 40, 72, 256
    a, sa = stored(M, K, seed=2)
    w, ws = stored(N, K)
    f = lambda out, bias=None, tile=4, splits=1: fp4.mm_tile(a, sa, w.t(), ws.t(), out, tile, splits, bias)
    out = torch.empty(M, N, device=DEV)
    short, pair = torch.zeros(N - 1, device=DEV), torch.zeros(1, N, device=DEV)
    bad = [lambda: f(torch.empty(M + 1, N, device=DEV)), lambda: f(torch.empty(M, device=DEV)), lambda: f(out.int()),
           lambda: f(out.double()), lambda: f(out.cpu()), lambda: f(out[:1].expand(M, N)), lambda: f(out, short),
           lambda: f(out, pair), lambda: f(out, pair[0].half()), lambda: f(out, pair[0].cpu()),
           lambda: f(out, tile=6), lambda: f(out, tile=-2), lambda: f(out, splits=-1)]
    for g in bad:
        with pytest.raises(ValueError):
            g()
    none = torch.zeros(5, 0, dtype=torch.uint8, device=DEV)
    out, bias = torch.full((5, 7), 3.0, device=DEV), normal(7, dtype=torch.float32)
    b = torch.zeros(0, 7, dtype=torch.uint8, device=DEV)
    fp4.mm_tile(none.view(F4), none.view(E8), b.view(F4), b.view(E8), out, -1, 0, bias)
    assert torch.equal(out, bias.expand(5, 7))


def test_rows_and_scales_more_than_4_mib_apart():
    M, N, K, far = 20, 24, 256, (1 << 22) + 64
    a, sa = stored(M, K, seed=2)
    w, ws = stored(N, K)
    want = fp4.mm(a, sa, w.t(), ws.t(), torch.float32)
    pool = torch.zeros(N * far, dtype=torch.uint8, device=DEV)
    apart = lambda t, d: pool[:t.shape[0] * far].view(t.shape[0], far)[:, :t.shape[1]].copy_(u8(t)).view(d)
    assert torch.equal(fp4.mm(apart(a, F4), sa, w.t(), ws.t(), torch.float32), want)
    assert torch.equal(fp4.mm(a, sa, apart(w, F4).t(), ws.t(), torch.float32), want)
    assert torch.equal(fp4.mm(a, sa, w.t(), apart(ws, E8).t(), torch.float32), want)
    for x in (normal(M, K), normal(3, K)):
        y = fp4.linear(x, w, ws)
        assert torch.equal(fp4.linear(x, apart(w, F4), ws), y) and torch.equal(fp4.linear(x, w, apart(ws, E8)), y)


@pytest.mark.parametrize("ldw", [0, 16, 1 << 40])
@pytest.mark.parametrize("K", [288, 250, 1024])
def test_linear_of_a_single_weight_row(K, ldw):
    """The C entry point with one weight row: the bytes between rows address nothing, whatever a caller holds there."""
    w, ws = stored(1, K)
    for M in (1, 7, 40, 300):
        x = normal(M, K)
        y = torch.full((M, 1), 7.0, dtype=torch.float16, device=DEV)
        n = _ops.linear_fp4_workspace(M, 1, K, w.data_ptr(), ldw)
        held = torch.full((max(n, 1),), 255, dtype=torch.uint8, device=DEV)
        args = (x.data_ptr(), 0, K, 1, w.data_ptr(), ldw, ws.data_ptr(), 1, 1, None, y.data_ptr(), M, 1, K, held.data_ptr(), n)
        assert _ops.linear_fp4(*args, torch.cuda.current_stream().cuda_stream) == 0
        ref.check_product(y, ref.rounded(x), ref.values(w, ws, K))
        assert torch.equal(y, fp4.linear(x, w, ws))


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 7, 31), (40, 72, 333), (300, 130, 1025), (20, 40, 8961)])
def test_mm_of_an_odd_number_of_values(M, N, K):
    """The C entry point: the high half of a row's last byte is no value of an odd K, whatever it holds."""
    (a, sa), (w, ws) = stored(M, K, seed=2), stored(N, K)
    for q, code in ((a, 0x70), (w, 0xa0)):
        u8(q)[:, -1] += code
    stride = lambda q, s: (q.data_ptr(), *q.stride(), s.data_ptr(), *s.stride(), 0)
    for x, y in ((a, w), (u8(a).t().contiguous().t(), u8(w).t().contiguous().t())):
        n = _ops.mm_fp4_workspace(x.data_ptr(), *x.stride(), 0, y.data_ptr(), *y.stride(), 0, M, N, K, -1, 0)
        held = torch.full((max(n, 1),), 255, dtype=torch.uint8, device=DEV)
        c = torch.full((M, N), 7.0, device=DEV)
        assert _ops.mm_fp4(*stride(x, sa), *stride(y, ws), None, c.data_ptr(), N, 1, M, N, K, 2, -1, 0, held.data_ptr(), n,
                           torch.cuda.current_stream().cuda_stream) == 0
        ref.check_product(c, ref.values(a, sa, K), ref.values(w, ws, K))


@pytest.mark.parametrize("N", [(1 << 27) - 16, (1 << 27) - 1])
def test_linear_of_more_weight_rows_than_a_launch_of_the_small_kernel_holds(N):
    """One value times each of 2^27 weights: products of a power of two and a 4-bit value, exact."""
    w = torch.arange(N, device=DEV).bitwise_and_(15).to(torch.uint8)[:, None]
    s = torch.full((N, 1), 127, dtype=torch.uint8, device=DEV)
    y = fp4.linear(torch.full((1, 1), 4.0, dtype=torch.float16, device=DEV), w.view(F4), s.view(E8))
    table = 4 * ref.unpack(torch.arange(16, dtype=torch.uint8)[:, None], 1).half().to(DEV)[:, 0]
    assert torch.equal(y[0, :N // 16 * 16].view(-1, 16), table.expand(N // 16, 16))
    assert torch.equal(y[0, N // 16 * 16:], table[:N % 16])


@pytest.mark.parametrize("M,N,K", [(1, 8000, 5001), (16, 300, 1001), (3, 500, 4096)])
def test_few_tokens_allocate_the_result_alone(M, N, K):
    """A weight of odd rows is not copied for them, and no room for a copy is asked for."""
    x, (w, ws) = normal(M, K), stored(N, K)
    assert _ops.linear_fp4_few(M, N, K, 1) == 1
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y = fp4.linear(x, w, ws)
    assert torch.cuda.max_memory_allocated() - before <= -(-2 * M * N // 512) * 512
    ref.check_product(y, ref.rounded(x), ref.values(w, ws, K))
    z = torch.empty_like(y)
    assert _ops.linear_fp4(x.data_ptr(), 0, K, 1, w.data_ptr(), w.stride(0), ws.data_ptr(), *ws.stride(), None, z.data_ptr(), M, N,
                           K, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(z, y)
    every = normal(M, 2 * K)[:, ::2]  # (columns apart: the tiles, with a workspace)
    ref.check_product(fp4.linear(every, w, ws), ref.rounded(every), ref.values(w, ws, K))


@pytest.mark.parametrize("N,K,most", [(40, 100, 16), (530, 3000, 16), (520, 3200, 16), (4112, 2048, 16), (4096, 4000, 16),
                                      (4096, 4096, 16), (4100, 4097, 7), (8192, 4096, 8)])
@pytest.mark.parametrize("dtype", TYPES)
def test_few_tokens_results_do_not_depend_on_those_beside_them(N, K, most, dtype):
    """Bit for bit, for as many tokens as one kernel takes."""
    x, (w, ws) = normal(most, K, dtype=dtype), stored(N, K)
    assert _ops.linear_fp4_few(most, N, K, 1) == 1 and (most == 16 or _ops.linear_fp4_few(most + 1, N, K, 1) == 0)
    rows = torch.cat([fp4.linear(x[i:i + 1], w, ws) for i in range(most)])
    for M in range(2, most + 1):
        assert torch.equal(fp4.linear(x[:M], w, ws), rows[:M])
    assert torch.equal(fp4.linear(x.flip(0), w, ws).flip(0), rows)

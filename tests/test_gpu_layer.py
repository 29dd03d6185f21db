"""The whole mixture-of-experts layer on the GPU: the router's product, the choice, the experts."""

import itertools

import pytest
import torch

from f16acc_amd import _ops, moe
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, F8, normal, weight
from tests.test_gpu_moe import check_experts

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
OPTIONS = [dict(), dict(scoring="sigmoid"), dict(renormalize=False, scale=2.5)]


def layer(T, E, D, I, dtype=torch.float16, rtype=None, seed=0):
    """x, router, (w1, s1, w2, s2)."""
    x = normal(T, D, dtype=dtype, seed=seed)
    router = normal(E, D, dtype=rtype or dtype, seed=seed + 7, std=1.5 / D ** 0.5)
    return x, router, (*weight(E, 2, I, D, seed=seed + 1), *weight(E, D, I, seed=seed + 2))


def logits_of(x, router):
    """In 64 bits, one rounding."""
    return (x.cpu().double() @ router.cpu().double().t()).float()


def check_layer(y, x, router, k, w, **kw):
    """By the experts' bound.  The choice is FP32's of logits that are rounded once: it is the reference's unless two
    keys lie closer than FP32 tells apart, which these inputs do not hold."""
    bias = kw.get("bias")
    weights, ids, gap = ref.route(logits_of(x, router), k, **kw)
    assert gap > 1e-6 or bias is None
    check_experts(y, (x, weights, ids, *w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,k,D,I", [(1, 1, 1, 16, 16), (1, 8, 3, 256, 128), (2, 4, 4, 130, 70), (3, 20, 4, 1040, 720),
                                       (4, 9, 4, 200, 300), (1, 64, 6, 2048, 1024), (1, 1024, 16, 128, 128),
                                       (2, 300, 8, 384, 132), (5, 3, 2, 200, 300), (16, 8, 4, 256, 384), (40, 5, 2, 272, 144),
                                       (17, 130, 3, 128, 128), (300, 3, 3, 384, 256), (1, 30, 17, 128, 128),
                                       (1, 600, 2, 8, 8), (2, 16, 8, 4096, 512)])
def test_layer(T, E, k, D, I, dtype):
    x, router, w = layer(T, E, D, I, dtype)
    y = moe.layer(x, router, k, *w)
    assert y.dtype == dtype and y.shape == x.shape
    check_layer(y, x, router, k, w)


@pytest.mark.parametrize("T,E,k,D,I", [(2, 16, 8, 256, 4096), (4, 9, 4, 1100, 2000), (1, 20, 16, 300, 3000)])
def test_more_pieces_than_workgroups_at_once(T, E, k, D, I):
    x, router, w = layer(T, E, D, I, torch.bfloat16)
    for _ in range(3):
        check_layer(moe.layer(x, router, k, *w), x, router, k, w)


@pytest.mark.parametrize("T,E,D,dtype,rtype", [(2017, 490, 100, torch.float16, torch.float16),
                                               (1000, 1024, 130, torch.bfloat16, torch.float32),
                                               (33000, 20, 48, torch.float32, torch.bfloat16)])
def test_many_logits(T, E, D, dtype, rtype):
    """Sums of whole numbers, exact in any order: tiles of 32 tokens and 32 experts, ragged at their ends."""
    g = torch.Generator().manual_seed(T)
    x = torch.randint(-3, 4, (T, D), generator=g).to(dtype).to(DEV)
    router = torch.randint(-3, 4, (E, D), generator=g).to(rtype).to(DEV) / 16
    w1, s1 = weight(1, 2, 16, D)
    w2, s2 = weight(1, D, 16)
    scale = s2.repeat(E, 1, 1) * torch.exp2(torch.arange(E, device=DEV) % 16).float()[:, None, None]  # the choice shows
    w = (w1.expand(E, 2, 16, D).contiguous(), s1.repeat(E, 1, 1, 1), w2.expand(E, D, 16).contiguous(), scale)
    weights, ids = moe.route((x.double() @ router.double().t()).float(), 2)
    assert torch.equal(moe.layer(x, router, 2, *w), moe.experts(x, weights, ids, *w))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 33])
@pytest.mark.parametrize("dtype,rtype", list(itertools.product(TYPES, TYPES)))
def test_router_types(T, dtype, rtype):
    x, router, w = layer(T, 12, 200, 144, dtype, rtype, seed=3)
    check_layer(moe.layer(x, router, 3, *w), x, router, 3, w)


@pytest.mark.parametrize("T", [1, 4, 20])
@pytest.mark.parametrize("E", [24, 96, 200, 520])
def test_options(T, E):
    x, router, w = layer(T, E, 256, 128, seed=E)
    bias = normal(E, dtype=torch.float32, seed=5, std=0.2)
    for kw in (*OPTIONS, dict(groups=4, top_groups=2), dict(scoring="sigmoid", groups=8, top_groups=3),
               dict(scoring="sigmoid", groups=E // 2, top_groups=E // 4) if E <= 96 else dict(groups=8, top_groups=8)):
        check_layer(moe.layer(x, router, 4, *w, **kw), x, router, 4, w, **kw)
        kw = dict(kw, bias=bias)
        check_layer(moe.layer(x, router, 4, *w, **kw), x, router, 4, w, **kw)


def test_a_token_chooses_alike_in_every_batch():
    """Logits an FP32 sum's error apart (8 steps of FP32 at 64 here): the choice is that of the 64-bit sums, for every
    number of tokens beside it, and so is each token's result up to its kernel's own sums."""
    D, E = 1024, 16
    x = normal(40, D, dtype=torch.float32, seed=1)
    router = normal(1, D, dtype=torch.float32, seed=2).expand(E, D).contiguous()
    router[:, 0] += torch.arange(E, device=DEV) * 2.0 ** -18  # every token's 16 logits lie within 1e-4
    w1, s1 = weight(1, 2, 128, D)
    w2, s2 = weight(1, D, 128)
    s2 = s2.repeat(E, 1, 1) * torch.exp2(torch.arange(E, device=DEV).float())[:, None, None]  # the choice shows
    w = (w1.expand(E, 2, 128, D).contiguous(), s1.repeat(E, 1, 1, 1), w2.expand(E, D, 128).contiguous(), s2)
    rows = moe.layer(x, router, 2, *w)
    for n in (1, 2, 3, 4, 7, 19):
        for t in range(0, 40 - n, 5):
            y = moe.layer(x[t:t + n], router, 2, *w)
            assert bool(((y - rows[t:t + n]).norm(dim=1) <= 2e-2 * rows[t:t + n].norm(dim=1)).all()), (n, t)
    weights, ids, _ = ref.route(logits_of(x, router), 2)  # (equal logits: the lowest expert first)
    check_experts(rows, (x, weights, ids, *w))


@pytest.mark.parametrize("T", [1, 3, 40])
def test_ties_and_padding_rows(T):
    """Rows of zeros have logits of zero: the lowest experts, in order."""
    x, router, w = layer(T, 20, 256, 128)
    x[T - 1] = 0.0
    assert bool((moe.layer(x, router, 3, *w)[T - 1] == 0).all())
    x[0] = 1.0
    router[:] = 0.25
    weights, ids = torch.full((T, 3), 1.0 / 3, device=DEV), torch.arange(3, device=DEV).expand(T, 3)
    check_experts(moe.layer(x, router, 3, *w), (x, weights, ids, *w))


@pytest.mark.parametrize("T", [1, 2, 4, 6, 60])
def test_experts_that_are_not_available(T):
    """A router row with an infinity makes its logits -inf or NaN for the tokens that reach it."""
    x, router, w = layer(T, 6, 256, 128)
    x = x.abs()
    good = moe.layer(x, router, 2, *w)
    router[1:, 5] = -float("inf")  # one expert is left
    y = moe.layer(x, router, 2, *w)
    weights = torch.zeros(T, 2, device=DEV)
    weights[:, 0] = 1.0
    ids = torch.tensor([0, -1], device=DEV).expand(T, 2)
    check_experts(y, (x, weights, ids, *w))
    router[0, 5] = -float("inf")  # none is left
    assert bool((moe.layer(x, router, 2, *w) == 0).all())
    router = normal(6, 256, seed=7, std=0.1)
    bad = x.clone()
    bad[T - 1, 17] = float("nan")
    y, want = moe.layer(bad, router, 2, *w), moe.layer(x, router, 2, *w)
    assert bool(torch.isnan(y[T - 1]).all()) and torch.equal(y[:T - 1], want[:T - 1])
    assert bool(torch.isfinite(good).all())


@pytest.mark.parametrize("T", [1, 4, 9, 100])
def test_views_and_leading_dimensions(T):
    x, router, w = layer(T, 20, 256, 144)
    want = moe.layer(x, router, 3, *w)
    views = [torch.cat([x, x], 1)[:, :256], x.t().contiguous().t(), torch.cat([x[:, :1], x], 1)[:, 1:],
             x.repeat_interleave(3, 0)[::3], x.repeat_interleave(2, 1)[:, ::2]]
    for v in views:
        check_experts(moe.layer(v, router, 3, *w), (x, *ref.route(logits_of(x, router), 3)[:2], *w))
    for r in (router.t().contiguous().t(), torch.cat([router[:, :1], router], 1)[:, 1:], router.repeat(2, 1)[:20]):
        assert torch.equal(moe.layer(x, r, 3, *w), want)
    moved = (w[0].transpose(2, 3).contiguous().transpose(2, 3), w[1].transpose(2, 3).contiguous().transpose(2, 3),
             torch.cat([w[2].view(torch.uint8)] * 2, 2).view(F8)[:, :, :144], w[3].repeat(1, 2, 1)[:, :2])
    assert torch.equal(moe.layer(x, router, 3, *moved), want)
    odd = torch.cat([w[2].view(torch.uint8)[:, :, :1], w[2].view(torch.uint8)], 2)[:, :, 1:].view(F8)
    assert torch.equal(moe.layer(x, router, 3, w[0], w[1], odd, w[3]), want)
    y = moe.layer(x[None, :, None], router, 3, *w)
    assert y.shape == (1, T, 1, 256) and torch.equal(y.view(T, 256), want)
    assert moe.layer(x[:0], router, 3, *w).shape == (0, 256)
    if T == 1:
        assert torch.equal(moe.layer(x[0], router, 3, *w), want[0])


@pytest.mark.parametrize("T", [1, 3, 50])
def test_same_bits_any_stream_several_at_once_and_graph_replays(T):
    x, router, w = layer(T, 40, 512, 384)
    want = moe.layer(x, router, 4, *w)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for side in sides:  # calls that run beside each other share nothing
            with torch.cuda.stream(side):
                outs.append(moe.layer(x, router, 4, *w))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = moe.layer(x, router, 4, *w)
            z = moe.layer(y, router, 4, *w)
        graphs.append((graph, y, z))
    for i in range(3):
        x.copy_(normal(T, 512, seed=30 + i))
        for graph, y, z in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = moe.layer(x, router, 4, *w)
        for graph, y, z in graphs:
            assert torch.equal(y, want) and torch.equal(z, moe.layer(want, router, 4, *w))


def test_workspace_of_garbage_and_rows_around():
    """The C entry point on a workspace of NaN bytes, results between rows that keep what they hold."""
    for T, k in ((1, 3), (4, 4), (30, 2)):
        E, D, I = 10, 256, 128
        x, router, (w1, s1, w2, s2) = layer(T, E, D, I)
        want = moe.layer(x, router, k, w1, s1, w2, s2)
        n = _ops.layer_workspace(T, k, E, D, I)
        ws = torch.full((n + 256,), 255, dtype=torch.uint8, device=DEV)
        out = torch.full((T + 2, D), 7.0, dtype=torch.float16, device=DEV)
        stream = torch.cuda.current_stream().cuda_stream
        args = [x.data_ptr(), 0, T, D, 1, router.data_ptr(), 0, D, 1, E, k, 0, None, 1, 1, 1, 1.0, D, I, w1.data_ptr(),
                2 * I * D, I * D, D, s1.data_ptr(), *s1.stride(), w2.data_ptr(), I * D, I, s2.data_ptr(), *s2.stride(),
                out[1].data_ptr(), ws.data_ptr()]
        for _ in range(2):  # and on what the first call left there
            assert _ops.layer(*args, n, stream) == 0
            assert torch.equal(out[1:-1], want)
        assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all()) and bool((ws[n:] == 255).all())
        assert _ops.layer(*args, n - 1, stream) == _ops.E_WORKSPACE


def test_layer_is_route_and_experts():
    for T in (4, 64, 700):
        x, router, w = layer(T, 16, 256, 128, torch.bfloat16)
        with torch.inference_mode():
            y = moe.layer(x, router, 4, *w, scoring="sigmoid", scale=1.5)
            weights, ids = moe.route(logits_of(x, router).to(DEV), 4, scoring="sigmoid", scale=1.5)
            z = moe.experts(x, weights, ids, *w)
        check_experts(y, (x, weights, ids, *w))
        assert (y - z).float().norm() <= 1e-2 * z.float().norm()


def test_refusals():
    x, router, w = layer(4, 8, 256, 128)
    args = [x, router, 2, *w]

    def swap(i, v, **kw):
        a = list(args)
        a[i] = v
        return lambda: moe.layer(*a, **kw)

    bad = [swap(0, x.double()), swap(0, x[:, :128]), swap(0, x.cpu()), swap(1, router[:7]), swap(1, router[:, :128]),
           swap(1, router.double()), swap(1, router.to(F8)), swap(1, router.cpu()), swap(2, 0), swap(2, 9), swap(3, w[0].half()),
           swap(3, w[0][:7]), swap(4, w[1].half()), swap(5, w[2][:, :128]), swap(6, w[3][:, :1]),
           swap(2, 2, scoring="relu"), swap(2, 2, groups=3), swap(2, 5, groups=4, top_groups=2), swap(2, 2, groups=2, top_groups=3),
           swap(2, 2, bias=normal(8)), swap(2, 2, bias=normal(7, dtype=torch.float32))]
    bad += [swap(i, args[i].detach().clone().requires_grad_()) for i in (0, 1, 3, 4, 5, 6)]
    bad += [swap(2, 2, bias=normal(8, dtype=torch.float32).requires_grad_())]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with torch.no_grad():
        moe.layer(x.clone().requires_grad_(), *args[1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 3, 4, 5, 40, 1100])
def test_choice_of_exact_sums_is_the_same_in_every_batch(T, dtype):
    """Logits of 35 bits, exact in 64 in any order, that lie two steps of FP32 apart (or one, or none) where an FP32 sum is
    off by more: the kernels for few, some and many tokens choose alike."""
    E, D, I = 1024, 256, 16
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-7, 8, (1100, D), generator=g).float()
    x[:, 0] = 1.0
    base = torch.randint(-2 ** 23 + 2 ** 17, 2 ** 23 - 2 ** 17, (D,), generator=g).float()
    router = base.repeat(E, 1)
    router[:, 0] = 64.0 * torch.randperm(E, generator=g)
    router = (router * 2.0 ** -26).to(DEV)
    x = x.to(dtype).to(DEV)[1100 - T:]
    w1, s1 = weight(1, 2, I, D)
    w2, s2 = weight(1, D, I)
    scale = s2.repeat(E, 1, 1) * torch.exp2(torch.arange(E, device=DEV) % 16).float()[:, None, None]  # the choice shows
    w = (w1.expand(E, 2, I, D).contiguous(), s1.repeat(E, 1, 1, 1), w2.expand(E, D, I).contiguous(), scale)
    weights, ids = moe.route(logits_of(x, router).to(DEV), 3)
    y = moe.layer(x, router, 3, *w)
    if T > 4:
        assert torch.equal(y, moe.experts(x, weights, ids, *w))
    else:
        check_experts(y, (x, weights, ids, *w))


@pytest.mark.parametrize("T,E,k,D,I", [(1, 8, 2, 256, 6000), (2, 16, 8, 256, 4096), (4, 9, 4, 1104, 2000), (3, 6, 1, 136, 9001),
                                       (4, 5, 2, 1040, 3117), (1, 20, 16, 304, 3000)])
def test_wide_hidden_layers_of_few_tokens(T, E, k, D, I):
    """Far more hidden columns than workgroups at once: the composed kernels where x's rows load wide, the two launches
    where they do not (and compute each other's pieces); weights whose rows start anywhere; tokens of NaN and without experts."""
    x, router, w = layer(T, E, D, I, torch.bfloat16)
    apart = torch.cat([x[:, :1], x], 1)[:, 1:]
    odd = torch.cat([w[2].view(torch.uint8)[:, :, :1], w[2].view(torch.uint8)], 2)[:, :, 1:].view(F8)
    for v in (x, apart):
        y = moe.layer(v, router, k, *w)
        check_layer(y, x, router, k, w)
        for _ in range(3):
            assert torch.equal(moe.layer(v, router, k, *w), y)
        assert torch.equal(moe.layer(v, router, k, w[0], w[1], odd, w[3]), y)
        bad = v.clone() if v is x else torch.cat([x[:, :1], x], 1)[:, 1:]
        bad[T - 1, 17] = float("nan")
        z = moe.layer(bad, router, k, *w)
        assert bool(torch.isnan(z[T - 1]).all()) and torch.equal(z[:T - 1], y[:T - 1])
        none = router.clone()
        none[:, 5] = -float("inf")
        assert bool((moe.layer(v.abs() + 1, none, k, *w) == 0).all())


def test_more_tokens_than_a_launch_addresses_go_in_parts():
    """Rows of 4 MiB quantised: 511 tokens a part, the last part's two tokens by the kernels for few."""
    T, D, I = 513, 1 << 22, 16
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(T, D, generator=g, device=DEV, dtype=torch.bfloat16)
    router = torch.randn(2, D, generator=g, device=DEV, dtype=torch.bfloat16) * D ** -0.5
    w = []
    for shape in ((2, 2, I, D), (2, D, I)):
        w.append((torch.randn(*shape, generator=g, device=DEV) * 100).clamp_(-448, 448).to(F8))
        blocks = (*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128))
        w.append(torch.rand(*blocks, generator=g, device=DEV) * 2e-5)
    y = moe.layer(x, router, 1, *w)
    assert bool(torch.isfinite(y).all())
    assert torch.equal(y[:511], moe.layer(x[:511], router, 1, *w)) and torch.equal(y[511:], moe.layer(x[511:], router, 1, *w))
    weights, ids = moe.route((x[505:].double() @ router.double().t().contiguous()).float(), 1)
    z = moe.experts(x[505:], weights, ids, *w).float()
    assert len(ids.unique()) == 2 and bool(((y[505:].float() - z).norm(dim=1) <= 1e-2 * z.norm(dim=1)).all())


def test_wide_hidden_layers_on_a_workspace_of_garbage():
    T, k, E, D, I = 2, 4, 10, 256, 4000
    x, router, (w1, s1, w2, s2) = layer(T, E, D, I)
    want = moe.layer(x, router, k, w1, s1, w2, s2)
    n = _ops.layer_workspace(T, k, E, D, I)
    ws = torch.full((n + 256,), 255, dtype=torch.uint8, device=DEV)
    out = torch.full((T + 2, D), 7.0, dtype=torch.float16, device=DEV)
    for _ in range(2):
        assert _ops.layer(x.data_ptr(), 0, T, D, 1, router.data_ptr(), 0, D, 1, E, k, 0, None, 1, 1, 1, 1.0, D, I, w1.data_ptr(),
                          2 * I * D, I * D, D, s1.data_ptr(), *s1.stride(), w2.data_ptr(), I * D, I, s2.data_ptr(), *s2.stride(),
                          out[1].data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[1:-1], want)
    assert bool((out[0] == 7).all()) and bool((out[-1] == 7).all()) and bool((ws[n:] == 255).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = moe.layer(x, router, k, w1, s1, w2, s2)
    for i in range(3):
        x.copy_(normal(T, D, seed=30 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, moe.layer(x, router, k, w1, s1, w2, s2))

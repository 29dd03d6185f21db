"""Routing and the experts' feed-forward on the GPU against plain 64-bit statements."""

import pytest
import torch

from f16acc_amd import fp8, moe
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, normal, weight

pytestmark = pytest.mark.gpu
INF = float("inf")


def grid(T, E, seed=0, step=64, dtype=torch.float32):
    """Scores on a grid, so that keys are either tied or clearly apart."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-4 * step, 4 * step + 1, (T, E), generator=g).float() / step).to(dtype).to(DEV)


def check_route(x, k, **kw):
    w, i = moe.route(x, k, **kw)
    want_w, want_i, gap = ref.route(x, k, **kw)
    assert gap > 1e-6, "the inputs hold keys that FP32 cannot tell apart"
    assert i.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(i.cpu().long(), want_i)
    assert bool(((w.cpu().double() - want_w).abs() <= 1e-6 * kw.get("scale", 1.0)).all())
    return w, i


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 60, 4), (70, 64, 6), (5, 65, 64), (9, 128, 8), (33, 256, 8),
                                   (4, 257, 5), (6, 512, 10), (3, 1000, 7), (2, 1024, 64)])
def test_route(T, E, k, scoring):
    for renormalize in (True, False):
        check_route(grid(T, E), k, scoring=scoring, renormalize=renormalize)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_route_types_and_strides(dtype):
    x = grid(20, 40, step=8, dtype=dtype)
    want = check_route(x, 4, scale=2.5)
    for v in (x.t().contiguous().t(), torch.cat([x, x], 1)[:, :40], x.repeat_interleave(3, 1)[:, ::3]):
        got = moe.route(v, 4, scale=2.5)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    w, i = moe.route(x.view(4, 5, 40), 4, scale=2.5)
    assert w.shape == i.shape == (4, 5, 4) and torch.equal(i.view(20, 4), want[1])
    one = moe.route(x[3], 4, scale=2.5)
    assert torch.equal(one[1], want[1][3])
    w, i = moe.route(x[:0], 4)
    assert w.shape == i.shape == (0, 4)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top,k", [(256, 8, 4, 8), (60, 4, 2, 6), (16, 16, 3, 3), (64, 64, 8, 8), (48, 2, 1, 24),
                                            (1024, 8, 3, 16), (30, 5, 5, 4)])
def test_route_groups(E, groups, top, k, scoring):
    check_route(grid(25, E, seed=2), k, scoring=scoring, groups=groups, top_groups=top)


def test_route_bias_changes_the_choice_and_not_the_weights():
    bias = (torch.arange(32) % 7).float().mul(0.061).to(DEV)
    for scoring in ("sigmoid", "softmax"):
        check_route(grid(40, 32, step=16), 4, scoring=scoring, bias=bias)
    check_route(grid(40, 32, step=16), 4, scoring="sigmoid", bias=bias, groups=4, top_groups=2)
    bias[3] = -INF
    w, i = check_route(grid(40, 32, step=16), 4, scoring="sigmoid", bias=bias)
    assert not bool((i == 3).any())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(scoring):
    x = torch.zeros(3, 200, device=DEV)
    x[1, ::2] = -0.0
    x[2, 150:] = 1.0
    _, i = moe.route(x, 5, scoring=scoring)
    assert i.tolist() == [[0, 1, 2, 3, 4], [0, 1, 2, 3, 4], [150, 151, 152, 153, 154]]
    _, i = moe.route(x, 3, scoring=scoring, groups=10, top_groups=2)
    # groups of 20: 150 .. 159 lie in group 7 (half of it), 160 .. in group 8; tied groups go to the lower one
    assert i.tolist() == [[0, 1, 2], [0, 1, 2], [150, 151, 152]]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masks(scoring):
    x = grid(12, 24, seed=5)
    x[0] = -INF                     # nothing left
    x[1, 2:] = -INF                 # two left of four
    x[2, ::2] = -INF
    x[3, :] = torch.finfo(torch.float32).min  # the lowest value everywhere: a row like any other
    x[4, 5:] = torch.finfo(torch.float32).min
    w, i = check_route(x, 4, scoring=scoring)
    assert i[0].tolist() == [-1] * 4 and w[0].tolist() == [0.0] * 4
    assert sorted(i[1].tolist()) == [-1, -1, 0, 1]
    check_route(x, 4, scoring=scoring, groups=6, top_groups=3)
    x[5, 7] = float("nan")
    w, i = moe.route(x, 4, scoring=scoring)
    assert bool(torch.isnan(w[5]).all()) and not bool((i[5] == 7).any()) and bool((i[5] >= 0).all())
    assert not bool(torch.isnan(w[[j for j in range(12) if j != 5]]).any())


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 5, 2), (70, 60, 4), (9, 300, 8), (3, 1024, 20)])
def test_route_gradient(T, E, k, dtype, renormalize, scoring):
    x = grid(T, E, step=16, dtype=dtype)
    if T > 2:
        x[1, ::3] = -INF
        x[2] = -INF
    x = x.requires_grad_()
    w, i = moe.route(x, k, scoring=scoring, renormalize=renormalize, scale=1.5)
    assert not i.requires_grad
    dw = normal(T, k, dtype=torch.float32, seed=3)
    dx, = torch.autograd.grad(w, x, dw)
    assert dx.dtype == dtype
    want = ref.route_grad(x, i.cpu().long(), dw, scoring, renormalize, 1.5)
    # FP32 sums of at most 1024 terms of size at most |dw| scale, one rounding
    bound = 1e-6 * 1.5 * dw.abs().sum(1, keepdim=True).cpu().double() + ref.ROUND[dtype] * want.abs() + 2.0 ** -24
    assert bool(((dx.cpu().double() - want).abs() <= bound).all())
    strided, = torch.autograd.grad(moe.route(x, k, scoring=scoring, renormalize=renormalize, scale=1.5)[0], x,
                                   dw.t().contiguous().t())
    assert torch.equal(strided, dx)


def test_route_gradient_against_differences():
    for kw in (dict(scoring="softmax"), dict(scoring="sigmoid"), dict(scoring="softmax", renormalize=False)):
        x = grid(4, 12, seed=8).requires_grad_()
        dw = normal(4, 3, dtype=torch.float32, seed=6)
        w, i = moe.route(x, 3, **kw)
        dx, = torch.autograd.grad(w, x, dw)
        h = 2.0 ** -8
        for t, e in ((0, int(i[0, 0])), (1, int(i[1, 2])), (2, 5), (3, int(i[3, 1]))):
            d = torch.zeros(4, 12, device=DEV)
            d[t, e] = h
            up, ui = moe.route(x.detach() + d, 3, **kw)
            down, di = moe.route(x.detach() - d, 3, **kw)
            assert torch.equal(ui, i) and torch.equal(di, i)
            slope = ((up.double() - down.double()) * dw.double()).sum().item() / (2 * h)
            # third derivative at most |dw|: h^2 / 6 of it; FP32 weights: 2 x 6e-8 / 2 h
            assert abs(slope - dx[t, e].item()) <= dw.abs().sum().item() * (h * h / 6 + 6e-8 / h) + 1e-6


def test_route_refusals():
    x = grid(4, 16)
    bad = [lambda: moe.route(x, 0), lambda: moe.route(x, 17), lambda: moe.route(x, 4, scoring="relu"),
           lambda: moe.route(x, 4, groups=3), lambda: moe.route(x, 4, groups=4, top_groups=5),
           lambda: moe.route(x, 5, groups=4, top_groups=1), lambda: moe.route(x.cpu(), 2), lambda: moe.route(x.int(), 2),
           lambda: moe.route(x, 2, bias=x[0].half()), lambda: moe.route(x, 2, bias=x[0, :8]),
           lambda: moe.route(torch.zeros(2, 1025, device=DEV), 2), lambda: moe.route(torch.zeros((), device=DEV), 1),
           lambda: moe.route(torch.zeros(2, 130, device=DEV), 2, groups=65),
           lambda: moe.route(torch.zeros(2, 100, device=DEV), 65)]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def layer(T, E, k, D, I, dtype=torch.float16, seed=0, dropped=0.0):
    g = torch.Generator().manual_seed(seed)
    x = normal(T, D, dtype=dtype, seed=seed)
    ids = torch.rand(T, E, generator=g).topk(k, dim=1).indices.to(torch.int32)
    ids[torch.rand(T, k, generator=g) < dropped] = -1
    weights = torch.rand(T, k, generator=g)
    w1, s1 = weight(E, 2, I, D, seed=seed + 1)
    w2, s2 = weight(E, D, I, seed=seed + 2)
    return x, weights.to(DEV), ids.to(DEV), w1, s1, w2, s2


def check_experts(y, args):
    """By the 2-norm: an e4m3 value that the products' error (1e-4) puts on the other side of a tie moves by a
    step, 2^-3 at most: about 1e-4 / 2^-4 of the values, so sqrt(1.6e-3) x 2^-3 = 5e-3, twice that here."""
    want = ref.experts(*args)
    assert bool(torch.isfinite(y).all())
    n = want.norm().item()
    assert (y.cpu().double() - want).norm().item() <= (1e-2 + ref.ROUND[y.dtype]) * n + 1e-30


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,D,I", [(1, 1, 1, 16, 16), (1, 8, 3, 256, 128), (2, 4, 4, 130, 70), (5, 3, 2, 200, 300),
                                       (16, 8, 4, 256, 384), (40, 5, 2, 272, 144), (200, 4, 2, 256, 260), (300, 3, 3, 384, 256),
                                       (700, 4, 2, 128, 640), (1, 1024, 64, 128, 128), (3, 20, 20, 128, 140), (8, 16, 16, 130, 128),
                                       (9, 24, 16, 128, 128), (5, 1000, 3, 128, 16)])
def test_experts(T, E, k, D, I, dtype):
    args = layer(T, E, k, D, I, dtype)
    y = moe.experts(*args)
    assert y.dtype == dtype and y.shape == args[0].shape
    check_experts(y, args)


def test_experts_each_token_gets_its_own():
    """One expert per token, every expert scaling by a factor of its own: a token sent elsewhere shows."""
    for T in (9, 64, 500, 3000):
        x, weights, ids, w1, s1, w2, s2 = layer(T, 40, 1, 128, 128)
        w1[:], w2[:] = w1[:1].clone(), w2[:1].clone()
        s1[:], s2[:] = s1[:1].clone(), s2[:1].clone()
        s2 *= torch.exp2(torch.arange(40, device=DEV).float() % 9).view(40, 1, 1)
        y = moe.experts(x.float(), weights, ids, w1, s1, w2, s2)
        base = moe.experts(x.float(), weights, torch.zeros_like(ids), w1, s1, w2, s2)
        want = base * torch.exp2(ids.float() % 9)
        # the two differ by what their kernels' products do (see check_experts)
        assert ((y - want).norm(dim=1) <= 0.1 * want.norm(dim=1)).all()


@pytest.mark.parametrize("T", [1, 7, 30, 400])
def test_experts_ids_that_are_none(T):
    args = list(layer(T, 6, 3, 256, 128, dropped=0.4))
    check_experts(moe.experts(*args), args)
    args[1] = args[1].masked_fill(args[2] < 0, float("nan"))  # weights of no expert are not read
    assert bool(torch.isfinite(moe.experts(*args)).all())
    args[2] = torch.where(args[2] < 0, torch.tensor([-5, 6, 2 ** 31 - 1], dtype=torch.int32, device=DEV), args[2])
    got = moe.experts(*args)
    assert bool(torch.isfinite(got).all())
    wide = args[2].long()
    wide[args[2] > 5] += 2 ** 32
    assert torch.equal(moe.experts(*args[:2], wide, *args[3:]), got)
    args[2] = torch.full_like(args[2], -1)
    assert bool((moe.experts(*args) == 0).all())


def test_experts_one_expert_has_all_and_uneven_loads():
    for T in (20, 300):
        args = list(layer(T, 7, 2, 256, 256))
        args[2][:] = torch.tensor([3, 5], dtype=torch.int32)
        check_experts(moe.experts(*args), args)
        args[2][:T // 2, 0] = 0
        args[2][:1, 1] = 6
        check_experts(moe.experts(*args), args)
        args[2][:] = 4  # the same expert twice for a token
        check_experts(moe.experts(*args), args)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,E,k,D,I", [(12, 8, 2, 512, 256), (77, 20, 3, 400, 260), (90, 4, 2, 1024, 256),
                                       (800, 4, 2, 512, 256)])
def test_experts_sums_are_exact_for_results_that_show_it(T, E, k, D, I, dtype):
    """By the 2-norm.  Gate and up in FP32 are off by some 5e-7: 8e-6 of the hidden values cross an e4m3 tie and
    move by 2^-3 at most, 3.5e-4 of the norm.  A slot's sum and the result each round to 11 bits: 2^-11 / sqrt(3).
    The root of the squares' sum is 5.3e-4.  (Sums good to 1.5e-5 would cross thirty times as many: 2e-3.)"""
    args = layer(T, E, k, D, I, dtype, seed=11)
    want = ref.experts(*args)
    assert (moe.experts(*args).cpu().double() - want).norm().item() <= 6e-4 * want.norm().item()


def test_experts_views_types_and_leading_dimensions():
    args = list(layer(24, 5, 2, 256, 128))
    want = moe.experts(*args)
    a = list(args)
    a[0] = torch.cat([args[0], args[0]], 1)[:, :256]
    a[1] = args[1].t().contiguous().t()
    a[2] = args[2].long().t().contiguous().t()
    a[3] = args[3].transpose(2, 3).contiguous().transpose(2, 3)
    a[5] = torch.cat([args[5].view(torch.uint8)] * 2, 2).view(args[5].dtype)[:, :, :128]
    a[4], a[6] = (s.transpose(-1, -2).contiguous().transpose(-1, -2) for s in (args[4], args[6]))
    assert torch.equal(moe.experts(*a), want)
    y = moe.experts(args[0].view(2, 12, 256), args[1].view(2, 12, 2), args[2].view(2, 12, 2), *args[3:])
    assert torch.equal(y.view(24, 256), want)
    few = [args[0][:2].clone(), args[1][:2], args[2][:2], *args[3:]]
    check_experts(moe.experts(*few), few)
    few[0] = torch.cat([few[0][:, :1], few[0]], 1)[:, 1:]  # rows that no 16-byte load fits
    check_experts(moe.experts(*few), few)
    empty = moe.experts(args[0][:0], args[1][:0], args[2][:0], *args[3:])
    assert empty.shape == (0, 256)


def test_experts_offsets_past_32_bits():
    T, D = 1100000, 2048
    _, _, _, *w = layer(1, 4, 1, D, 128)
    x = torch.zeros(T, D, dtype=torch.float16, device=DEV)
    tail = normal(600, D)
    x[-600:] = tail
    ids = (torch.arange(T, device=DEV) % 5 - 1).to(torch.int32).view(T, 1)  # -1 .. 3
    weights = torch.ones(T, 1, device=DEV)
    y = moe.experts(x, weights, ids, *w)
    assert bool((y[:-600] == 0).all())
    check_experts(y[-600:], (tail, weights[-600:], ids[-600:], *w))


def test_experts_non_finite_tokens_stay_apart():
    for T in (6, 60, 500):
        args = list(layer(T, 4, 2, 256, 128))
        good = moe.experts(*args)
        args[0][2, 100] = INF
        args[0][4, 3] = float("nan")
        y = moe.experts(*args)
        rest = [t for t in range(T) if t not in (2, 4)]
        assert torch.equal(y[rest], good[rest])
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4]).all())


def test_experts_same_bits_any_stream_and_graph_replays():
    for T in (2, 50, 600):
        args = list(layer(T, 8, 2, 256, 256))
        want = moe.experts(*args)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            outs = [moe.experts(*args) for _ in range(3)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(o, want) for o in outs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = moe.experts(*args)
        for i in range(3):
            args[0].copy_(normal(T, 256, seed=30 + i))
            args[2].copy_(layer(T, 8, 2, 256, 256, seed=40 + i)[2])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, moe.experts(*args))


def test_routed_layer_from_logits():
    x, _, _, *w = layer(100, 16, 4, 256, 128)
    logits = grid(100, 16)
    with torch.inference_mode():
        weights, ids = moe.route(logits, 4)
        y = moe.experts(x, weights, ids, *w)
    want = ref.route(logits, 4)
    check_experts(y, (x, want[0], want[1], *w))


def test_experts_refusals():
    x, wt, ids, w1, s1, w2, s2 = args = layer(4, 4, 2, 256, 128)

    def swap(i, v):
        a = list(args)
        a[i] = v
        return lambda: moe.experts(*a)

    bad = [swap(0, x.double()), swap(0, x[:, :128]), swap(0, x.cpu()), swap(1, wt.half()), swap(1, wt[:, :1]),
           swap(2, ids.float()), swap(2, ids[:3]), swap(3, w1.half()), swap(3, w1[:, :1]), swap(4, s1[:, :, :, :1]),
           swap(4, s1.half()), swap(5, w2[:3]), swap(5, w2.float()), swap(6, s2[:, :1]), swap(0, x.clone().requires_grad_()),
           swap(1, wt.clone().requires_grad_())]
    for f in bad:
        with pytest.raises(ValueError):
            f()

"""The 8-bit layer and the routing inside a training step."""

import pytest
import torch
import torch.nn.functional as F

from f16acc_amd import fp8, moe
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, F8, normal, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(), (5,), (2, 3)])
def test_results_can_be_changed_in_place(lead):
    """y += residual and an in-place activation, as after F.linear; the gradients are those of the plain forms."""
    x, w = normal(*lead, 40).requires_grad_(), normal(30, 40, seed=2).requires_grad_()
    b, (q, s) = normal(30, seed=3).requires_grad_(), weight(30, 40)
    r = normal(*lead, 30, seed=4)
    for f in (lambda: fp8.linear(x, w), lambda: fp8.linear(x, w, bias=b), lambda: fp8.linear(x, q, s, b)):
        y = f()
        y += r
        F.relu(y, inplace=True)
        z = F.relu(f() + r)
        assert torch.equal(y, z)
        got, want = (torch.autograd.grad(v.float().square().sum(), (x, w, b), allow_unused=True) for v in (y, z))
        assert [g is None for g in got] == [g is None for g in want]
        assert all(torch.equal(a, c) for a, c in zip(got, want) if a is not None)
    p, ids = moe.route(x, 3)
    p *= 2.0
    got, = torch.autograd.grad(p.square().sum(), x)
    want, = torch.autograd.grad((2.0 * moe.route(x, 3)[0]).square().sum(), x)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 30, 40), (12, 130, 200), (300, 257, 384), (64, 256, 1500)])
def test_a_bias_is_added_before_the_one_rounding(M, N, K, dtype):
    x, w = normal(M, K, dtype=dtype), normal(N, K, dtype=dtype, seed=2)
    b = normal(2 * N, dtype=dtype, seed=3, std=30.0)[::2]  # (strided)
    want = ref.rounded(x), ref.rounded(w, 128, 128)
    y = fp8.linear(x, w, bias=b)
    ref.check_product(y, *want, b)
    for leaves in ((x,), (w,), (b,), (x, w, b)):
        grown = [t.detach().requires_grad_(any(t is u for u in leaves)) for t in (x, w, b)]
        z = fp8.linear(*grown[:2], bias=grown[2])
        assert torch.equal(z, y) and z.requires_grad
        got = torch.autograd.grad(z.float().sum(), [t for t in grown if t.requires_grad])
        assert all(torch.isfinite(g).all() for g in got)
        if leaves[-1] is b:
            assert torch.equal(got[-1], torch.full_like(b, M))


def test_a_bias_that_a_second_rounding_would_lose():
    # 448 x 4.5 + 32 + 1 = 2049 lies between two binary16 values; with the bias it is 2050, which is one
    x = torch.tensor([[448.0, 1.0, 1.0]], device=DEV).half()
    w = torch.tensor([[4.5, 32.0, 1.0], [448.0, 0.0, 0.0]], device=DEV).half()
    b = torch.ones(2, device=DEV).half()
    for lead in (x.requires_grad_(), x.detach()):
        assert fp8.linear(lead, w, bias=b)[0, 0].item() == 2050.0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N", [(1, 1), (2, 300), (700, 1), (3000, 65), (16384, 40), (257, 2048)])
def test_bias_gradient(M, N, dtype):
    """The sum of a column's gradients in FP32, one rounding; strided and expanded gradients."""
    x, w = normal(M, 16, dtype=dtype), normal(N, 16, dtype=dtype, seed=2)
    q, s = fp8.quantize_weight(w)
    for dy in (normal(M, N, dtype=dtype, seed=3), normal(N, M, dtype=dtype, seed=4).t(),
               normal(N, dtype=dtype, seed=5).expand(M, N), normal(M, 3 * N + 1, dtype=dtype, seed=6)[:, 1::3]):
        exact = dy.double().sum(0)
        bound = M * 2.0 ** -23 * dy.double().abs().sum(0) + ref.ROUND[dtype] * exact.abs() + 2.0 ** -25
        for layer in ((w,), (q, s)):
            b = normal(N, dtype=dtype, seed=7).requires_grad_()
            db, = torch.autograd.grad(fp8.linear(x, *layer, bias=b), b, dy)
            assert db.dtype == dtype and db.shape == b.shape
            assert bool(((db.double() - exact).abs() <= bound).all())
            again, = torch.autograd.grad(fp8.linear(x, *layer, bias=b), b, dy)
            assert torch.equal(again, db)


@pytest.mark.parametrize("M,N,K", [(100, 64, 128), (16384, 1536, 256), (40000, 200, 128)])
def test_recorded_training_steps_replay(M, N, K):
    """Forward and backward in one graph, replayed with other gradients and the program's own sums in between."""
    g = torch.Generator(device=DEV).manual_seed(5)
    fresh = lambda *shape: torch.randn(*shape, generator=g, device=DEV).half()
    x, w, b = fresh(M, K).requires_grad_(), fresh(N, K).requires_grad_(), fresh(N).requires_grad_()
    q, s = fp8.quantize_weight(w.detach())
    dy = fresh(M, N)

    def step():
        return (*torch.autograd.grad(fp8.linear(x, w, bias=b), (x, w, b), dy),
                *torch.autograd.grad(fp8.linear(x, q, s, b), (x, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        dy.copy_(fresh(M, N))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.randn(1000, 1000, device=DEV).sum()
        torch.cuda.synchronize()
        for name, a, c in zip(("dx", "dw", "db", "stored dx", "stored db"), out, want):
            assert torch.equal(a, c), name


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 130, 200), (3, 1, 70), (9, 128, 128), (17, 260, 129), (130, 96, 272),
                                   (257, 300, 520), (500, 77, 1000)])
def test_stored_weight_gradients(M, N, K, dtype):
    x = normal(M, K, dtype=dtype).requires_grad_()
    b = normal(N, dtype=dtype, seed=5).requires_grad_()
    w, s = weight(N, K)
    dy = normal(M, N, dtype=dtype, seed=3)
    dx, db = torch.autograd.grad(fp8.linear(x, w, s, b), (x, b), dy)
    ref.check_product(dx, ref.rounded(dy), ref.values(w, s, 128).t())
    exact = dy.double().sum(0).cpu()
    # FP32 sums of M terms, one rounding
    bound = M * 2.0 ** -23 * dy.double().abs().sum(0).cpu() + ref.ROUND[dtype] * exact.abs() + 1e-30
    assert db.dtype == dtype and bool(((db.double().cpu() - exact).abs() <= bound).all())
    alone, = torch.autograd.grad(fp8.linear(x, w, s), x, dy)
    assert torch.equal(alone, dx)
    # the same weight in other layouts, the same gradient of another
    wide = torch.full((N, K + 5), float("nan")).to(F8).to(DEV)
    wide[:, 3:K + 3] = w
    for v in (w.t().contiguous().t(), wide[:, 3:K + 3]):
        other, = torch.autograd.grad(fp8.linear(x, v, s, b), x, dy.t().contiguous().t())
        assert torch.equal(other, dx)
    cube = x.detach().view(M, 1, K).requires_grad_()
    other, = torch.autograd.grad(fp8.linear(cube, w, s), cube, dy.view(M, 1, N))
    assert torch.equal(other.view(M, K), dx)

"""The 8-bit layer and the routing inside a training step."""

import pytest
import torch
import torch.nn.functional as F

from f16acc_amd import fp8, moe
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, normal, weight

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

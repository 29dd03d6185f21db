"""The 8-bit layer and the routing inside a training step."""

import pytest
import torch
import torch.nn.functional as F

from f16acc_amd import fp8, moe
from tests.test_gpu_fp8 import normal, weight

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

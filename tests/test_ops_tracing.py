"""What records or differentiates a call by other means than running it: the operators write
through pointers, so they refuse a trace (it would replay the allocation alone), a forward-mode
tangent (it would be dropped) and tensors that are not plain memory."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from f16acc_amd import fp8, moe

F8 = torch.float8_e4m3fn


def calls(device):
    """Every operator as a function of one floating point [128, 128] tensor."""
    one = torch.ones(1, 1, device=device)
    q = torch.ones(128, 128, device=device).to(F8)
    w1, w2 = q.expand(2, 2, 128, 128).contiguous(), q.expand(2, 128, 128).contiguous()
    s1, s2 = torch.ones(2, 2, 1, 1, device=device), torch.ones(2, 1, 1, device=device)
    long = torch.ones(128, 128 * 128, device=device).to(F8)
    wide, ones = long.t(), one.expand(128, 1)
    weights, ids = torch.ones(128, 1, device=device), torch.zeros(128, 1, dtype=torch.int32, device=device)
    return {
        "quantize": lambda x: fp8.quantize(x)[0],
        "quantize_weight": lambda x: fp8.quantize_weight(x)[1],
        "mm": lambda x: fp8.mm(long, x, wide, ones),
        "linear": lambda x: fp8.linear(x, x),
        "linear_stored": lambda x: fp8.linear(x, q, one),
        "route": lambda x: moe.route(x, 2)[0],
        "experts": lambda x: moe.experts(x, weights, ids, w1, s1, w2, s2),
    }


NAMES = sorted(calls("cpu"))


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(name):
    """No tensor is touched: the refusal comes before the check for a GPU."""
    x = torch.ones(128, 128)
    f = calls("cpu")[name]
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(f, x)
    for kw in (dict(), dict(tracing_mode="fake"), dict(pre_dispatch=True)):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(f, **kw)(x)
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError, match="traced"):
        f(torch.ones(128, 128))
    for transform in (torch.func.vmap(f), torch.func.grad(lambda x: f(x).float().sum()),
                      torch.func.functionalize(f)):
        with pytest.raises(NotImplementedError, match="traced"):
            transform(x)


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    f = calls("cpu")[name]
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(128, 128), torch.ones(128, 128))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(x)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="GPU"):
            f(x)  # (nothing is differentiated: the next check speaks)


class Wrapper(torch.Tensor):
    """A tensor that stands for another one."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

    def __init__(self, t):
        self.t = t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        plain = lambda a: a.t if isinstance(a, Wrapper) else a
        return func(*map(plain, args), **{k: plain(v) for k, v in (kwargs or {}).items()})


class Sub(torch.Tensor):
    pass


class Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_refusals_and_what_still_runs_on_the_gpu(name):
    f = calls("cuda")[name]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(128, 128, generator=g).cuda()
    want = f(x)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(f, x)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(f)(x)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        f(forward_ad.make_dual(x, x.clone()))
    z = torch.complex(x, x).conj()
    assert z.imag.is_neg()
    for bad in (z.imag, Wrapper(x), x.to_sparse()):
        with pytest.raises(ValueError, match="plain"):
            f(bad)
    # neither a subclass without behaviour of its own nor a mode that only watches is in the way
    same = lambda a, b: torch.equal(a.float(), b.float())
    assert same(f(x.as_subclass(Sub)), want) and same(f(torch.nn.Parameter(x, requires_grad=False)), want)
    with Watch():
        got = f(x)
    assert same(got, want)


@pytest.mark.gpu
def test_gradients_under_a_trace_and_batched_are_refused():
    x = torch.randn(128, 128, device="cuda", requires_grad=True)
    q, s = fp8.quantize_weight(torch.randn(128, 128, device="cuda"))
    for y in (fp8.linear(x, x), fp8.linear(x, q, s), moe.route(x, 2)[0]):
        dy = torch.ones_like(y)
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(lambda dy: torch.autograd.grad(y, x, dy, retain_graph=True)[0])(dy)
        with pytest.raises(ValueError, match="plain"):
            torch.autograd.grad(y, x, torch.stack([dy, dy]), is_grads_batched=True, retain_graph=True)
        want, = torch.autograd.grad(y, x, -2 * dy, retain_graph=True)
        negated = torch.complex(dy, 2 * dy).conj().imag
        assert negated.is_neg()
        assert torch.equal(torch.autograd.grad(y, x, negated)[0], want)

"""The whole layer without a GPU: what the C ABI and the Python function refuse."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from f16acc_amd import _ops, moe

T, E, K, D, I = 2, 8, 3, 256, 128
NEED = _ops.layer_workspace(T, K, E, D, I)


def call(x=256, t=0, T=T, r=256, rt=0, E=E, k=K, sig=0, groups=1, top=1, D=D, I=I, w1=256, w1e=2 * I * D, ld1=D, s1=256, w2=256,
         ld2=I, s2=256, s2e=2, y=256, ws=256, n=NEED):
    return _ops.layer(x, t, T, D, 1, r, rt, D, 1, E, k, sig, None, groups, top, 1, 1.0, D, I, w1, w1e, I * D, ld1, s1, 4, 2, 2,
                      1, w2, I * D, ld2, s2, s2e, 1, 1, y, ws, n, None)


def test_checks():
    for few in (2, 40):  # the kernels for a few tokens, and the others
        n = dict(T=few, n=_ops.layer_workspace(few, K, E, D, I))
        assert call(**n, x=None) == call(**n, t=3) == call(**n, r=None) == call(**n, rt=-1) == call(**n, k=0) == _ops.E_ARG
        assert call(**n, E=0) == call(**n, D=0) == call(**n, I=0) == call(**n, w1=None) == call(**n, s1=None) == _ops.E_ARG
        assert call(**n, w2=None) == call(**n, s2=None) == call(**n, y=None) == call(**n, w1e=-16) == _ops.E_ARG
        assert call(**n, groups=3) == call(**n, groups=0) == call(**n, groups=4, top=5) == call(**n, s2e=-1) == _ops.E_ARG
        assert call(**n, groups=4, top=1) == call(**n, E=2) == _ops.E_ARG  # fewer experts than k
        n["n"] -= 1
        assert call(**n) == _ops.E_WORKSPACE
    assert call(ws=None) == call(ws=64) == _ops.E_WORKSPACE and call(T=-1) == _ops.E_ARG and call(T=0) == 0
    assert call(E=1025, n=1 << 40) == call(E=200, k=65, n=1 << 40) == call(E=130, groups=65, k=2, n=1 << 40) == _ops.E_UNSUPPORTED
    assert call(T=40, ld1=128, n=1 << 40) == call(T=40, w1=264, n=1 << 40) == call(T=1 << 40, n=1 << 62) == _ops.E_UNSUPPORTED


def test_a_workspace_holds_fewer_tokens_too():
    for k, E, D, I in ((8, 64, 2048, 1024), (1, 1, 16, 16), (16, 16, 16, 4096), (3, 20, 1040, 720), (4, 1000, 128, 4096), (2, 3, 8, 20000)):
        most = 0
        for t in [*range(1, 700), *range(700, 40000, 97)]:
            need = _ops.layer_workspace(t, k, E, D, I)
            assert need >= most, (k, E, D, I, t)
            most = need


def test_cpu_tensors_traces_and_tangents_are_refused():
    x = torch.zeros(4, 16)
    f = lambda x: moe.layer(x, x, 2, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        f(x)
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(f)(x)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.func.vmap(f)(x)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        f(forward_ad.make_dual(x, x.clone()))

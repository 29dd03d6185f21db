"""mm and the patched F.linear under torch.jit.trace and make_fx: both write through pointers, so a trace would
replay the output's allocation alone."""

import pytest
import torch
import torch.nn.functional as F
from torch.fx.experimental.proxy_tensor import make_fx

import f16acc_amd as f16acc
from f16acc_amd import kernel

CALLS = {
    "mm": lambda a, b: f16acc.mm(a, b),
    "mm_bias": lambda a, b: kernel.mm_bias(a, b, b[0]),
    "mm_flags": lambda a, b: kernel.mm_flags(a, b)[0],
    "mm_tile": lambda a, b: kernel.mm_tile(a, b, "128x128"),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_traces_of_mm_are_refused(name):
    a, b = torch.zeros(8, 16).half(), torch.zeros(16, 24).half()
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(CALLS[name], (a, b))
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(CALLS[name])(a, b)
    with pytest.raises(ValueError):
        CALLS[name](a, b)


@pytest.mark.gpu
def test_a_traced_linear_layer_replays_torchs():
    g = torch.Generator().manual_seed(1)
    layer = torch.nn.Linear(256, 192).cuda().half()
    x, other = (torch.randn(200, 256, generator=g).cuda().half() for _ in range(2))
    want = layer(other)
    f16acc.enable()
    try:
        with torch.no_grad():
            for trace in (torch.jit.trace(layer, x), make_fx(layer)(x)):
                before = dict(f16acc.calls)
                assert torch.equal(trace(other), want)
                assert f16acc.calls == before  # (the trace holds torch's layer)
            layer(x)
            assert f16acc.calls["chunked"] == before["chunked"] + 1
    finally:
        f16acc.disable()


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(CALLS))
def test_traces_of_mm_are_refused_on_the_gpu(name):
    a, b = torch.ones(256, 64, device="cuda").half(), torch.ones(64, 128, device="cuda").half()
    want = CALLS[name](a, b)
    with pytest.raises(NotImplementedError, match="traced"):
        torch.jit.trace(CALLS[name], (a, b))
    with pytest.raises(NotImplementedError, match="traced"):
        make_fx(CALLS[name])(a, b)
    assert torch.equal(CALLS[name](a, b), want)

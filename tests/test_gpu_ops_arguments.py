"""Arguments of the operators at the edges of what they take, and what mm_tile refuses."""

import pytest
import torch

from f16acc_amd import fp8
from tests import ops_reference as ref
from tests.test_gpu_fp8 import DEV, normal, weight

pytestmark = pytest.mark.gpu


def test_mm_tile_refuses_what_does_not_fit():
    M, N, K = 40, 72, 256
    a, sa = fp8.quantize(normal(M, K))
    w, ws = weight(N, K)
    f = lambda out, bias=None, tile=4, splits=1: fp8.mm_tile(a, sa, w.t(), ws.t(), out, tile, splits, bias)
    out = torch.empty(M, N, device=DEV)
    short, pair = torch.zeros(N - 1, device=DEV), torch.zeros(1, N, device=DEV)
    bad = [lambda: f(torch.empty(M + 1, N, device=DEV)), lambda: f(torch.empty(M, N + 200, device=DEV)),
           lambda: f(torch.empty(M, device=DEV)), lambda: f(out.int()), lambda: f(out.double()), lambda: f(out.cpu()),
           lambda: f(out[:1].expand(M, N)), lambda: f(out, short), lambda: f(out, pair), lambda: f(out, pair[0].half()),
           lambda: f(out, pair[0].cpu()), lambda: f(out, tile=6), lambda: f(out, tile=-2), lambda: f(out, splits=-1),
           lambda: fp8.mm_tile(a, sa, w.t(), ws.t().repeat_interleave(128, 1)[:, :N], out, 1, 1)]
    for g in bad:
        with pytest.raises(ValueError):
            g()
    bias = normal(3 * N, dtype=torch.float32)[::3]
    f(out, bias)
    ref.check_product(out, ref.values(a, sa), ref.values(w, ws, 128), bias)


def test_mm_tile_without_a_product_is_the_bias():
    M, N = 5, 7
    z = lambda *s: torch.zeros(*s, device=DEV)
    out, bias = torch.full((M, N), 3.0, device=DEV), normal(N, dtype=torch.float32)
    a, b = z(M, 0).to(torch.float8_e4m3fn), z(0, N).to(torch.float8_e4m3fn)
    fp8.mm_tile(a, z(M, 0), b, z(0, 1), out, -1, 0)
    assert bool((out == 0).all())
    fp8.mm_tile(a, z(M, 0), b, z(0, 1), out, -1, 0, bias)
    assert torch.equal(out, bias.expand(M, N))

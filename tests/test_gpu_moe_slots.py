"""The experts' results on their way to the weighted sum: no column's value depends on the columns beside it,
and FP32 results keep FP32's accuracy."""

import pytest
import torch

from f16acc_amd import fp8, moe
from tests import ops_reference as ref
from tests.test_gpu_moe import check_experts, layer

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
TOKENS = [3, 20, 100, 500]  # over 2 experts, 1 a token: the kernels for few tokens, tiles of 32, 128 and 256


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", TOKENS)
def test_a_column_does_not_see_its_neighbours(T, dtype):
    """One row of w2 holds a NaN, or is 2^18 times as large as the others: every other column keeps its bits."""
    x, weights, ids, w1, s1, w2, s2 = layer(T, 2, 1, 256, 128, dtype)
    row = 37
    w2 = w2.float().div(120.0 * 512.0).clamp(-2.0 ** -6, 2.0 ** -6).to(F8)  # (e4m3's smallest values)
    w2[:, row] = torch.zeros((), device=w2.device).to(F8)
    others = [n for n in range(256) if n != row]
    want = moe.experts(x, weights, ids, w1, s1, w2, s2)
    assert bool((want[:, others] != 0).any())
    spoilt = w2.clone()
    spoilt[:, row, 5] = torch.tensor(float("nan"), device=w2.device).to(F8)
    y = moe.experts(x, weights, ids, w1, s1, spoilt, s2)
    assert bool(torch.isnan(y[:, row]).all()) and torch.equal(y[:, others], want[:, others])
    large = w2.clone()
    large[:, row] = torch.tensor(448.0, device=w2.device).to(F8)
    y = moe.experts(x, weights, ids, w1, s1, large, s2)
    assert torch.equal(y[:, others], want[:, others])


@pytest.mark.parametrize("T", TOKENS)
def test_fp32_results_are_summed_in_fp32(T):
    """Each column of the result is one hidden value times a power of two, so what rounds is FP32 alone: the gate's
    and the up's sums of 128 exact products (good to 1e-6 at worst: sums of up to 30 times the result), SiLU and the
    scales.  Of the 8-bit hidden values 1e-5 may lie on the other side of a tie: of at most 128000 values 1.3 are expected,
    and 12 are let pass."""
    x, weights, ids, w1, s1, w2, s2 = layer(T, 2, 2, 128, 128, torch.float32, seed=21)
    w2 = torch.eye(128, device=x.device).mul(2.0).to(F8).expand(2, 128, 128).contiguous()
    s2 = torch.full_like(s2, 0.25)
    y = moe.experts(x, weights, ids, w1, s1, w2, s2).cpu().double()
    want, parts = torch.zeros(y.shape, dtype=torch.float64), torch.zeros(y.shape, dtype=torch.float64)
    for j in range(2):
        one = torch.full_like(ids, -1)
        one[:, j] = ids[:, j]
        part = ref.experts(x, weights, one, w1, s1, w2, s2)
        want, parts = want + part, parts + part.abs()
    off = (y - want).abs() > 2e-5 * parts
    assert int(off.sum()) <= 12, (int(off.sum()), ((y - want).abs() / parts.clamp(min=1e-30)).median().item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 20, 16), (4, 9, 4), (2, 8, 8), (3, 1000, 5), (4, 1, 1), (5, 6, 3), (1, 30, 17), (2, 9, 9)])
def test_around_the_limits_of_the_kernels_for_few_tokens(T, E, k, dtype):
    """4 tokens and 16 slots: distinct experts, the same one in several slots of a token, and none."""
    args = list(layer(T, E, k, 144, 130, dtype, seed=T))
    check_experts(moe.experts(*args), args)
    args[2][:, ::2] = E - 1
    check_experts(moe.experts(*args), args)
    args[2][-1, :] = torch.arange(k) % 2 - 1  # -1, 0, -1, 0 ...
    check_experts(moe.experts(*args), args)


@pytest.mark.parametrize("T,D,I", [(1, 1000, 300), (4, 250, 130), (2, 129, 17)])
def test_few_tokens_read_weights_of_any_alignment_in_place(T, D, I):
    """No copy of the experts' weights: NaN bytes around the rows are not read as values, and the call needs less
    memory than one expert."""
    E = 40
    x, weights, ids, w1, s1, w2, s2 = layer(T, E, 3, D, I)
    x = torch.nn.functional.pad(x, (0, -D % 8))[:, :D]  # (rows that 16-byte loads fit)
    aligned = [torch.zeros(*w.shape[:-1], -(-w.shape[-1] // 16) * 16, dtype=torch.uint8, device=x.device).view(F8) for w in (w1, w2)]
    for a, w in zip(aligned, (w1, w2)):
        a[..., :w.shape[-1]] = w
    want = moe.experts(x, weights, ids, aligned[0][..., :D], s1, aligned[1][..., :I], s2)
    check_experts(want, (x, weights, ids, w1, s1, w2, s2))
    odd = []
    for w in (w1, w2):
        hold = torch.full((w.numel() // w.shape[-1] * (w.shape[-1] + 5) + 64,), float("nan")).to(F8).to(x.device)
        v = hold[3:3 + w.numel() // w.shape[-1] * (w.shape[-1] + 5)].view(*w.shape[:-1], w.shape[-1] + 5)[..., :w.shape[-1]]
        odd.append(v.copy_(w))
    for a, b in ((w1, w2), odd):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = moe.experts(x, weights, ids, a, s1, b, s2)
        assert torch.equal(got, want)
        assert torch.cuda.max_memory_allocated() - before < 30 * D * I

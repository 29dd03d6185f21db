"""Products of microscaled 4-bit operands: blocks of 32 values with a power of two each.

    q, s = fp4.quantize(x)                 # blocks of 1 x 32, activations and weights alike
    x = fp4.dequantize(q, s)
    c = fp4.mm(q, s, wq.t(), ws.t())       # like f16acc_amd.mm: (M, K) @ (K, N)
    y = fp4.linear(x, wq, ws, bias)        # for a stored weight, wq, ws = fp4.quantize(w)
    y = fp4.linear(x, w)                   # 16- or 32-bit weight, with gradients

Values are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to an element of
torch.float4_e2m1fn_x2, the first in its low half; scales are torch.float8_e8m0fnu.  A block's
scale is s = 2^e with 2^e <= m / 3.5 < 2^(e + 1), m = max(|x|, 2^-100), its values
e2m1(x / s), nearest, ties to even: no value is off by more than half a step.  A block that
holds an infinity or a NaN has the scale NaN, so the results that read it are NaN.  Last
blocks may be short; an odd last value has its element to itself, the high half zero.  A product is exact within
a block and added in FP32 over the blocks, rounded once to the result's type.

Everything runs on the current torch stream of the operands' GPU, allocates
through torch, and does not synchronise.  Wrong arguments raise ValueError; a call
that torch traces (torch.jit.trace, make_fx, export, torch.func) or differentiates
forward raises NotImplementedError.
"""

import torch

from ._ops import host

__all__ = ["quantize", "dequantize", "mm", "linear"]


def quantize(x, transposed=False):
    """Blocks of 32 along the last dimension.

    x: [..., K] float16, bfloat16 or float32, any strides.  Returns (q, scale):
    float4_e2m1fn_x2 [..., ceil(K / 2)] (its rows lie 64-byte aligned, zero to the next multiple of
    128 values) and float8_e8m0fnu [..., ceil(K / 32)], without gradients.  transposed: for a 2-d x, the
    same of x.t(), in blocks of 32 rows of x: q [K, ceil(M / 2)], scale [K, ceil(M / 32)]."""
    return host.fp4_quantize(x, transposed)


def dequantize(q, scale, dtype=torch.float32):
    """The values of q [..., P] with its scales [..., ceil(P / 16)], any strides: [..., 2 P] float16, bfloat16 or
    float32, each rounded once, without gradients.  (Of an odd number of values the last is the padding's zero.)"""
    return host.fp4_dequantize(q, scale, dtype)


def mm(a, a_scale, b, b_scale, out_dtype=torch.float16):
    """c = (a * a_scale) @ (b * b_scale), block by block, with P = K / 2 elements of two values along K.

    a: float4_e2m1fn_x2 [M, P], a_scale: float8_e8m0fnu [M, ceil(P / 16)]
    b: float4_e2m1fn_x2 [P, N], b_scale: float8_e8m0fnu [ceil(P / 16), N]
    Any strides; operands whose elements are contiguous along K, in whole blocks of 16, with 16-byte aligned rows at most 4 MiB
    apart (b = w.t() of a stored [N, P] weight) are read as they are, others copied on every call.  No gradients."""
    return host.fp4_mm(a, a_scale, b, b_scale, out_dtype, None, None, -1, 0)


def mm_tile(a, a_scale, b, b_scale, out, tile, splits, bias=None):
    """mm into `out` ([M, N], any strides) with the tile (0 to 5) and the number of parts of K forced, and a bias
    [N] in out's type: for tuning and tests."""
    return host.fp4_mm(a, a_scale, b, b_scale, out.dtype, bias, out, tile, splits)


def linear(x, w, w_scale=None, bias=None):
    """y = x @ w.T + bias in 4 bits, in x's type.

    x: [..., K] float16, bfloat16 or float32, quantised in blocks of 1 x 32
    w, w_scale: a stored float4_e2m1fn_x2 [N, ceil(K / 2)] weight with its float8_e8m0fnu
       [N, ceil(K / 32)] scales; gradients reach x and bias.  That of x is the product of dy and of w's
       values, quantised again along N (blocks of 32 rows of w) on every call.  Rows that no 16-byte load
       fits (K no multiple of 32 among them) are copied on every call, except for few
       tokens (at most 16, fewer with large weights, their values next to each other): one kernel reads the rows as they
       are, without a workspace, and a token's result there does not depend on those beside it
    w alone: a float16, bfloat16 or float32 [N, K] weight, quantised on every call; gradients reach x, w
       and bias, their products in 4 bits too, every operand quantised along its product's sum:
       dx = Q(dy) Q(w) in blocks along N, dw = Q(dy).T Q(x) in blocks along the tokens
    bias: [N] in x's type, or None."""
    return host.fp4_linear(x, w, w_scale, bias)

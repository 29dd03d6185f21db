"""Mixture of experts: routing, the experts' gated feed-forward in 8 bits, and both with the
router's product as one call.

    weights, ids = moe.route(logits, k=8)          # logits [T, E]
    y = moe.experts(x, weights, ids, w1, w1_scale, w2, w2_scale)
    y = moe.layer(x, router, 8, w1, w1_scale, w2, w2_scale)

Everything runs on the current torch stream of the operands' GPU, allocates
through torch, and does not synchronise: the tokens are sorted by expert on the
device.  Wrong arguments raise ValueError; a call that torch traces (torch.jit.trace,
make_fx, export, torch.func) or differentiates forward raises NotImplementedError.
"""

from ._ops import host

__all__ = ["route", "experts", "layer"]


def route(logits, k, *, scoring="softmax", bias=None, groups=1, top_groups=1, renormalize=True, scale=1.0):
    """The k experts of each token and their weights.

    logits: [..., E] float16, bfloat16 or float32, any strides; E at most 1024
    scoring: "softmax" or "sigmoid" of the logits, in FP32
    bias: float32 [E] added to the scores for the choice alone (balance), or None
    groups, top_groups: only the experts of the best top_groups of `groups` equal
       groups of consecutive experts take part.  A group counts as its best
       expert (softmax) or as the sum of its best two (sigmoid)
    renormalize: divide the chosen scores by their sum (plus 1e-20)
    scale: factor of the weights

    Returns (weights float32 [..., k], ids int32 [..., k]), best first, ties to
    the lowest index.  An expert whose logit (or biased score) is -inf or NaN is not
    available; where fewer than k are, ids are -1 and weights 0.  A token with a
    NaN logit has NaN weights.  Gradients reach the logits through the weights."""
    return host.route(logits, k, scoring, bias, groups, top_groups, renormalize, scale)


def experts(x, weights, ids, w1, w1_scale, w2, w2_scale):
    """The routed experts' gated feed-forward, in 8 bits:

        y[t] = sum_j weights[t, j] * (silu(x[t] w1[e, 0].T) * (x[t] w1[e, 1].T)) w2[e].T,  e = ids[t, j]

    x: [..., D] float16, bfloat16 or float32, quantised in blocks of 1 x 128, as are
       the FP32 hidden values
    weights: float32 [..., k];  ids: int32 or int64 [..., k]; an id outside
       0 .. E - 1 (-1) adds nothing, and its weight is not read
    w1: float8_e4m3fn [E, 2, I, D] (gate, up), w1_scale: float32 [E, 2, ceil(I / 128), ceil(D / 128)]
    w2: float8_e4m3fn [E, D, I], w2_scale: float32 [E, ceil(D / 128), ceil(I / 128)]
    Returns [..., D] in x's type, the sum over the experts in FP32.  Weights whose rows no
    16-byte load fits (D or I not a multiple of 16, views at odd addresses or over 4 MiB
    apart) are copied on every call, those of all experts, except for 1 to 4 tokens with at most
    16 ids in all, rows of x that 16-byte loads fit and K-contiguous weights, which read the
    routed experts' rows as they are.
    The products of gate and up are exact in FP32, except for bfloat16 x with 192 or more tokens
    an expert on average; those and the products of w2 have the block sums of fp8.mm.  For
    inference: operands that require gradients are refused where gradients are
    enabled."""
    return host.experts(x, weights, ids, w1, w1_scale, w2, w2_scale)


def layer(x, router, k, w1, w1_scale, w2, w2_scale, *, scoring="softmax", bias=None, groups=1, top_groups=1,
          renormalize=True, scale=1.0):
    """The whole layer: route of the logits x @ router.T, and experts of what it chooses.

    x: [..., D] float16, bfloat16 or float32, any strides
    router: [E, D] float16, bfloat16 or float32, any strides.  The logits are summed in
       64 bits and rounded once to FP32.  The order of a sum goes by the number of tokens: where
       a sum is exact in 64 bits a token's logits, and its choice, are the same in every batch; else they may
       differ where the 64-bit sum lies within its own rounding (2^-53 of its terms' magnitudes for each
       addition) of the middle between two FP32 values.  A token with a NaN logit gives NaN
    k and the options are route's, the weights and their scales experts'
    Returns [..., D] in x's type.  For inference: operands that require gradients are refused
    where gradients are enabled."""
    return host.layer(x, router, k, w1, w1_scale, w2, w2_scale, scoring, bias, groups, top_groups, renormalize, scale)

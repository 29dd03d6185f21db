"""Mixture of experts: routing, and the experts' gated feed-forward in 8 bits.

    weights, ids = moe.route(logits, k=8)          # logits [T, E]
    y = moe.experts(x, weights, ids, w1, w1_scale, w2, w2_scale)

Everything runs on the current torch stream of the operands' GPU, allocates
through torch, and does not synchronise: the tokens are sorted by expert on the
device.
"""

import torch

from . import _ops
from ._ops import FP8, TYPES, blocks, call, on_gpu, ptr
from .fp8 import _check_float, _packed, _rows

__all__ = ["route", "experts"]

_SCORING = {"softmax": 0, "sigmoid": 1}


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, args):
        weights, ids = _route(logits, *args)
        ctx.mark_non_differentiable(ids)
        ctx.save_for_backward(logits, ids)
        ctx.args = args
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dw, _):
        logits, ids = ctx.saved_tensors
        k, sigmoid, _, _, _, renormalize, scale = ctx.args
        x = _rows(logits)
        dw = _rows(dw)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        call(_ops.route_grad, x.device, ptr(x), TYPES[x.dtype], x.shape[0], x.stride(0), x.stride(1), x.shape[1], k,
             sigmoid, renormalize, scale, ptr(ids), ptr(dw), dw.stride(0), dw.stride(1), ptr(dx))
        return dx.view(logits.shape), None


def _route(logits, k, sigmoid, bias, groups, top_groups, renormalize, scale):
    x = _rows(logits)
    T, E = x.shape
    weights = torch.empty(T, k, dtype=torch.float32, device=x.device)
    ids = torch.empty(T, k, dtype=torch.int32, device=x.device)
    call(_ops.route, x.device, ptr(x), TYPES[x.dtype], T, x.stride(0), x.stride(1), E, k, sigmoid, ptr(bias), groups,
         top_groups, renormalize, scale, ptr(weights), ptr(ids))
    lead = logits.shape[:-1]
    return weights.view(*lead, k), ids.view(*lead, k)


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
    on_gpu("route", logits, bias)
    _check_float("route", logits)
    if logits.dim() < 1:
        raise ValueError("route needs [..., E] logits")
    E = logits.shape[-1]
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {tuple(_SCORING)}, not {scoring!r}")
    if not 1 <= E <= 1024:
        raise ValueError(f"route needs 1 to 1024 experts, got {E}")
    if groups < 1 or E % groups or groups > 64 or not 1 <= top_groups <= groups:
        raise ValueError(f"{E} experts in {groups} groups of which {top_groups} stay: not equal groups, or over 64")
    if not 1 <= k <= min(64, E // groups * top_groups):
        raise ValueError(f"k must be 1 to 64 and at most the experts of the groups that stay, got {k}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (E,)):
        raise ValueError(f"bias must be float32 [{E}], got {bias.dtype} {tuple(bias.shape)}")
    bias = None if bias is None else bias.detach().contiguous()
    args = (k, _SCORING[scoring], bias, groups, top_groups, int(bool(renormalize)), float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Route.apply(logits, args)
    return _route(logits, *args)


def experts(x, weights, ids, w1, w1_scale, w2, w2_scale):
    """The routed experts' gated feed-forward, in 8 bits:

        y[t] = sum_j weights[t, j] * (silu(x[t] w1[e, 0].T) * (x[t] w1[e, 1].T)) w2[e].T,  e = ids[t, j]

    x: [..., D] float16, bfloat16 or float32, quantised in blocks of 1 x 128, as are
       the FP32 hidden values
    weights: float32 [..., k];  ids: int32 or int64 [..., k]; an id outside
       0 .. E - 1 (-1) adds nothing, and its weight is not read
    w1: float8_e4m3fn [E, 2, I, D] (gate, up), w1_scale: float32 [E, 2, ceil(I / 128), ceil(D / 128)]
    w2: float8_e4m3fn [E, D, I], w2_scale: float32 [E, ceil(D / 128), ceil(I / 128)]
    Returns [..., D] in x's type, the sum over the experts in FP32.  For
    inference: operands that require gradients are refused where gradients are
    enabled."""
    dev = on_gpu("experts", x, weights, ids, w1, w1_scale, w2, w2_scale)
    _check_float("experts", x)
    if x.dim() < 1 or w1.dim() != 4 or w1.shape[1] != 2 or w2.dim() != 3:
        raise ValueError(f"experts needs x [..., D], w1 [E, 2, I, D] and w2 [E, D, I], got {tuple(x.shape)}, "
                         f"{tuple(w1.shape)}, {tuple(w2.shape)}")
    E, _, I, D = w1.shape
    if x.shape[-1] != D or w2.shape != (E, D, I) or not 1 <= E <= 1024 or D == 0 or I == 0:
        raise ValueError(f"experts needs x [..., D], w1 [E, 2, I, D] and w2 [E, D, I], got {tuple(x.shape)}, "
                         f"{tuple(w1.shape)}, {tuple(w2.shape)} (E 1 to 1024, D and I positive)")
    if w1.dtype != FP8 or w2.dtype != FP8:
        raise ValueError("experts needs float8_e4m3fn weights")
    for name, s, shape in (("w1_scale", w1_scale, (E, 2, blocks(I), blocks(D))),
                           ("w2_scale", w2_scale, (E, blocks(D), blocks(I)))):
        if s.dtype != torch.float32 or s.shape != shape:
            raise ValueError(f"{name} must be float32 {shape}, got {s.dtype} {tuple(s.shape)}")
    if ids.shape != weights.shape or ids.dim() < 1 or ids.shape[:-1] != x.shape[:-1] or ids.shape[-1] < 1:
        raise ValueError(f"weights and ids must be [..., k] over x's tokens, got {tuple(weights.shape)} and "
                         f"{tuple(ids.shape)} for {tuple(x.shape)}")
    if weights.dtype != torch.float32 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"experts needs float32 weights and int32 or int64 ids, got {weights.dtype} and {ids.dtype}")
    if torch.is_grad_enabled() and (x.requires_grad or weights.requires_grad):
        raise ValueError("experts has no backward pass: call it under torch.no_grad() or torch.inference_mode()")
    k = ids.shape[-1]
    x2, wt = _rows(x), _rows(weights)
    T = x2.shape[0]
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    if T == 0:
        return y
    ids2 = _rows(ids)
    if ids2.dtype == torch.int64:
        ids2 = ids2.clamp(-1, E)  # (before the 32-bit cast, which would wrap)
    ids2 = ids2.to(torch.int32).contiguous()
    w1p, ld1 = _packed(w1)
    w2p, ld2 = _packed(w2)
    ws = torch.empty(_ops.experts_workspace(T, k, E, D, I), dtype=torch.uint8, device=dev)
    call(_ops.experts, dev, ptr(x2), TYPES[x.dtype], T, x2.stride(0), x2.stride(1), ptr(wt), wt.stride(0),
         wt.stride(1), ptr(ids2), k, E, D, I, ptr(w1p), w1p.stride(0), w1p.stride(1), ld1, ptr(w1_scale),
         *w1_scale.stride(), ptr(w2p), w2p.stride(0), ld2, ptr(w2_scale), *w2_scale.stride(), ptr(y), ptr(ws),
         ws.numel())
    return y

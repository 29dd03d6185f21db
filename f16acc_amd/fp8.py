"""Products of 8-bit floating point operands with a scale for each block of 128.

    q, s = fp8.quantize(x)                 # activations: blocks of 1 x 128
    wq, ws = fp8.quantize_weight(w)        # weights: blocks of 128 x 128
    c = fp8.mm(q, s, wq.t(), ws.t())       # like f16acc_amd.mm: (M, K) @ (K, N)
    y = fp8.linear(x, wq, ws, bias)        # both at once, for a stored weight
    y = fp8.linear(x, w)                   # 16- or 32-bit weight, with gradients

Values are torch.float8_e4m3fn.  A block's scale is s = m / 448 with
m = max(|x|, 2^-100), its values e4m3(x * (448 / m)), every step rounded to FP32
once; a block that holds an infinity or a NaN has the scale NaN, so the results that
read it are NaN.  Last blocks may be short.  A product adds each block's FP32
sum, times its two scales, in FP32 in the order of K, and rounds once to the
result's type.

Everything runs on the current torch stream of the operands' GPU, allocates
through torch, and does not synchronise.
"""

import torch

from . import _ops
from ._ops import BLOCK, FP8, TYPES, blocks, call, on_gpu, ptr, up

__all__ = ["quantize", "quantize_weight", "mm", "linear"]


def _check_float(name, x):
    dev = on_gpu(name, x)
    if x.dtype not in TYPES:
        raise ValueError(f"{name} needs torch.float16, bfloat16 or float32, not {x.dtype}")
    return dev


def _rows(x):
    """x as a [rows, K] view (or copy, where its leading dimensions do not merge)."""
    return x if x.dim() == 2 else x.reshape(x.shape[:-1].numel(), x.shape[-1])


def _quant_rows(x):
    """(q [rows, up(K, 128)] zero padded, scales [blocks, rows]) of a 2-d x."""
    M, K = x.shape
    q = torch.empty(M, up(K, BLOCK), dtype=FP8, device=x.device)
    s = torch.empty(blocks(K), M, dtype=torch.float32, device=x.device)
    call(_ops.quant_rows, x.device, ptr(x), TYPES[x.dtype], M, K, x.stride(0), x.stride(1), ptr(q), q.shape[1],
         ptr(s), M)
    return q, s


def _quant_both(x, rows=True, cols=True):
    """_quant_rows(x) and _quant_rows(x.t()), from one pass over x."""
    M, K = x.shape
    q = s = qt = st = None
    if rows:
        q = torch.empty(M, up(K, BLOCK), dtype=FP8, device=x.device)
        s = torch.empty(blocks(K), M, dtype=torch.float32, device=x.device)
    if cols:
        qt = torch.empty(K, up(M, BLOCK), dtype=FP8, device=x.device)
        st = torch.empty(blocks(M), K, dtype=torch.float32, device=x.device)
    call(_ops.quant_both, x.device, ptr(x), TYPES[x.dtype], M, K, x.stride(0), x.stride(1), ptr(q), up(K, BLOCK),
         ptr(s), M, ptr(qt), up(M, BLOCK), ptr(st), K)
    return q, s, qt, st


def _quant_weight(w, transposed=False):
    """(q [N, up(K, 128)], scales [blocks(N), blocks(K)], q transposed [K, up(N, 128)] or None) of a 2-d w."""
    N, K = w.shape
    q = torch.empty(N, up(K, BLOCK), dtype=FP8, device=w.device)
    s = torch.empty(blocks(N), blocks(K), dtype=torch.float32, device=w.device)
    qt = torch.empty(K, up(N, BLOCK), dtype=FP8, device=w.device) if transposed else None
    call(_ops.quant_weight, w.device, ptr(w), TYPES[w.dtype], N, K, w.stride(0), w.stride(1), ptr(q), q.shape[1],
         ptr(s), blocks(K), ptr(qt), up(N, BLOCK))
    return q, s, qt


def quantize(x, transposed=False):
    """Activations in blocks of 128 along the last dimension.

    x: [..., K] float16, bfloat16 or float32, any strides.  Returns (q, scale):
    float8_e4m3fn [..., K] (its rows lie 128-byte aligned, zero to the next
    multiple of 128) and float32 [..., ceil(K / 128)].  transposed: for a 2-d x, the
    same of x.t(), in blocks of 128 rows of x: q [K, M], scale [K, ceil(M / 128)]."""
    _check_float("quantize", x)
    if x.dim() < 1 or (transposed and x.dim() != 2):
        raise ValueError(f"quantize needs {'a 2-d tensor to transpose' if transposed else 'one dimension or more'}, "
                         f"got {tuple(x.shape)}")
    if transposed:
        _, _, q, s = _quant_both(x, rows=False)
        return q[:, :x.shape[0]], s.t()
    lead = x.shape[:-1]
    q, s = _quant_rows(_rows(x))
    return q[:, :x.shape[-1]].view(*lead, x.shape[-1]), s.t().view(*lead, s.shape[0])


def quantize_weight(w):
    """Weights [..., N, K] in blocks of 128 x 128: (float8_e4m3fn [..., N, K],
    float32 [..., ceil(N / 128), ceil(K / 128)])."""
    _check_float("quantize_weight", w)
    if w.dim() < 2:
        raise ValueError(f"quantize_weight needs [..., N, K], got {tuple(w.shape)}")
    N, K = w.shape[-2:]
    lead = w.shape[:-2]
    q = torch.empty(*lead, N, up(K, BLOCK), dtype=FP8, device=w.device)
    s = torch.empty(*lead, blocks(N), blocks(K), dtype=torch.float32, device=w.device)
    w3, q3, s3 = (t.reshape(-1, *t.shape[-2:]) for t in (w, q, s))
    for wi, qi, si in zip(w3, q3, s3):
        call(_ops.quant_weight, w.device, ptr(wi), TYPES[w.dtype], N, K, wi.stride(0), wi.stride(1), ptr(qi),
             q.shape[-1], ptr(si), blocks(K), None, 0)
    return q[..., :K], s


def _packed(q):
    """q [..., rows, K] with rows the products read: 16-byte aligned, unit
    stride, and K a multiple of 16 or rows copied with zeros to the next one."""
    rows, K = q.shape[-2:]
    s = q.stride()
    ld = s[-2] if rows > 1 else up(K, 16)
    if (K % 16 == 0 and (s[-1] == 1 or K <= 1) and ld >= K and all(v % 16 == 0 for v in s[:-2]) and ld % 16 == 0
            and q.data_ptr() % 16 == 0):
        return q, ld
    out = torch.empty(*q.shape[:-1], up(K, 16), dtype=FP8, device=q.device)
    src = q if q.dim() == 2 else q.reshape(-1, K)  # (leading dimensions that do not merge are copied)
    call(_ops.pack8, q.device, ptr(src), ptr(out), src.shape[0], K, src.stride(0), src.stride(1), out.shape[-1])
    return out, out.shape[-1]


def _product(x, ldx, sx, w, ldw, sw, M, N, K, out, row_scales, bias=None, tile=-1, splits=0):
    """out [M, N] from x [M, K] and w [N, K]; sx and sw are ([m], [kb]) and
    ([n or n / 128], [kb]) indexed.  tile, splits: force the library's choices (tuning, tests)."""
    n = _ops.mm_fp8_workspace(M, N, K, int(row_scales), tile, splits)
    ws = torch.empty(n, dtype=torch.uint8, device=out.device) if n else None
    call(_ops.mm_fp8, out.device, ptr(x), ldx, ptr(sx), sx.stride(0), sx.stride(1), ptr(w), ldw, ptr(sw),
         sw.stride(0), sw.stride(1), int(row_scales), ptr(bias), ptr(out), out.stride(0), out.stride(1), M, N, K,
         TYPES[out.dtype], tile, splits, ptr(ws), n)
    return out


def mm(a, a_scale, b, b_scale, out_dtype=torch.float16):
    """c = (a * a_scale) @ (b * b_scale), block by block.

    a: float8_e4m3fn [M, K], a_scale: float32 [M, ceil(K / 128)]
    b: float8_e4m3fn [K, N], b_scale: float32 [ceil(K / 128), ceil(N / 128)] for
       square blocks, or [ceil(K / 128), N] for a scale for each column of b
    Any strides; K-contiguous operands with 16-byte aligned rows (b = w.t() of a
    stored [N, K] weight) are read as they are, others copied once."""
    dev = on_gpu("fp8.mm", a, a_scale, b, b_scale)
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"fp8.mm needs (M, K) @ (K, N), got {tuple(a.shape)} @ {tuple(b.shape)}")
    M, K = a.shape
    N = b.shape[1]
    if a.dtype != FP8 or b.dtype != FP8 or a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise ValueError("fp8.mm needs float8_e4m3fn operands and float32 scales")
    if a_scale.shape != (M, blocks(K)):
        raise ValueError(f"a_scale must be {(M, blocks(K))}, got {tuple(a_scale.shape)}")
    row_scales = b_scale.shape == (blocks(K), N) and N > 1
    if not row_scales and b_scale.shape != (blocks(K), blocks(N)):
        raise ValueError(f"b_scale must be {(blocks(K), blocks(N))} or {(blocks(K), N)}, got {tuple(b_scale.shape)}")
    if out_dtype not in TYPES:
        raise ValueError(f"fp8.mm writes torch.float16, bfloat16 or float32, not {out_dtype}")
    out = torch.empty(M, N, dtype=out_dtype, device=dev)
    if M == 0 or N == 0:
        return out
    if K == 0:
        return out.zero_()
    x, ldx = _packed(a)
    w, ldw = _packed(b.t())
    return _product(x, ldx, a_scale, w, ldw, b_scale.t(), M, N, K, out, row_scales)


class _Train(torch.autograd.Function):
    """y = x w^T; dx = dy w, dw = dy^T x, each from operands quantised along its
    own contraction: x and dy in rows of 128 channels and in columns of 128
    tokens, w in squares, which serve both of its products."""

    @staticmethod
    def forward(ctx, x, w):
        x2 = _rows(x)
        M, K = x2.shape
        N = w.shape[0]
        need_x, need_w = ctx.needs_input_grad
        q, s, qt, st = _quant_both(x2, cols=need_w)
        wq, ws, wqt = _quant_weight(w, transposed=need_x)
        y = _product(q, q.shape[1], s.t(), wq, wq.shape[1], ws, M, N, K, x2.new_empty(M, N), False)
        ctx.save_for_backward(qt, st, wqt, ws)
        ctx.sizes = x.shape, M, N, K, w.dtype
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        qt, st, wqt, ws = ctx.saved_tensors
        shape, M, N, K, w_dtype = ctx.sizes
        need_x, need_w = ctx.needs_input_grad
        dy = _rows(dy)
        q, s, dqt, dst = _quant_both(dy, rows=need_x, cols=need_w)
        dx = dw = None
        if need_x:
            dx = _product(q, q.shape[1], s.t(), wqt, wqt.shape[1], ws.t(), M, K, N, dy.new_empty(M, K), False)
            dx = dx.view(shape)
        if need_w:
            dw = torch.empty(N, K, dtype=w_dtype, device=dy.device)
            _product(dqt, dqt.shape[1], dst.t(), qt, qt.shape[1], st.t(), N, K, M, dw, True)
        return dx, dw


class _Stored(torch.autograd.Function):
    """linear on a stored 8-bit weight, with the gradient of x."""

    @staticmethod
    def forward(ctx, x, w, w_scale, bias):
        ctx.save_for_backward(w, w_scale)
        ctx.x_shape = x.shape
        return _stored(x, w, w_scale, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        w, w_scale = ctx.saved_tensors
        N, K = w.shape
        dx = db = None
        if ctx.needs_input_grad[0]:
            dy2 = _rows(dy)
            q, s = _quant_rows(dy2)
            wt, ld = _packed(w.t())
            dx = _product(q, q.shape[1], s.t(), wt, ld, w_scale.t(), dy2.shape[0], K, N,
                          dy2.new_empty(dy2.shape[0], K), False).view(ctx.x_shape)
        if ctx.needs_input_grad[3]:
            db = _rows(dy).sum(0)
        return dx, None, None, db


def _stored(x, w, w_scale, bias):
    x2 = _rows(x)
    M, K = x2.shape
    N = w.shape[0]
    y = x.new_empty(*x.shape[:-1], N)
    w, ldw = _packed(w)
    ws = torch.empty(_ops.linear_fp8_workspace(M, N, K), dtype=torch.uint8, device=x.device)
    call(_ops.linear_fp8, x.device, ptr(x2), TYPES[x.dtype], x2.stride(0), x2.stride(1), ptr(w), ldw, ptr(w_scale),
         w_scale.stride(0), w_scale.stride(1), ptr(bias), ptr(y), M, N, K, ptr(ws), ws.numel())
    return y


def linear(x, w, w_scale=None, bias=None):
    """y = x @ w.T + bias in 8 bits, in x's type.

    x: [..., K] float16, bfloat16 or float32, quantised in blocks of 1 x 128
    w, w_scale: a stored float8_e4m3fn [N, K] weight with its float32
       [ceil(N / 128), ceil(K / 128)] scales; gradients reach x and bias
    w alone: a float16, bfloat16 or float32 [N, K] weight, quantised in squares
       on every call; gradients reach x, w and bias, their products in 8 bits too
    bias: [N] in x's type, or None."""
    dev = _check_float("fp8.linear", x)
    on_gpu("fp8.linear", x, w, w_scale, bias)
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"fp8.linear needs [..., K] and [N, K], got {tuple(x.shape)} and {tuple(w.shape)}")
    N, K = w.shape
    if bias is not None and (bias.shape != (N,) or bias.dtype != x.dtype):
        raise ValueError(f"bias must be {x.dtype} [{N}], got {bias.dtype} {tuple(bias.shape)}")
    if w_scale is None:
        if w.dtype not in TYPES:
            raise ValueError(f"fp8.linear needs w_scale for a {w.dtype} weight")
    elif w.dtype != FP8 or w_scale.dtype != torch.float32 or w_scale.shape != (blocks(N), blocks(K)):
        raise ValueError(f"fp8.linear needs a float8_e4m3fn weight with float32 {(blocks(N), blocks(K))} scales, got "
                         f"{w.dtype} with {w_scale.dtype} {tuple(w_scale.shape)}")
    if x.numel() == 0 or N == 0:  # nothing to multiply: torch gives the empty (or zero) result and its gradients
        y = x @ (w if w_scale is None else w.to(x.dtype)).to(x.dtype).t()
        return y if bias is None else y + bias
    if w_scale is None:
        if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
            y = _Train.apply(x, w)
        else:
            x2 = _rows(x)
            q, s = _quant_rows(x2)
            wq, ws, _ = _quant_weight(w)
            y = _product(q, q.shape[1], s.t(), wq, wq.shape[1], ws, x2.shape[0], N, K,
                         x2.new_empty(x2.shape[0], N), False).view(*x.shape[:-1], N)
        return y if bias is None else y + bias
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        return _Stored.apply(x, w, w_scale, bias)
    return _stored(x, w, w_scale, bias)

/*
 * f16acc for MI355X (gfx950): C ABI of the 8-bit block-scaled products and of
 * the mixture-of-experts operators (libf16acc_ops.so).
 *
 * Plain C types only.  Nothing allocates, synchronises or keeps state between
 * calls: outputs and workspaces are the caller's, work is launched on `stream`
 * (hipStream_t, NULL = the null stream) of the current device.  Return codes:
 * 0, a positive hipError_t, or a negative F16ACC_OPS_E_* for arguments
 * rejected before anything is launched.
 *
 * 8-bit values are e4m3 (OCP: 448 largest, no infinity).  A block of 128
 * values x is held as q and an FP32 scale s:
 *     m = max(|x|, 2^-100)   s = m / 448   q = e4m3(x * (448 / m))
 * every step rounded to FP32 once; a block holding an infinity or a NaN has
 * the scale NaN.  Row blocks are 1 x 128 (activations, one scale per row and block),
 * squares 128 x 128 (weights).  Last blocks may be short.
 */
#ifndef F16ACC_OPS_H
#define F16ACC_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define F16ACC_TYPE_F16 0
#define F16ACC_TYPE_BF16 1
#define F16ACC_TYPE_F32 2

#define F16ACC_OPS_E_ARG (-1)         /* negative size, null pointer with work to do, bad enum */
#define F16ACC_OPS_E_UNSUPPORTED (-2) /* an extent, stride or alignment this build cannot address */
#define F16ACC_OPS_E_WORKSPACE (-3)   /* workspace missing, misaligned or too small */

/*
 * Row blocks of x [rows, cols] (element strides sr, sc; any): q [rows][ldq]
 * bytes, ldq a multiple of 128 and at least cols, zero from cols on, 16-byte
 * aligned; the scale of (row, block) at s[block * lds + row], for the ceil(cols / 128) blocks that hold
 * a column; lds at least rows.
 */
int f16acc_quant_rows(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                      int64_t ldq, float* s, int64_t lds, void* stream);

/*
 * x read once and quantised in both directions: row blocks as above, ldq the next multiple of
 * 128 from cols (q NULL: not wanted), and blocks of 128 rows of each column, transposed: qt
 * [cols][ldqt], ldqt the next multiple of 128 from rows, zero from rows on, the
 * scale of (column, row block) at st[block * ldst + column] (qt NULL: not wanted).
 */
int f16acc_quant_both(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                      int64_t ldq, float* s, int64_t lds, uint8_t* qt, int64_t ldqt, float* st, int64_t ldst,
                      void* stream);

/*
 * Square blocks: q [rows][ldq], the scale of a block at s[rowblock * lds +
 * block]; with qt the same values transposed, [cols][ldqt], whose scales are s read
 * the other way round.  ldq and ldqt as in f16acc_quant_both.
 */
int f16acc_quant_weight(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                        int64_t ldq, float* s, int64_t lds, uint8_t* qt, int64_t ldqt, void* stream);

/* dst[r][c] = src[r * s_r + c * s_c] (bytes) for c < cols, zero up to ld, a multiple of 16. */
int f16acc_pack8(const uint8_t* src, uint8_t* dst, int64_t rows, int64_t cols, int64_t s_r, int64_t s_c, int64_t ld,
                 void* stream);

/*
 * out[c] = sum over r of x[r][c] in FP32, rounded once: a bias's gradient.  x [rows, cols] of `type` (element
 * strides sr, sc; any), out [cols] of the same type.  Workspace of
 * f16acc_column_sums_workspace bytes (0 where one pass does), 256-byte aligned.
 */
size_t f16acc_column_sums_workspace(int64_t rows, int64_t cols);
int f16acc_column_sums(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, void* out,
                       void* workspace, size_t ws_bytes, void* stream);

/*
 * c[m][n] = sum over k of (x[m][k] sx[m][k / 128]) (w[n][k] sw[n'][k / 128]) + bias[n],
 * n' = n / 128 (row_scales 0) or n (row_scales 1).  Each block's sum is the 8-bit
 * matrix instructions' (eight products at a time, each cut to a multiple of 2^-13 of two to their
 * largest sum of exponents; the groups in FP32), the blocks are added in FP32 in K order,
 * one rounding to ctype.
 *   K at least 1 where M and N are
 *   x [M][ldx], w [N][ldw]: bytes, rows 16-byte aligned and zero from K to the
 *   next multiple of 16
 *   sx, sw: element strides (sxm, sxk), (swn, swk), non-negative
 *   bias: [N] of ctype, or NULL;  c: element strides scm, scn
 *   tile, splits: -1 and 0 leave the choice to the library; a tile number (0 to 5) and a number of parts
 *   of K force them, for tuning
 *   workspace: f16acc_mm_fp8_workspace bytes for exactly these sizes (FP32 sums of the parts of
 *   K, 0 if not split; fewer rows may need more), 256-byte aligned
 */
int f16acc_mm_fp8(const uint8_t* x, int64_t ldx, const float* sx, int64_t sxm, int64_t sxk, const uint8_t* w,
                  int64_t ldw, const float* sw, int64_t swn, int64_t swk, int row_scales, const void* bias, void* c,
                  int64_t scm, int64_t scn, int64_t M, int64_t N, int64_t K, int ctype, int tile, int splits,
                  void* workspace, size_t ws_bytes, void* stream);
size_t f16acc_mm_fp8_workspace(int64_t M, int64_t N, int64_t K, int row_scales, int tile, int splits);

/*
 * y = x w^T + bias with x [M, K] of `type` (element strides sr, sc) quantised in row blocks on
 * the way; w [N][ldw] bytes of any alignment, ldw at least K, with square-block scales sw as in
 * f16acc_mm_fp8; y [M][N] contiguous and bias of x's type; K at least 1.
 * Workspace of f16acc_linear_fp8_workspace bytes for exactly these sizes, 256-byte aligned.
 */
size_t f16acc_linear_fp8_workspace(int64_t M, int64_t N, int64_t K, const uint8_t* w, int64_t ldw);
int f16acc_linear_fp8(const void* x, int type, int64_t sr, int64_t sc, const uint8_t* w, int64_t ldw, const float* sw,
                      int64_t swn, int64_t swk, const void* bias, void* y, int64_t M, int64_t N, int64_t K,
                      void* workspace, size_t ws_bytes, void* stream);

/*
 * Routing of T tokens over E experts (at most 1024) to k of them (at most 64):
 * p = softmax or sigmoid of the logits [T][E] (element strides st, se), FP32.
 * Experts are ranked by key = logit (softmax without a bias) or p + bias; an
 * expert whose logit or key is -inf or NaN is not available.  With groups > 1 only the
 * `top` best of the groups of E / groups consecutive experts take part: a
 * group counts as its best key (softmax) or its best two's sum (sigmoid).
 * The k largest keys are taken in order, ties to the lowest index:
 *   ids [T][k], -1 where none is left; weights [T][k] = scale * p (0 for -1),
 *   divided by (their sum + 1e-20) before the scale if renorm.
 * A token with a NaN logit gets NaN weights.
 */
int f16acc_route(const void* logits, int type, int64_t T, int64_t st, int64_t se, int E, int k, int sigmoid,
                 const float* bias, int groups, int top, int renorm, float scale, float* weights, int* ids,
                 void* stream);

/* Gradient of f16acc_route's weights: dw [T][k] (element strides dwt, dwk) to dlogits [T][E], contiguous, 16-byte
 * aligned, of the logits' type. */
int f16acc_route_grad(const void* logits, int type, int64_t T, int64_t st, int64_t se, int E, int k, int sigmoid,
                      int renorm, float scale, const int* ids, const float* dw, int64_t dwt, int64_t dwk,
                      void* dlogits, void* stream);

/*
 * The gated FFN of the routed experts: for a token's expert e with weight a,
 *   y += a * (silu(x w1[e][0]^T) * (x w1[e][1]^T)) w2[e]^T
 * x [T, D] (element strides sr, sc) and the FP32 hidden values are quantised in row blocks; ids [T][k]
 * contiguous (outside 0 .. E - 1: no expert), weights element strides wt, wk; y [T][D] contiguous, of
 * x's type.  Weights are square-block e4m3, rows as in f16acc_mm_fp8 (where
 * f16acc_experts_any_rows says 1, at any address and with anything behind them):
 *   w1 [E][2][I][D] (gate, up), expert stride w1e bytes, up at w1u, rows ld1
 *   s1 of (e, gate or up, n / 128, k / 128): strides s1e, s1u, s1n, s1k
 *   w2 [E][D][I], strides w2e, ld2;  s2: s2e, s2n, s2k
 * Workspace of f16acc_experts_workspace bytes, 256-byte aligned; it is enough for any smaller T too.
 */
int f16acc_experts_any_rows(const void* x, int type, int64_t T, int64_t sr, int64_t sc, int k);
size_t f16acc_experts_workspace(int64_t T, int k, int E, int64_t D, int64_t I);
int f16acc_experts(const void* x, int type, int64_t T, int64_t sr, int64_t sc, const float* weights, int64_t wt,
                   int64_t wk, const int* ids, int k, int E, int64_t D, int64_t I, const uint8_t* w1, int64_t w1e,
                   int64_t w1u, int64_t ld1, const float* s1, int64_t s1e, int64_t s1u, int64_t s1n, int64_t s1k,
                   const uint8_t* w2, int64_t w2e, int64_t ld2, const float* s2, int64_t s2e, int64_t s2n,
                   int64_t s2k, void* y, void* workspace, size_t ws_bytes, void* stream);

/* Short text for a return code of this library (never NULL). */
const char* f16acc_ops_strerror(int code);

/* Bumped whenever a signature above changes. */
int f16acc_ops_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* F16ACC_OPS_H */

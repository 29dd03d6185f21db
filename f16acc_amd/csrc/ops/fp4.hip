// C ABI of the microscaled 4-bit products (include/f16acc_ops.h): argument checks, the
// choice of a kernel, workspaces.
#include "fp4.h"

#include "common.h"
#include "fp4_mm.h"
#include "fp4_small.h"
#include "launch.h"

#include <utility>

using namespace f16ops;

namespace {

int64_t quads_of(int64_t v) { return cdiv(v, kQuad); }

constexpr int64_t kMaxThreads = (int64_t)1 << 32;  // a launch has fewer

uint32_t grid_of(int64_t units, int64_t per_group) {
  const int64_t groups = cdiv(units, per_group);
  return (uint32_t)(groups < 16 * kCus ? groups : 16 * kCus);
}

int64_t tiles_of(const MxQuantArgs& p) { return quads_of(p.rows) * quads_of(p.cols); }

uint32_t quant_grid(const MxQuantArgs& p) {
  const int64_t quads = quads_of(p.cols);
  return p.s.quad == 4 ? grid_of(p.rows * quads, 16) : grid_of(cdiv(p.rows, 16) * quads, 1);
}

int scales_check(const MxScales& s) {
  if (!s.s || s.row < 0 || s.quad < 0) return F16ACC_OPS_E_ARG;
  return (uintptr_t)s.s % 4 || s.row % 4 || s.quad % 4 ? F16ACC_OPS_E_UNSUPPORTED : 0;
}

int out4_check(const uint8_t* q, int64_t ldq, int64_t cols, const MxScales& s) {
  if (!q) return F16ACC_OPS_E_ARG;
  if (ldq != 64 * quads_of(cols) || !aligned16(q)) return F16ACC_OPS_E_UNSUPPORTED;
  return scales_check(s);
}

int matrix_check(const MxQuantArgs& p, int type) {
  int rc = quant_check(p.x, type, p.rows, p.cols);
  if (rc || p.rows == 0 || p.cols == 0) return rc;
  if (!p.q && !p.qt) return F16ACC_OPS_E_ARG;
  if (p.q && (rc = out4_check(p.q, p.ldq, p.cols, p.s))) return rc;
  if (p.qt && (rc = out4_check(p.qt, p.ldqt, p.rows, p.st))) return rc;
  return tiles_of(p) >= kMaxThreads / 512 ? F16ACC_OPS_E_UNSUPPORTED : 0;  // (two matrices, 256 threads a tile)
}

// a and b (rows 0: none), whose tiles are wanted transposed.
template <class T>
int launch_tile(const MxQuantArgs& a, const MxQuantArgs& b, hipStream_t stream) {
  const uint32_t first = (uint32_t)tiles_of(a), all = first + (uint32_t)tiles_of(b);
  if (!std::is_same_v<T, Fp4Source> && a.sc == 1 && (b.sc == 1 || !b.rows))
    hipLaunchKernelGGL((mx_quant_tile_kernel<T, !std::is_same_v<T, Fp4Source>>), dim3(all), dim3(256), 0, stream, a, b, first);
  else
    hipLaunchKernelGGL((mx_quant_tile_kernel<T, false>), dim3(all), dim3(256), 0, stream, a, b, first);
  return hip_status();
}

template <class T>
int launch_rows(const MxQuantArgs& p, hipStream_t stream) {
  const dim3 grid(quant_grid(p));
  if (p.sc == 1)
    hipLaunchKernelGGL((mx_prepare_kernel<T, true>), grid, dim3(256), 0, stream, p, MxScaleArgs{}, Pack8Args{}, 0u, 0u);
  else
    hipLaunchKernelGGL((mx_prepare_kernel<T, false>), grid, dim3(256), 0, stream, p, MxScaleArgs{}, Pack8Args{}, 0u, 0u);
  return hip_status();
}

// The tiles: tokens x weight rows.  A stage of 256 columns everywhere: rows of whole 128-byte lines (with 128
// columns a stage and twice the stages in the ring 8192^3 took 7 % longer).
using Tile0 = Mx4Cfg<256, 256, 4, 2, 256, 2, 2>;
using Tile1 = Mx4Cfg<128, 256, 2, 4, 256, 3, 2>;
using Tile2 = Mx4Cfg<128, 128, 2, 2, 256, 2, 2>;
using Tile3 = Mx4Cfg<64, 128, 2, 2, 256, 3, 2>;
using Tile4 = Mx4Cfg<64, 64, 2, 1, 256, 3, 2>;
using Tile5 = Mx4Cfg<32, 64, 1, 2, 256, 4, 2>;
// What a tile costs, in microseconds, fitted to 2491 timed (shape, tile, split) triples (M 16 .. 8192, N 256 ..
// 16384, K 1536 .. 12288, weights out of the cache, in a graph): a workgroup alone on its CU takes start + step for
// each stage, each further one beside it adds `share` of the stages' time; `per_cu` fit.  The picks made
// with it take 0.1 % longer than the best triple on geometric mean, 3 % at worst.
struct TileInfo {
  int bm, bn, bk, per_cu;
  double start, step, share;
};
constexpr TileInfo kTiles[] = {
    {256, 256, 256, 1, 5.98, 1.134, 0.0}, {128, 256, 256, 1, 3.6, 0.82, 0.0},   {128, 128, 256, 2, 1.9, 0.638, 0.62},
    {64, 128, 256, 2, 2.03, 0.491, 0.46}, {64, 64, 256, 3, 1.97, 0.369, 0.36}, {32, 64, 256, 3, 1.26, 0.349, 0.4},
};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);
constexpr int kThreads[kNumTiles] = {Tile0::THREADS, Tile1::THREADS, Tile2::THREADS,
                                     Tile3::THREADS, Tile4::THREADS, Tile5::THREADS};

struct Plan {
  int tile, ksplit, splits;  // ksplit 0: not split
};

Plan split_of(int tile, int64_t nk, int64_t splits) {
  if (splits > nk) splits = nk;
  const int64_t ks = cdiv(nk, splits), n = cdiv(nk, ks);
  return Plan{tile, n > 1 ? (int)ks : 0, (int)n};
}

double cost_of(const Plan& plan, int64_t M, int64_t N, int64_t K) {
  const TileInfo& t = kTiles[plan.tile];
  const int64_t nk = cdiv(K, t.bk), kb = plan.ksplit ? plan.ksplit : nk;
  const int64_t deep = cdiv(cdiv(M, t.bm) * cdiv(N, t.bn) * plan.splits, kCus);  // workgroups on a CU
  const int64_t full = deep / t.per_cu, rest = deep % t.per_cu;
  double us = full * (t.start + t.step * kb * (1 + (t.per_cu - 1) * t.share));
  if (rest) us += t.start + t.step * kb * (1 + (rest - 1) * t.share);
  const double floor = ((double)N * K + (double)M * K) * 0.107e-6;  // the operands from HBM
  if (us < floor) us = floor;
  const double outputs = (double)M * N * 1e-6;
  us += 0.33 * outputs;
  if (plan.splits > 1) us += 2.64 + 0.28 * plan.splits + 1.33 * plan.splits * outputs;
  return us;
}

Plan plan_of(int64_t M, int64_t N, int64_t K, int tile, int splits) {
  Plan best{};
  double least = 0;
  for (int t = 0; t < kNumTiles; ++t) {
    if (tile >= 0 && t != tile) continue;
    const int64_t nk = cdiv(K, kTiles[t].bk), tiles = cdiv(M, kTiles[t].bm) * cdiv(N, kTiles[t].bn);
    for (const int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
      // (a part of at least two stages; workgroups beyond a few rounds are not split)
      if (splits <= 0 && s > 1 && (s > nk / 2 || tiles * s > 4 * kCus)) break;
      const Plan plan = split_of(t, nk, splits > 0 ? splits : s);
      const double us = cost_of(plan, M, N, K);
      if (least == 0 || us < least) {
        best = plan;
        least = us;
      }
      if (splits > 0) break;
    }
  }
  return best;
}

// Whether a launch holds the product's tiles.
bool launches(const Plan& plan, int64_t M, int64_t N) {
  return cdiv(M, kTiles[plan.tile].bm) * cdiv(N, kTiles[plan.tile].bn) < kMaxThreads / kThreads[plan.tile];
}

size_t parts_bytes(const Plan& plan, int64_t M, int64_t N) {
  return plan.splits > 1 ? up256((size_t)plan.splits * M * N * 4) : 0;
}

int run_product(Mx4Args p, const Plan& plan, void* parts, hipStream_t stream) {
  p.ksplit = plan.ksplit;
  p.parts = (float*)parts;
  int rc = F16ACC_OPS_E_ARG;
  switch (plan.tile) {
    case 0: rc = launch_mm_fp4<Tile0>(p, stream, plan.splits); break;
    case 1: rc = launch_mm_fp4<Tile1>(p, stream, plan.splits); break;
    case 2: rc = launch_mm_fp4<Tile2>(p, stream, plan.splits); break;
    case 3: rc = launch_mm_fp4<Tile3>(p, stream, plan.splits); break;
    case 4: rc = launch_mm_fp4<Tile4>(p, stream, plan.splits); break;
    case 5: rc = launch_mm_fp4<Tile5>(p, stream, plan.splits); break;
  }
  if (rc || plan.splits == 1) return rc;
  FinishArgs f{p.parts, p.M, p.N, p.scm, p.scn, plan.splits, p.bias, p.c};
  return by_type(p.ctype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const int64_t groups = cdiv(p.M * p.N, p.N % 4 ? 256 : 1024);
    hipLaunchKernelGGL((mm_finish_kernel<T>), dim3((uint32_t)(groups < 8 * kCus ? groups : 8 * kCus)), dim3(256), 0,
                       stream, f);
    return hip_status();
  });
}

// Scales of the products' own order: the dword of (row, quad) at (quad * rows + row) * 4.
size_t scale_bytes(int64_t rows, int64_t K) { return up256(quads_of(K) * rows * 4); }

// An operand as a caller has it: bytes of strides (r, c), scales of strides (sr, sb) or, with sq, quads.
struct Stored4 {
  const uint8_t* q;
  int64_t r, c;
  const uint8_t* s;
  int64_t sr, sb, sq;
  int64_t rows;
  bool as_it_is(int64_t K) const {
    return (c == 1 || K <= 2) && aligned16(q) && (rows == 1 || (r % 16 == 0 && r >= cdiv(K, 2) && r <= kMaxRow)) &&
           (K % kMx == 0 || sq);
  }
};

// The workspace of a product: rows that have to be copied, single scale bytes in quads, the parts of a split of K.
struct MmPlan4 {
  Plan plan;
  int64_t ld;
  size_t w, sx, sw, parts, total;
  MmPlan4(const Stored4& x, const Stored4& wt, int64_t K, int tile, int splits) {
    plan = plan_of(x.rows, wt.rows, K, tile, splits);
    ld = cdiv(K, kMx) * 16;
    w = x.as_it_is(K) ? 0 : up256(x.rows * ld);
    sx = w + (wt.as_it_is(K) ? 0 : up256(wt.rows * ld));
    sw = sx + (x.sq ? 0 : scale_bytes(x.rows, K));
    parts = sw + (wt.sq ? 0 : scale_bytes(wt.rows, K));
    total = parts + parts_bytes(plan, x.rows, wt.rows);
  }
};

// Up to 16 tokens in one kernel as long as its workgroups, 16 weight rows each, do not spend more on
// quantising the tokens than the preparing launch costs.  In graphs, cold weights, one kernel / tiles, us: 8960 x 1536
// one token 5.1 / 8.6, eight 7.0 / 8.7, 16 9.5 / 8.6; 4096 x 4096 eight 7.5 / 11.2, 16 10.0 / 11.5; 1024 x 4096 16
// 9.2 / 10.4; 8192 x 4096 eight 12.0 / 12.5, 12 14.6 / 12.6; 1536 x 8960 four 8.6 / 12.3, 12 13.4 / 12.1; 14336 x 4096 two
// 13.1 / 14.9, four 15.4 / 15.0, eight 19.1 / 14.7; 28672 x 7168 one 27.8 / 30.3, eight 46 / 30.
bool few4(int64_t M, int64_t N, int64_t K) {
  return M <= 16 && K < 65536 && cdiv(N, 16) < kMaxThreads / 512 && M * K * cdiv(cdiv(N, 16), kCus) <= 65536;  // (small4_lds at most 36 KB)
}

// Its workgroups have 16 waves where there are no more of them than compute units and K is long enough to give
// each work; 8 otherwise.  (Not by the number of tokens: a token's sums stay in one order, whatever is beside it.)
// 16 waves / 8, us: 1536 x 8960 one token 6.8 / 8.1, eight 10.8 / 13.7; 4096 x 4096 one 5.7 / 5.4, eight 7.6 / 8.1;
// 1536 x 1536 one 3.6 / 3.4, eight 4.1 / 4.2; 8960 x 1536 one 7.8 / 5.1.
bool few4_wide(int64_t N, int64_t K) { return cdiv(N, 16) <= kCus && quads_of(K) >= 24; }

// Bytes between weight rows.  That of a single row addresses nothing, and a caller may hold anything there: the row's
// own extent, which bounds the product's reads.
int64_t row_stride(int64_t N, int64_t K, int64_t ldw) { return N > 1 ? ldw : cdiv(K, kMx) * 16; }

// The workspace of linear: the quantised tokens and their scales, the weight's scales in the
// products' order, the weight where its rows have to be copied, the parts of a split of K.
struct LinearPlan4 {
  Plan plan;
  bool packed;
  int64_t ld;
  size_t sx, sw, weight, parts, total;
  LinearPlan4(int64_t M, int64_t N, int64_t K, const uint8_t* w, int64_t ldw) {
    plan = plan_of(M, N, K, -1, 0);
    packed = !aligned16(w) || ldw % 16 || K % kMx || ldw > kMaxRow;
    ld = cdiv(K, kMx) * 16;
    sx = up256(M * 64 * quads_of(K));
    sw = sx + scale_bytes(M, K);
    weight = sw + scale_bytes(N, K);
    parts = weight + (packed ? up256(N * ld) : 0);
    total = parts + parts_bytes(plan, M, N);
  }
};

}  // namespace

extern "C" {

int f16acc_fp4_quant(const f16acc_fp4_matrix* a, const f16acc_fp4_matrix* b, int type, void* stream_) {
  if (!a) return F16ACC_OPS_E_ARG;
  MxQuantArgs m[2] = {};
  for (int i = 0; i < 2; ++i) {
    const f16acc_fp4_matrix* f = i ? b : a;
    if (!f) continue;
    m[i] = {f->x, f->rows, f->cols, f->sr, f->sc, f->q, f->ldq, {f->s, f->s_row, f->s_quad}, f->qt, f->ldqt,
            {f->st, f->st_row, f->st_quad}, nullptr, 0, 0};
    const int rc = matrix_check(m[i], type);
    if (rc) return rc;
    if (f->rows == 0 || f->cols == 0) m[i].rows = 0;
  }
  hipStream_t stream = (hipStream_t)stream_;
  if (!m[0].rows) std::swap(m[0], m[1]);
  if (!m[0].rows) return 0;
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (m[0].qt && (m[1].qt || !m[1].rows)) return launch_tile<T>(m[0], m[1], stream);
    for (const MxQuantArgs& p : m) {
      const int rc = !p.rows ? 0 : p.qt ? launch_tile<T>(p, MxQuantArgs{}, stream) : launch_rows<T>(p, stream);
      if (rc) return rc;
    }
    return 0;
  });
}

int f16acc_fp4_transpose(const uint8_t* x, int64_t sr, int64_t sc, const uint8_t* s, int64_t s_r, int64_t s_b,
                         int64_t rows, int64_t cols, uint8_t* qt, int64_t ldqt, uint8_t* st, int64_t st_row,
                         int64_t st_quad, void* stream) {
  if (rows > 0 && cols > 0 && !s) return F16ACC_OPS_E_ARG;
  const MxQuantArgs p{x, rows, cols, sr, sc, nullptr, 0, {nullptr, 0, 0}, qt, ldqt, {st, st_row, st_quad}, s, s_r, s_b};
  const int rc = matrix_check(p, 0);
  if (rc || rows == 0 || cols == 0) return rc;
  return launch_tile<Fp4Source>(p, MxQuantArgs{}, (hipStream_t)stream);
}

int f16acc_fp4_values(const uint8_t* q, int64_t q_r, int64_t q_c, const uint8_t* s, int64_t s_r, int64_t s_b,
                      int64_t rows, int64_t cols, void* out, int type, void* stream) {
  int rc = quant_check(q, type, rows, cols);
  if (rc || rows == 0 || cols == 0) return rc;
  if (!s || !out) return F16ACC_OPS_E_ARG;
  if (!aligned16(out)) return F16ACC_OPS_E_UNSUPPORTED;
  const MxValuesArgs p{q, q_r, q_c, s, s_r, s_b, rows, cols, out};
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((mx_values_kernel<T>), dim3(grid_of(rows * cdiv(cols, 8), 256)), dim3(256), 0,
                       (hipStream_t)stream, p);
    return hip_status();
  });
}

size_t f16acc_mm_fp4_workspace(const uint8_t* x, int64_t xr, int64_t xc, int64_t sxq, const uint8_t* w, int64_t wr,
                               int64_t wc, int64_t swq, int64_t M, int64_t N, int64_t K, int tile, int splits) {
  if (M <= 0 || N <= 0 || K <= 0 || tile < -1 || tile >= kNumTiles || splits < 0) return 0;
  return MmPlan4({x, xr, xc, nullptr, 0, 0, sxq, M}, {w, wr, wc, nullptr, 0, 0, swq, N}, K, tile, splits).total;
}

int f16acc_mm_fp4(const uint8_t* x, int64_t xr, int64_t xc, const uint8_t* sx, int64_t sxm, int64_t sxb, int64_t sxq,
                  const uint8_t* w, int64_t wr, int64_t wc, const uint8_t* sw, int64_t swn, int64_t swb, int64_t swq,
                  const void* bias, void* c, int64_t scm, int64_t scn, int64_t M, int64_t N, int64_t K, int ctype,
                  int tile, int splits, void* workspace, size_t ws_bytes, void* stream_) {
  if (tile < -1 || tile >= kNumTiles || splits < 0) return F16ACC_OPS_E_ARG;
  if (M < 0 || N < 0 || K < 0 || ctype < 0 || ctype > F16ACC_TYPE_F32) return F16ACC_OPS_E_ARG;
  if (M == 0 || N == 0) return 0;
  if (K == 0 || !c) return F16ACC_OPS_E_ARG;
  const int64_t blocks = cdiv(K, kMx), bytes = cdiv(K, 2), ld = blocks * 16;
  if (ld > kMaxRow || M > 0x7fffffff || N > 0x7fffffff) return F16ACC_OPS_E_UNSUPPORTED;
  const Stored4 in[2] = {{x, xr, xc, sx, sxm, sxb, sxq, M}, {w, wr, wc, sw, swn, swb, swq, N}};
  int rc = 0;
  for (const Stored4& o : in) {
    if (!o.q || !o.s || o.r < 0 || o.c < 0 || o.sr < 0 || o.sb < 0 || o.sq < 0) return F16ACC_OPS_E_ARG;
    if (o.sq && ((rc = scales_check({(uint8_t*)o.s, o.sr, o.sq})) || o.sr > kMaxRow || !o.as_it_is(K)))
      return rc ? rc : F16ACC_OPS_E_UNSUPPORTED;
  }
  const MmPlan4 plan(in[0], in[1], K, tile, splits);
  if (!launches(plan.plan, M, N)) return F16ACC_OPS_E_UNSUPPORTED;
  if (plan.total && (!workspace || (uintptr_t)workspace % 256 || ws_bytes < plan.total)) return F16ACC_OPS_E_WORKSPACE;
  char* ws = (char*)workspace;
  hipStream_t stream = (hipStream_t)stream_;
  Mx4Args p{x, xr, sx, sxm, sxq, w, wr, sw, swn, swq, bias, c, scm, scn, M, N, K, ctype, 0, nullptr};
  Pack8Args pack[2] = {};
  MxScaleArgs scales[2] = {};
  uint32_t np[2] = {}, ns[2] = {};
  for (int i = 0; i < 2; ++i) {
    const Stored4& o = in[i];
    if (!o.as_it_is(K)) {
      uint8_t* to = (uint8_t*)ws + (i ? plan.w : 0);
      pack[i] = {o.q, to, o.rows, bytes, o.r, o.c, ld};
      np[i] = grid_of(o.rows * (ld / 16), 256);
      (i ? p.w : p.x) = to, (i ? p.ldw : p.ldx) = ld;
    } else if (o.rows == 1) {
      (i ? p.ldw : p.ldx) = ld;  // (the stride of a single row addresses nothing)
    }
    if (!o.sq) {
      uint8_t* to = (uint8_t*)ws + (i ? plan.sw : plan.sx);
      scales[i] = {o.s, o.rows, blocks, o.sr, o.sb, (uint32_t*)to, o.rows};
      ns[i] = grid_of(mx_scales_tiles(scales[i]), 1);
      (i ? p.sw : p.sx) = to, (i ? p.swm : p.sxm) = 4, (i ? p.swq : p.sxq) = 4 * o.rows;
    }
  }
  if (const uint32_t grid = np[0] + np[1] + ns[0] + ns[1]) {
    hipLaunchKernelGGL((K % 2 ? mx_pack_kernel<true> : mx_pack_kernel<false>), dim3(grid), dim3(256), 0, stream, pack[0],
                       pack[1], scales[0], scales[1], np[0], np[1], ns[0]);
    if ((rc = hip_status())) return rc;
  }
  return run_product(p, plan.plan, ws + plan.parts, stream);
}

int f16acc_linear_fp4_few(int64_t M, int64_t N, int64_t K, int64_t sc) {
  return M > 0 && N > 0 && K > 0 && few4(M, N, K) && (sc == 1 || K == 1);
}

size_t f16acc_linear_fp4_workspace(int64_t M, int64_t N, int64_t K, const uint8_t* w, int64_t ldw) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return LinearPlan4(M, N, K, w, row_stride(N, K, ldw)).total;
}

int f16acc_linear_fp4(const void* x, int type, int64_t sr, int64_t sc, const uint8_t* w, int64_t ldw,
                      const uint8_t* sw, int64_t swn, int64_t swb, const void* bias, void* y, int64_t M, int64_t N,
                      int64_t K, void* workspace, size_t ws_bytes, void* stream_) {
  int rc = quant_check(x, type, M, K);
  if (rc) return rc;
  if (N < 0) return F16ACC_OPS_E_ARG;
  if (M == 0 || N == 0) return 0;
  if (K == 0 || !w || !sw || !y || swn < 0 || swb < 0) return F16ACC_OPS_E_ARG;
  ldw = row_stride(N, K, ldw);
  if (ldw < cdiv(K, 2) || 64 * quads_of(K) > kMaxRow || M > 0x7fffffff || N > 0x7fffffff)
    return F16ACC_OPS_E_UNSUPPORTED;
  hipStream_t stream = (hipStream_t)stream_;
  if (f16acc_linear_fp4_few(M, N, K, sc)) {
    const Small4Args a{x, sr, w, ldw, sw, swn, swb, bias, y, M, N, K};
    const size_t lds = small4_lds(M, K);
    return by_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      auto go = [&](auto odd) {
        if (few4_wide(N, K))
          hipLaunchKernelGGL((linear_fp4_small_kernel<T, 16, odd.value>), dim3((uint32_t)cdiv(N, 16)), dim3(1024), lds,
                             stream, a);
        else
          hipLaunchKernelGGL((linear_fp4_small_kernel<T, 8, odd.value>), dim3((uint32_t)cdiv(N, 16)), dim3(512), lds,
                             stream, a);
      };
      if ((uintptr_t)w % 4 || ldw % 4)
        go(std::true_type{});
      else
        go(std::false_type{});
      return hip_status();
    });
  }
  const bool wide = sc == 1;  // (rows of any alignment)
  const LinearPlan4 plan(M, N, K, w, ldw);
  if (!launches(plan.plan, M, N)) return F16ACC_OPS_E_UNSUPPORTED;
  if (!workspace || (uintptr_t)workspace % 256 || ws_bytes < plan.total) return F16ACC_OPS_E_WORKSPACE;
  char* ws = (char*)workspace;
  Mx4Args p{};
  p.x = (const uint8_t*)ws, p.ldx = 64 * quads_of(K);
  p.sx = (const uint8_t*)ws + plan.sx, p.sxm = 4, p.sxq = 4 * M;
  p.w = plan.packed ? (const uint8_t*)ws + plan.weight : w, p.ldw = plan.packed ? plan.ld : ldw;
  p.sw = (const uint8_t*)ws + plan.sw, p.swm = 4, p.swq = 4 * N;
  p.bias = bias, p.c = y, p.scm = N, p.scn = 1, p.M = M, p.N = N, p.K = K, p.ctype = type;
  const MxQuantArgs q{x, M, K, sr, sc, (uint8_t*)ws, p.ldx, {(uint8_t*)p.sx, p.sxm, p.sxq}, nullptr, 0, {nullptr, 0, 0},
                      nullptr, 0, 0};
  const MxScaleArgs s{sw, N, cdiv(K, kMx), swn, swb, (uint32_t*)p.sw, N};
  const Pack8Args pk{w, (uint8_t*)p.w, N, cdiv(K, 2), ldw, 1, plan.ld};
  const uint32_t packs = plan.packed ? grid_of(N * (plan.ld / 16), 256) : 0, scales = grid_of(mx_scales_tiles(s), 1);
  const dim3 grid(packs + scales + quant_grid(q));
  rc = by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (wide)
      hipLaunchKernelGGL((mx_prepare_kernel<T, true>), grid, dim3(256), 0, stream, q, s, pk, packs, scales);
    else
      hipLaunchKernelGGL((mx_prepare_kernel<T, false>), grid, dim3(256), 0, stream, q, s, pk, packs, scales);
    return hip_status();
  });
  if (rc) return rc;
  return run_product(p, plan.plan, ws + plan.parts, stream);
}

}  // extern "C"

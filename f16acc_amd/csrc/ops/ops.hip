// C ABI of the 8-bit block-scaled products and the mixture-of-experts
// operators (include/f16acc_ops.h): argument checks, the choice of a kernel,
// workspaces.
#include "common.h"
#include "launch.h"
#include "layer.h"
#include "mm.h"
#include "moe.h"
#include "quant.h"
#include "small.h"
#include "sums.h"

using namespace f16ops;

namespace {

__global__ __launch_bounds__(256) void pack8_kernel(Pack8Args p) { pack8(p, blockIdx.x, gridDim.x); }

// by_type, and by the groups of four tokens (1, 2 or 4) that hold `tokens`.
template <class F>
int by_tokens(int tokens, int type, F f) {
  return by_type(type, [&](auto* t) {
    if (tokens <= 4) return f(t, std::integral_constant<int, 1>());
    if (tokens <= 8) return f(t, std::integral_constant<int, 2>());
    return f(t, std::integral_constant<int, 4>());
  });
}

int out_check(const uint8_t* q, int64_t ldq, int64_t cols, const float* s) {
  if (!q || !s) return F16ACC_OPS_E_ARG;
  if (ldq < cols || ldq % kBlock || !aligned16(q)) return F16ACC_OPS_E_UNSUPPORTED;
  return 0;
}

int launch_quant_rows(const QuantArgs& p, int type, hipStream_t stream) {
  const int64_t groups = cdiv(p.rows * (p.ldq / kBlock), 16);
  if (groups == 0) return 0;
  const uint32_t grid = (uint32_t)(groups < 16 * kCus ? groups : 16 * kCus);
  const bool wide = wide_loads(p.x, type, p.sr, p.sc);
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (wide)
      hipLaunchKernelGGL((quant_rows_kernel<T, true>), dim3(grid), dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL((quant_rows_kernel<T, false>), dim3(grid), dim3(256), 0, stream, p);
    return hip_status();
  });
}

template <bool ROWS, bool COLS, bool SQUARE>
int quant_tile(const QuantArgs& p, int type, hipStream_t stream) {
  const int64_t gx = cdiv(p.cols, kBlock), gy = cdiv(p.rows, kBlock);
  if (gx == 0 || gy == 0) return 0;
  if (gx > 0x7fffffff || gy > 65535) return F16ACC_OPS_E_UNSUPPORTED;
  const bool wide = wide_loads(p.x, type, p.sr, p.sc);
  const dim3 grid((uint32_t)gx, (uint32_t)gy);
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (wide)
      hipLaunchKernelGGL((quant_tile_kernel<T, true, ROWS, COLS, SQUARE>), grid, dim3(512), 0, stream, p);
    else
      hipLaunchKernelGGL((quant_tile_kernel<T, false, ROWS, COLS, SQUARE>), grid, dim3(512), 0, stream, p);
    return hip_status();
  });
}

// Parts of the rows of a column sum: four workgroups a CU, of 256 rows at least.
int64_t sum_parts(int64_t rows, int64_t cols) {
  const int64_t want = cdiv(4 * kCus, cdiv(cols, 64)), most = cdiv(rows, 256);
  return want < most ? want : most > 1 ? most : 1;
}

int mm_check(const MmArgs& p) {
  if (p.M < 0 || p.N < 0 || p.K < 0 || p.ctype < 0 || p.ctype > F16ACC_TYPE_F32) return F16ACC_OPS_E_ARG;
  if (p.M == 0 || p.N == 0) return 0;
  if (p.K == 0 || !p.c || !p.x || !p.w || !p.sx || !p.sw) return F16ACC_OPS_E_ARG;
  if (p.sxm < 0 || p.sxk < 0 || p.swn < 0 || p.swk < 0) return F16ACC_OPS_E_ARG;
  if (p.ldx % 16 || p.ldw % 16 || p.ldx < p.K || p.ldw < p.K || p.ldx > kMaxRow || p.ldw > kMaxRow ||
      !aligned16(p.x) || !aligned16(p.w))
    return F16ACC_OPS_E_UNSUPPORTED;
  if (p.sxm > kMaxRow / 4 || p.swn > kMaxRow / 4 || p.M > 0x7fffffff || p.N > 0x7fffffff)
    return F16ACC_OPS_E_UNSUPPORTED;
  return 0;
}

// The tiles of one product (F16ACC_FP8_TILE_*): tokens x weight rows.
using Tile0 = MmCfg<256, 256, 4, 2, 2, 2>;
using Tile1 = MmCfg<128, 256, 2, 4, 3, 2>;
using Tile2 = MmCfg<128, 128, 2, 2, 2, 2>;
using Tile3 = MmCfg<64, 128, 2, 2, 3, 2>;
using Tile4 = MmCfg<64, 64, 2, 1, 3, 2>;
using Tile5 = MmCfg<32, 64, 1, 2, 4, 2>;
// What a tile costs, in microseconds, fitted to 5010 timed (shape, tile, split)
// triples (M 32 .. 8192, N 256 .. 8960, K 512 .. 9000, weights out of the cache; 438
// with row scales): a workgroup alone on its CU takes start + kb * block, each
// further one beside it adds `share` of the blocks' time; `per_cu` fit.  The
// picks made with it take 1.2 % (row scales 0.03 %) longer than the best triple on
// geometric mean, 10 % at worst (profiles/fp8_tile_choices.txt has each).
struct TileCost {
  double start, block, share;
};
struct TileInfo {
  int bm, bn, per_cu;
  TileCost square, row;  // row.block 0: not built with row scales
};
constexpr TileInfo kTiles[] = {
    {256, 256, 1, {3.8, 1.20, 0.6}, {7.1, 1.79, 0.6}},    {128, 256, 1, {2.3, 0.745, 0.6}, {}},
    {128, 128, 2, {2.2, 0.60, 0.61}, {3.2, 0.67, 0.62}},  {64, 128, 2, {1.9, 0.45, 0.55}, {}},
    {64, 64, 3, {1.7, 0.43, 0.33}, {2.1, 0.41, 0.34}},    {32, 64, 3, {1.3, 0.34, 0.32}, {}},
};
constexpr int kNumTiles = sizeof(kTiles) / sizeof(kTiles[0]);

struct MmPlan {
  int tile, ksplit, splits;  // ksplit 0: not split
};

MmPlan split_of(int tile, int64_t nk, int64_t splits) {
  if (splits > nk) splits = nk;
  const int64_t ks = cdiv(nk, splits), n = cdiv(nk, ks);
  return MmPlan{tile, n > 1 ? (int)ks : 0, (int)n};
}

double cost_of(const MmPlan& plan, int64_t M, int64_t N, int64_t K, bool row_scales) {
  const TileInfo& t = kTiles[plan.tile];
  const TileCost& c = row_scales ? t.row : t.square;
  const int64_t nk = cdiv(K, kBlock), kb = plan.ksplit ? plan.ksplit : nk;
  const int64_t deep = cdiv(cdiv(M, t.bm) * cdiv(N, t.bn) * plan.splits, kCus);  // workgroups on a CU
  const int64_t full = deep / t.per_cu, rest = deep % t.per_cu;
  double us = full * (c.start + c.block * kb * (1 + (t.per_cu - 1) * c.share));
  if (rest) us += c.start + c.block * kb * (1 + (rest - 1) * c.share);
  const double floor = ((double)N * K + (double)M * K) * 0.17e-6;  // the operands from HBM
  if (us < floor) us = floor;
  const double outputs = (double)M * N * 1e-6;
  if (t.per_cu == 1) us += 0.3 * outputs;  // no other workgroup runs while one stores
  if (plan.splits > 1) us += 2.1 + 0.25 * plan.splits + 1.36 * plan.splits * outputs;
  return us;
}

MmPlan mm_plan(int64_t M, int64_t N, int64_t K, bool row_scales, int tile, int splits) {
  const int64_t nk = cdiv(K, kBlock);
  MmPlan best{};
  double least = 0;
  for (int t = 0; t < kNumTiles; ++t) {
    if ((tile >= 0 && t != tile) || (row_scales && kTiles[t].row.block == 0)) continue;
    const int64_t tiles = cdiv(M, kTiles[t].bm) * cdiv(N, kTiles[t].bn);
    for (const int s : {1, 2, 3, 4, 6, 8, 12, 16}) {
      // (a part of at least two blocks; workgroups beyond a few rounds are not split)
      const int64_t want = splits > 0 ? splits : s;
      if (splits <= 0 && s > 1 && (s > nk / 2 || tiles * s > 4 * kCus)) break;
      const MmPlan plan = split_of(t, nk, want);
      const double us = cost_of(plan, M, N, K, row_scales);
      if (least == 0 || us < least) {
        best = plan;
        least = us;
      }
      if (splits > 0) break;
    }
  }
  return best;
}

size_t parts_bytes(const MmPlan& plan, int64_t M, int64_t N) {
  return plan.splits > 1 ? (size_t)plan.splits * M * N * 4 : 0;
}

template <bool ROW_SCALES>
int mm_run(MmArgs p, const MmPlan& plan, void* workspace, hipStream_t stream) {
  p.ksplit = plan.ksplit;
  p.parts = (float*)workspace;
  auto run = [&](auto* c) {
    using C = std::remove_pointer_t<decltype(c)>;
    return launch_mm<C, ROW_SCALES, false, kStore>(p, cdiv(p.M, C::BM), stream, plan.splits);
  };
  int rc = F16ACC_OPS_E_ARG;
  if constexpr (ROW_SCALES) {
    switch (plan.tile) {
      case 0: rc = run((Tile0*)nullptr); break;
      case 2: rc = run((Tile2*)nullptr); break;
      case 4: rc = run((Tile4*)nullptr); break;
    }
  } else {
    switch (plan.tile) {
      case 0: rc = run((Tile0*)nullptr); break;
      case 1: rc = run((Tile1*)nullptr); break;
      case 2: rc = run((Tile2*)nullptr); break;
      case 3: rc = run((Tile3*)nullptr); break;
      case 4: rc = run((Tile4*)nullptr); break;
      case 5: rc = run((Tile5*)nullptr); break;
    }
  }
  if (rc || plan.splits == 1) return rc;
  FinishArgs f{p.parts, p.M, p.N, p.scm, p.scn, plan.splits, p.bias, p.c};
  const int64_t groups = cdiv(p.M * p.N, p.N % 4 ? 256 : 1024);
  return by_type(p.ctype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((mm_finish_kernel<T>), dim3((uint32_t)(groups < 8 * kCus ? groups : 8 * kCus)), dim3(256), 0,
                       stream, f);
    return hip_status();
  });
}

// The workspace of linear: the quantised tokens and their scales, the weight where its rows
// have to be copied, the parts of a split of K.
struct LinearPlan {
  bool packed;
  int64_t ld;
  size_t scales, weight, parts, total;
  LinearPlan(int64_t M, int64_t N, int64_t K, const uint8_t* w, int64_t ldw) {
    packed = !aligned16(w) || ldw % 16 || K % 16 || ldw > kMaxRow;
    ld = cdiv(K, 16) * 16;
    scales = up256(M * up128(K));
    weight = scales + up256(M * cdiv(K, kBlock) * 4);
    parts = weight + (packed ? up256(N * ld) : 0);
    total = parts + up256(parts_bytes(mm_plan(M, N, K, false, -1, 0), M, N));
  }
};

// The experts' tiles by the mean number of tokens an expert has: gate and up (128
// columns of each), down.  In all, in us, bfloat16, in a graph, for 64 experts of 2048 x 1024 with 8 a
// token, 16 of 4096 x 2048 with 2, 128 of 1024 x 512 with 4:
//   16 tokens an expert: on 32 102, 112, 60; on 128 106, 110, 63
//   24 tokens an expert: on 32 119, 137, 70; on 128 108, 113, 65
//   192, 8-bit sums:     on 128 185, 164, 139; on 256 166, 153, 128
//   512, 8-bit sums:     on 128 421, 380, 314; on 256 391, 351, 282
// (the last with down on 128: 410, 361, 300).
template <int ROWS>
struct ExpertCfg;
template <>
struct ExpertCfg<32> {
  using GateUp = MmCfg<32, 256, 1, 4, 4, 1>;
  using Down = MmCfg<32, 64, 1, 2, 4, 2>;
};
template <>
struct ExpertCfg<128> {
  using GateUp = MmCfg<128, 256, 2, 4, 3, 2>;
  using Down = MmCfg<128, 128, 2, 2, 2, 2>;
};
template <>
struct ExpertCfg<256> {
  using GateUp = MmCfg<256, 256, 4, 2, 2, 2>;
  using Down = MmCfg<256, 256, 4, 2, 2, 2>;
};

int expert_tile(int64_t slots, int E) {
  const int64_t mean = slots / E;
  return mean >= 192 ? 256 : mean >= 24 ? 128 : 32;
}

// Whether the two kernels for a few tokens run (if x's rows allow their loads).
bool few_tokens(int64_t T, int k) { return T <= kFewTokens && T * k <= kFewSlots; }

int64_t tile_count(int64_t slots, int E, int bm) { return slots / bm + (slots < E ? slots : E); }

// Where things lie in the workspace, and its size, which is enough for any smaller T as well: the
// tile list has room for the smallest tiles, and the hidden values of the kernels for a few
// tokens for as many tokens as they may take.
struct ExpertsPlan {
  int64_t slots, chunks, max_tiles, Dp, Ip;
  int bm;
  int64_t ldy;
  size_t xq, xs, hq, hs, ys, counts, rows, pos, tiles, ntiles, total;
  ExpertsPlan(int64_t T, int k, int E, int64_t D, int64_t I) {
    slots = T * k;
    Dp = up128(D);
    Ip = up128(I);
    bm = expert_tile(slots, E);
    chunks = cdiv(slots, kSortChunk);
    max_tiles = tile_count(slots, E, bm);
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += up256(bytes);
      return here;
    };
    xq = take(T * Dp);
    xs = take(T * (Dp / kBlock) * 4);
    hq = take(slots * Ip);
    hs = take(slots * (Ip / kBlock) * 4);
    ldy = cdiv(D, 8) * 8;
    ys = take(slots * ldy * 4);
    counts = take(chunks * E * 4);
    rows = take(slots * 4);
    pos = take(slots * 4);
    tiles = take(tile_count(slots, E, 32) * 16);
    ntiles = take(4);
    total = at;
    if (few_tokens(1, k)) {
      const int64_t t = kFewSlots / k < kFewTokens ? kFewSlots / k : kFewTokens;
      const size_t hidden = up256((T < t ? T : t) * k * Ip * 4) + up256(sizeof(FewMap));
      if (total < hidden) total = hidden;
    }
  }
};

// The experts' weights as the C entry points get them.
struct ExpertWeights {
  const uint8_t* w1;
  int64_t w1e, w1u, ld1;
  const float* s1;
  int64_t s1e, s1u, s1n, s1k;
  const uint8_t* w2;
  int64_t w2e, ld2;
  const float* s2;
  int64_t s2e, s2n, s2k;
};

int experts_check(const void* x, int type, int64_t T, int k, int E, int64_t D, int64_t I, const ExpertWeights& w,
                  const void* y, bool few) {
  const int rc = quant_check(x, type, T, D);
  if (rc) return rc;
  if (k < 1 || E < 1 || D < 1 || I < 1) return F16ACC_OPS_E_ARG;
  if (T == 0) return 0;
  if (!w.w1 || !w.s1 || !w.w2 || !w.s2 || !y) return F16ACC_OPS_E_ARG;
  if (w.w1e < 0 || w.w1u < 0 || w.s1e < 0 || w.s1u < 0 || w.s1n < 0 || w.s1k < 0 || w.w2e < 0 || w.s2e < 0 ||
      w.s2n < 0 || w.s2k < 0)
    return F16ACC_OPS_E_ARG;
  if (E > kMaxExperts || w.ld1 < 0 || w.ld2 < 0 || up128(D) > kMaxRow || up128(I) > kMaxRow)
    return F16ACC_OPS_E_UNSUPPORTED;
  if (!few && (w.ld1 % 16 || w.ld2 % 16 || w.w1e % 16 || w.w1u % 16 || w.w2e % 16 || w.ld1 < D || w.ld2 < I ||
               w.ld1 > kMaxRow || w.ld2 > kMaxRow || !aligned16(w.w1) || !aligned16(w.w2)))
    return F16ACC_OPS_E_UNSUPPORTED;
  // the copies address a token's (a slot's) row by a 31-bit offset
  if (T > kOob / up128(D) || T > kOob / ((int64_t)k * up128(I))) return F16ACC_OPS_E_UNSUPPORTED;
  return 0;
}

// EXACT: gate and up on the 16-bit matrix instructions.  Up to 191 tokens an expert, where
// weights are most of the time, they always do (in all, 64 experts of 2048 x 1024, 8 a
// token, exact / 8-bit: 64 tokens 100 / 97 us, 512 132 / 117, 1024 185 / 153).  Past that
// matrix instructions are the time (4096: 525 / 358), and it goes by the type: results in
// binary16 and FP32 show the difference (2.7e-4 and 8e-5 of the 2-norm off, or 1.5e-3),
// beside bfloat16's own rounding of 1.7e-3 it makes 2.3e-3 and the 8-bit sums stay.
template <int BM, bool EXACT>
int expert_products(const MmArgs& gu, const MmArgs& down, int64_t max_tiles, hipStream_t stream) {
  using GateUp = typename ExpertCfg<EXACT && BM == 256 ? 128 : BM>::GateUp;
  const int rc = launch_mm<GateUp, false, true, EXACT ? kGatedExact : kGatedQuant>(gu, max_tiles * (BM / GateUp::BM), stream);
  if (rc) return rc;
  using Down = typename ExpertCfg<BM>::Down;
  return launch_mm<Down, false, true, kStore>(down, max_tiles * (BM / Down::BM), stream);
}

template <template <class, int> class Launch, class... A>
int by_experts(int E, int type, A&&... args) {
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (E <= 64) return Launch<T, 1>::go(args...);
    if (E <= 128) return Launch<T, 2>::go(args...);
    if (E <= 256) return Launch<T, 4>::go(args...);
    if (E <= 512) return Launch<T, 8>::go(args...);
    return Launch<T, 16>::go(args...);
  });
}
// What the scores' loads and the groups' exchanges rely on, for V experts a lane.
template <class T, int V>
RouteArgs route_args(RouteArgs a) {
  a.wide = a.se == 1 && a.E % V == 0 && a.st % V == 0 && (uintptr_t)a.x % (V * sizeof(T) < 16 ? V * sizeof(T) : 16) == 0;
  const int size = a.groups ? a.E / a.groups : 0, lanes = size / V;
  a.lanes = a.groups > 1 && size % V == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  return a;
}
template <class T, int V>
struct LaunchRoute {
  static int go(RouteArgs a, hipStream_t s) {
    a = route_args<T, V>(a);
    hipLaunchKernelGGL((route_kernel<T, V>), dim3((uint32_t)cdiv(a.T, 4)), dim3(256), 0, s, a);
    return hip_status();
  }
};
template <class T, int V>
struct LaunchRouteGrad {
  static int go(RouteArgs a, hipStream_t s) {
    a = route_args<T, V>(a);
    hipLaunchKernelGGL((route_grad_kernel<T, V>), dim3((uint32_t)cdiv(a.T, 4)), dim3(256), 0, s, a);
    return hip_status();
  }
};

// The router's product.  wide: rows of both as the loads of eight elements need them.
template <class T, class R>
void router_wide(RouterArgs& p) {
  p.wide = p.sc == 1 && p.rd == 1 && aligned16(p.x) && aligned16(p.r) && p.sr * (int64_t)sizeof(T) % 16 == 0 &&
           p.re * (int64_t)sizeof(R) % 16 == 0;
}
// Four waves of 32 x 32 where there are enough workgroups of them, 16 of 16 x 16 otherwise; 32 x 32 / 16 x 16, 2048 wide, us:
// 16384 tokens of 256 experts 342 / 528, of 64 108 / 136, 4096 of 256 (4096 wide) 201 / 245, of 64 40 / 29.
template <class T, class R>
int launch_router(RouterArgs p, hipStream_t stream) {
  router_wide<T, R>(p);
  if (cdiv(p.T, 32) * cdiv(p.E, 32) >= 4 * kCus)
    hipLaunchKernelGGL((router_kernel<T, R, 4, 2>), dim3((uint32_t)cdiv(p.T, 32), (uint32_t)cdiv(p.E, 32)), dim3(256),
                       0, stream, p);
  else
    hipLaunchKernelGGL((router_kernel<T, R, 16, 1>), dim3((uint32_t)cdiv(p.T, 16), (uint32_t)cdiv(p.E, 16)), dim3(1024),
                       0, stream, p);
  return hip_status();
}

template <class T, int V>
struct LaunchLayer {
  static int go(LayerArgs a, hipStream_t s) {
    a.route = route_args<float, V>(a.route);
    const int64_t grid = a.e.slots * (int64_t)a.pieces + cdiv(a.e.D, 16);
    hipLaunchKernelGGL((layer_few_kernel<V>), dim3((uint32_t)grid), dim3(64 * LayerFew::W), 0, s, a);
    return hip_status();
  }
};

// Whether a layer of few tokens takes two launches, or the router's product, route and experts one after another.  Each 16
// hidden columns of a slot are a workgroup, which chooses the experts for itself and starts on cold weights: many more of
// them than fit at once cost more than the launches they save, which the result's D / 16 workgroups hide the
// longer, the wider it is.  Two launches / one after another, in a graph, us, at 2, 4, 8, 12 and 16 slots: 64 experts,
// 2048 x 1024 17 / 25, 21 / 28, 32 / 35, 40 / 43, 47 to 54 / 47 to 50; 128 of 4096 x 1536 27 / 40, 37 / 45, 54 / 64, 77 / 82,
// 91 / 84; 32 of 7168 x 2048 43 / 62, 57 / 73, 95 / 106, 113 / 110, 158 / 161; 64 of 512 x 1536 16 / 22, 19 / 25, 32 / 32, 42 / 38,
// 60 / 47; 8 of 2048 x 5632 38 / 42, 61 / 60, 107 / 91, 128 / 89, 152 / 100; 8 of 4096 x 14336 68 to 106 / 59 to 109, 200 / 177,
// 340 / 258, 391 / 278, 464 / 308 (one slot 63 / 67).
bool layer_in_two(int64_t slots, int64_t D, int64_t I) { return slots * I < 9216 + 3 * D; }

// Where a layer's values lie in its workspace, and its size, which is enough for any smaller T as well: logits,
// weights and ids before the experts' own; or logits, quantised tokens, hidden values and counters of a few tokens.
struct LayerPlan {
  size_t logits, weights, ids, experts, xq, xs, h, sync, claims, total;
  LayerPlan(int64_t T, int k, int E, int64_t D, int64_t I) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += up256(bytes);
      return here;
    };
    logits = take(T * E * 4);
    weights = take(T * k * 4);
    ids = take(T * k * 4);
    experts = at;
    total = at + ExpertsPlan(T, k, E, D, I).total;
    if (few_tokens(1, k)) {
      const int64_t most = kFewSlots / k < kFewTokens ? kFewSlots / k : kFewTokens, t = T < most ? T : most;
      at = up256(t * E * 4);
      xq = take(t * up128(D));
      xs = take(t * (up128(D) / kBlock) * 4);
      h = take(t * k * up128(I) * 4);
      sync = take(sizeof(LayerSync));
      claims = take(t * k * cdiv(I, 16) * sizeof(Claim));
      if (total < at) total = at;
    }
  }
};

int route_check(const RouteArgs& a, int type) {
  if (a.T < 0 || type < 0 || type > F16ACC_TYPE_F32 || a.E < 1 || a.k < 1 || a.k > a.E) return F16ACC_OPS_E_ARG;
  if (a.E > kMaxExperts || a.k > 64 || a.T > 0x7fffffff) return F16ACC_OPS_E_UNSUPPORTED;
  if (a.T && (!a.x || !a.ids)) return F16ACC_OPS_E_ARG;
  return 0;
}

int groups_check(const RouteArgs& a) {
  if (a.groups < 1 || a.E % a.groups || a.top < 1 || a.top > a.groups || a.k > a.E / a.groups * a.top)
    return F16ACC_OPS_E_ARG;
  return a.groups > 64 ? F16ACC_OPS_E_UNSUPPORTED : 0;
}

}  // namespace

extern "C" {

int f16acc_quant_rows(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                      int64_t ldq, float* s, int64_t lds, void* stream) {
  int rc = quant_check(x, type, rows, cols);
  if (rc || rows == 0 || cols == 0) return rc;
  rc = out_check(q, ldq, cols, s);
  if (rc) return rc;
  QuantArgs p{x, rows, cols, sr, sc, q, ldq, s, lds, nullptr, 0, nullptr, 0};
  return launch_quant_rows(p, type, (hipStream_t)stream);
}

int f16acc_quant_both(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                      int64_t ldq, float* s, int64_t lds, uint8_t* qt, int64_t ldqt, float* st, int64_t ldst,
                      void* stream) {
  int rc = quant_check(x, type, rows, cols);
  if (rc || rows == 0 || cols == 0) return rc;
  if (!q && !qt) return F16ACC_OPS_E_ARG;
  if (q && (rc = out_check(q, ldq, cols, s))) return rc;
  if (qt && (rc = out_check(qt, ldqt, rows, st))) return rc;
  if (q && ldq != up128(cols)) return F16ACC_OPS_E_UNSUPPORTED;
  if (qt && ldqt != up128(rows)) return F16ACC_OPS_E_UNSUPPORTED;
  QuantArgs p{x, rows, cols, sr, sc, q, ldq, s, lds, qt, ldqt, st, ldst};
  if (q && qt) return quant_tile<true, true, false>(p, type, (hipStream_t)stream);
  if (qt) return quant_tile<false, true, false>(p, type, (hipStream_t)stream);
  return launch_quant_rows(p, type, (hipStream_t)stream);
}

int f16acc_quant_weight(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, uint8_t* q,
                        int64_t ldq, float* s, int64_t lds, uint8_t* qt, int64_t ldqt, void* stream) {
  int rc = quant_check(x, type, rows, cols);
  if (rc || rows == 0 || cols == 0) return rc;
  rc = out_check(q, ldq, cols, s);
  if (!rc && qt) rc = out_check(qt, ldqt, rows, s);
  if (rc) return rc;
  if (ldq != up128(cols) || (qt && ldqt != up128(rows))) return F16ACC_OPS_E_UNSUPPORTED;
  QuantArgs p{x, rows, cols, sr, sc, q, ldq, s, lds, qt, ldqt, nullptr, 0};
  return qt ? quant_tile<true, true, true>(p, type, (hipStream_t)stream)
            : quant_tile<true, false, true>(p, type, (hipStream_t)stream);
}

int f16acc_pack8(const uint8_t* src, uint8_t* dst, int64_t rows, int64_t cols, int64_t s_r, int64_t s_c, int64_t ld,
                 void* stream) {
  if (rows < 0 || cols < 0 || ld < cols) return F16ACC_OPS_E_ARG;
  if (rows == 0 || ld == 0) return 0;
  if (!dst || (cols && !src)) return F16ACC_OPS_E_ARG;
  if (ld % 16 || !aligned16(dst) || rows > kMaxExtent || ld > kMaxExtent) return F16ACC_OPS_E_UNSUPPORTED;
  Pack8Args p{src, dst, rows, cols, s_r, s_c, ld};
  const int64_t groups = cdiv(rows * (ld / 16), 256);
  hipLaunchKernelGGL(pack8_kernel, dim3((uint32_t)(groups < 16 * kCus ? groups : 16 * kCus)), dim3(256), 0,
                     (hipStream_t)stream, p);
  return hip_status();
}

size_t f16acc_column_sums_workspace(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || rows > kMaxExtent || cols > kMaxExtent) return 0;
  const int64_t parts = sum_parts(rows, cols);
  return parts > 1 ? up256(parts * cols * 4) : 0;
}

int f16acc_column_sums(const void* x, int type, int64_t rows, int64_t cols, int64_t sr, int64_t sc, void* out,
                       void* workspace, size_t ws_bytes, void* stream) {
  const int rc = quant_check(x, type, rows, cols);
  if (rc || cols == 0) return rc;
  if (!out) return F16ACC_OPS_E_ARG;
  if (cols > 0x3fffffff) return F16ACC_OPS_E_UNSUPPORTED;
  const size_t need = f16acc_column_sums_workspace(rows, cols);
  if (need && (!workspace || (uintptr_t)workspace % 256 || ws_bytes < need)) return F16ACC_OPS_E_WORKSPACE;
  const int64_t parts = sum_parts(rows, cols);
  const uint32_t gx = (uint32_t)cdiv(cols, 64);
  const SumArgs p{x, rows, cols, sr, sc, cdiv(rows, parts), parts > 1 ? workspace : out};
  const SumArgs join{workspace, parts, cols, cols, 1, parts, out};
  return by_type(type, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (parts == 1) {
      hipLaunchKernelGGL((column_sums_kernel<T, T>), dim3(gx), dim3(256), 0, (hipStream_t)stream, p);
    } else {
      hipLaunchKernelGGL((column_sums_kernel<T, float>), dim3(gx, (uint32_t)parts), dim3(256), 0, (hipStream_t)stream, p);
      hipLaunchKernelGGL((column_sums_kernel<float, T>), dim3(gx), dim3(256), 0, (hipStream_t)stream, join);
    }
    return hip_status();
  });
}

int f16acc_mm_fp8(const uint8_t* x, int64_t ldx, const float* sx, int64_t sxm, int64_t sxk, const uint8_t* w,
                  int64_t ldw, const float* sw, int64_t swn, int64_t swk, int row_scales, const void* bias, void* c,
                  int64_t scm, int64_t scn, int64_t M, int64_t N, int64_t K, int ctype, int tile, int splits,
                  void* workspace, size_t ws_bytes, void* stream) {
  if (row_scales != 0 && row_scales != 1) return F16ACC_OPS_E_ARG;
  if (tile < -1 || tile >= kNumTiles || splits < 0) return F16ACC_OPS_E_ARG;
  if (tile >= 0 && row_scales && kTiles[tile].row.block == 0) return F16ACC_OPS_E_ARG;
  MmArgs p{};
  p.x = x, p.ldx = ldx, p.sx = sx, p.sxm = sxm, p.sxk = sxk;
  p.w = w, p.ldw = ldw, p.sw = sw, p.swn = swn, p.swk = swk;
  p.bias = bias, p.c = c, p.scm = scm, p.scn = scn, p.M = M, p.N = N, p.K = K, p.ctype = ctype;
  const int rc = mm_check(p);
  if (rc || M == 0 || N == 0) return rc;
  const MmPlan plan = mm_plan(M, N, K, row_scales, tile, splits);
  const size_t need = parts_bytes(plan, M, N);
  if (need && (!workspace || (uintptr_t)workspace % 256 || ws_bytes < need)) return F16ACC_OPS_E_WORKSPACE;
  return row_scales ? mm_run<true>(p, plan, workspace, (hipStream_t)stream)
                    : mm_run<false>(p, plan, workspace, (hipStream_t)stream);
}

size_t f16acc_mm_fp8_workspace(int64_t M, int64_t N, int64_t K, int row_scales, int tile, int splits) {
  if (M <= 0 || N <= 0 || K <= 0 || tile < -1 || tile >= kNumTiles || splits < 0) return 0;
  if (tile >= 0 && row_scales && kTiles[tile].row.block == 0) return 0;
  return up256(parts_bytes(mm_plan(M, N, K, row_scales != 0, tile, splits), M, N));
}

size_t f16acc_linear_fp8_workspace(int64_t M, int64_t N, int64_t K, const uint8_t* w, int64_t ldw) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return LinearPlan(M, N, K, w, ldw).total;
}

int f16acc_linear_fp8(const void* x, int type, int64_t sr, int64_t sc, const uint8_t* w, int64_t ldw, const float* sw,
                      int64_t swn, int64_t swk, const void* bias, void* y, int64_t M, int64_t N, int64_t K,
                      void* workspace, size_t ws_bytes, void* stream_) {
  int rc = quant_check(x, type, M, K);
  if (rc) return rc;
  if (N < 0) return F16ACC_OPS_E_ARG;
  if (M == 0 || N == 0) return 0;
  if (K == 0 || !w || !sw || !y || swn < 0 || swk < 0) return F16ACC_OPS_E_ARG;
  if (ldw < K && N > 1) return F16ACC_OPS_E_UNSUPPORTED;
  hipStream_t stream = (hipStream_t)stream_;
  const LinearPlan plan(M, N, K, w, ldw);
  if (!workspace || (uintptr_t)workspace % 256 || ws_bytes < plan.total) return F16ACC_OPS_E_WORKSPACE;
  // Few tokens: one launch, from the rows as they are.  From 9 tokens on its quantising,
  // repeated by every workgroup, costs more than a pass of its own where there are many (16 tokens,
  // here / on the tiles, in a graph: 1536 x 1536 5.5 / 10.2 us, 4096 x 4096 10.7 / 12.6, 8960 x 1536
  // 11.3 / 10.2, 8192 x 8192 31 / 22; 8 tokens: 4.6 / 10.0, 8.4 / 12.3, 7.8 / 10.2, 21.4 / 21.2).
  if ((M <= 8 || (M <= 16 && N * K <= (1 << 25))) && wide_loads(x, type, sr, sc)) {
    SmallArgs a{x, sr, w, ldw, sw, swn, swk, bias, y, N, 1, M, N, K};
    return by_tokens((int)M, type, [&](auto* t, auto groups) {
      using T = std::remove_pointer_t<decltype(t)>;
      constexpr int G = decltype(groups)::value;
      // 16 waves deal K where no CU has two workgroups (one token: 4096 x 4096 7.3 us against 8.0
      // on 8 waves, 1536 x 8960 8.5 and 12.1, 1536 x 1536 4.1 and 4.5; 8960 x 1536 7.5 and 6.5)
      if (cdiv(N, 16) <= kCus && cdiv(K, kBlock) >= 12)
        hipLaunchKernelGGL((linear_small_kernel<T, 16, G>), dim3((uint32_t)cdiv(N, 16)), dim3(1024), 0, stream, a);
      else
        hipLaunchKernelGGL((linear_small_kernel<T, 8, G>), dim3((uint32_t)cdiv(N, 16)), dim3(512), 0, stream, a);
      return hip_status();
    });
  }
  char* ws = (char*)workspace;
  MmArgs p{};
  p.x = (const uint8_t*)ws, p.ldx = up128(K);
  p.sx = (const float*)(ws + plan.scales), p.sxm = 1, p.sxk = M;
  p.w = plan.packed ? (const uint8_t*)ws + plan.weight : w, p.ldw = plan.packed ? plan.ld : ldw;
  p.sw = sw, p.swn = swn, p.swk = swk;
  p.bias = bias, p.c = y, p.scm = N, p.scn = 1, p.M = M, p.N = N, p.K = K, p.ctype = type;
  rc = mm_check(p);
  if (rc) return rc;
  QuantArgs q{x, M, K, sr, sc, (uint8_t*)ws, p.ldx, (float*)p.sx, M, nullptr, 0, nullptr, 0};
  if (plan.packed) {
    Pack8Args pk{w, (uint8_t*)p.w, N, K, ldw, 1, plan.ld};
    const int64_t packs = cdiv(N * (plan.ld / 16), 256), groups = cdiv(M * (p.ldx / kBlock), 16);
    const uint32_t np = (uint32_t)(packs < 16 * kCus ? packs : 16 * kCus);
    const dim3 grid(np + (uint32_t)(groups < 16 * kCus ? groups : 16 * kCus));
    const bool wide = wide_loads(x, type, sr, sc);
    rc = by_type(type, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      if (wide)
        hipLaunchKernelGGL((quant_pack_kernel<T, true>), grid, dim3(256), 0, stream, q, pk, np);
      else
        hipLaunchKernelGGL((quant_pack_kernel<T, false>), grid, dim3(256), 0, stream, q, pk, np);
      return hip_status();
    });
  } else {
    rc = launch_quant_rows(q, type, stream);
  }
  if (rc) return rc;
  return mm_run<false>(p, mm_plan(M, N, K, false, -1, 0), ws + plan.parts, stream);
}

int f16acc_route(const void* logits, int type, int64_t T, int64_t st, int64_t se, int E, int k, int sigmoid,
                 const float* bias, int groups, int top, int renorm, float scale, float* weights, int* ids,
                 void* stream) {
  RouteArgs a{logits, T, st, se, E, k, sigmoid, bias, groups, top, renorm, scale, weights, ids, nullptr, 0, 0, nullptr, false, 0, false};
  int rc = route_check(a, type);
  if (!rc) rc = groups_check(a);
  if (rc) return rc;
  if (T && !weights) return F16ACC_OPS_E_ARG;
  if (T == 0) return 0;
  return by_experts<LaunchRoute>(E, type, a, (hipStream_t)stream);
}

int f16acc_route_grad(const void* logits, int type, int64_t T, int64_t st, int64_t se, int E, int k, int sigmoid,
                      int renorm, float scale, const int* ids, const float* dw, int64_t dwt, int64_t dwk,
                      void* dlogits, void* stream) {
  RouteArgs a{logits, T, st, se, E, k, sigmoid, nullptr, 1, 1, renorm, scale, nullptr, (int*)ids, dw, dwt, dwk, dlogits, false, 0, false};
  const int rc = route_check(a, type);
  if (rc) return rc;
  if (T && (!dw || !dlogits)) return F16ACC_OPS_E_ARG;
  if (!aligned16(dlogits)) return F16ACC_OPS_E_UNSUPPORTED;
  if (T == 0) return 0;
  return by_experts<LaunchRouteGrad>(E, type, a, (hipStream_t)stream);
}

int f16acc_experts_any_rows(const void* x, int type, int64_t T, int64_t sr, int64_t sc, int k) {
  return T > 0 && k > 0 && few_tokens(T, k) && wide_loads(x, type, sr, sc);
}

size_t f16acc_experts_workspace(int64_t T, int k, int E, int64_t D, int64_t I) {
  if (T <= 0 || k <= 0 || E <= 0 || D <= 0 || I <= 0) return 0;
  return ExpertsPlan(T, k, E, D, I).total;
}

int f16acc_experts(const void* x, int type, int64_t T, int64_t sr, int64_t sc, const float* weights, int64_t wt,
                   int64_t wk, const int* ids, int k, int E, int64_t D, int64_t I, const uint8_t* w1, int64_t w1e,
                   int64_t w1u, int64_t ld1, const float* s1, int64_t s1e, int64_t s1u, int64_t s1n, int64_t s1k,
                   const uint8_t* w2, int64_t w2e, int64_t ld2, const float* s2, int64_t s2e, int64_t s2n,
                   int64_t s2k, void* y, void* workspace, size_t ws_bytes, void* stream_) {
  const ExpertWeights w{w1, w1e, w1u, ld1, s1, s1e, s1u, s1n, s1k, w2, w2e, ld2, s2, s2e, s2n, s2k};
  const bool few = f16acc_experts_any_rows(x, type, T, sr, sc, k);
  int rc = experts_check(x, type, T, k, E, D, I, w, y, few);
  if (rc || T == 0) return rc;
  if (!weights || !ids) return F16ACC_OPS_E_ARG;
  const ExpertsPlan plan(T, k, E, D, I);
  if (!workspace || (uintptr_t)workspace % 256 || ws_bytes < plan.total) return F16ACC_OPS_E_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_;
  char* ws = (char*)workspace;
  if (few) {
    FewArgs f{x,   sr,  (int)T, k,   E,   (int)plan.slots, ids, weights, wt,  wk,  D,   I, w1,          w1e,     w1u,
              ld1, s1,  s1e,    s1u, s1n, s1k,             w2,  w2e,     ld2, s2,  s2e, s2n, s2k, (float*)ws, plan.Ip,
              (FewMap*)(ws + up256(plan.slots * plan.Ip * 4)), y};
    return by_type(type, [&](auto* t) {
      using U = std::remove_pointer_t<decltype(t)>;
      constexpr int G = (kFewTokens + 3) / 4;
      hipLaunchKernelGGL((few_gate_up_kernel<U, 8, G>), dim3((uint32_t)cdiv(I, 32), (uint32_t)plan.slots + 1), dim3(512), 0,
                         stream, f);
      hipLaunchKernelGGL((few_down_kernel<U, 16, G>), dim3((uint32_t)cdiv(D, 16)), dim3(1024), 0, stream, f);
      return hip_status();
    });
  }
  QuantArgs q{x, T, D, sr, sc, (uint8_t*)(ws + plan.xq), plan.Dp, (float*)(ws + plan.xs), T, nullptr, 0, nullptr, 0};
  SortArgs so{ids, plan.slots, E, k, plan.bm, (int*)(ws + plan.counts), (int*)(ws + plan.rows), (int*)(ws + plan.pos),
              (int4*)(ws + plan.tiles), (int*)(ws + plan.ntiles), (int)plan.chunks};
  const int64_t groups = cdiv(T * (plan.Dp / kBlock), 16);
  const dim3 quant_grid((uint32_t)(so.chunks + (groups < 16 * kCus ? groups : 16 * kCus)));
  const bool wide = wide_loads(x, type, sr, sc);
  rc = by_type(type, [&](auto* t) {
    using U = std::remove_pointer_t<decltype(t)>;
    if (wide)
      hipLaunchKernelGGL((quant_count_kernel<U, true>), quant_grid, dim3(256), 0, stream, q, so);
    else
      hipLaunchKernelGGL((quant_count_kernel<U, false>), quant_grid, dim3(256), 0, stream, q, so);
    hipLaunchKernelGGL(sort_place_kernel, dim3(so.chunks), dim3(1024), 0, stream, so);
    return hip_status();
  });
  if (rc) return rc;

  MmArgs gu{};
  gu.x = q.q, gu.ldx = plan.Dp, gu.sx = q.s, gu.sxm = 1, gu.sxk = T;
  gu.w = w1, gu.ldw = ld1, gu.sw = s1, gu.swn = s1n, gu.swk = s1k, gu.we = w1e, gu.swe = s1e, gu.up = w1u, gu.sup = s1u;
  gu.M = plan.slots, gu.N = I, gu.K = D;
  gu.tiles = so.tiles, gu.ntiles = so.ntiles, gu.rows = so.rows, gu.xrows = T;
  gu.q = (uint8_t*)(ws + plan.hq), gu.ldq = plan.Ip, gu.sq = (float*)(ws + plan.hs), gu.ldsq = plan.slots;
  MmArgs down{};
  down.x = gu.q, down.ldx = plan.Ip, down.sx = gu.sq, down.sxm = 1, down.sxk = plan.slots;
  down.w = w2, down.ldw = ld2, down.sw = s2, down.swn = s2n, down.swk = s2k, down.we = w2e, down.swe = s2e;
  down.c = ws + plan.ys, down.scm = plan.ldy, down.scn = 1;
  gu.tile_rows = down.tile_rows = plan.bm;
  down.M = plan.slots, down.N = D, down.K = I;
  down.tiles = so.tiles, down.ntiles = so.ntiles, down.rows = nullptr, down.xrows = plan.slots;
  rc = plan.bm == 32    ? expert_products<32, true>(gu, down, plan.max_tiles, stream)
       : plan.bm == 128 ? expert_products<128, true>(gu, down, plan.max_tiles, stream)
       : type == F16ACC_TYPE_BF16 ? expert_products<256, false>(gu, down, plan.max_tiles, stream)
                                  : expert_products<256, true>(gu, down, plan.max_tiles, stream);
  if (rc) return rc;

  CombineArgs co{(const float*)(ws + plan.ys), plan.ldy, weights, wt, wk, so.pos, T, D, k, y};
  const dim3 grid((uint32_t)T, (uint32_t)cdiv(cdiv(D, 8), 256));
  return by_type(type, [&](auto* t) {
    using U = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL((combine_kernel<U>), grid, dim3(256), 0, stream, co);
    return hip_status();
  });
}

int f16acc_layer_any_rows(int64_t T, int k, int64_t D, int64_t I) {
  return T > 0 && k > 0 && few_tokens(T, k) && D >= 16 && I >= 16;
}

size_t f16acc_layer_workspace(int64_t T, int k, int E, int64_t D, int64_t I) {
  if (T <= 0 || k <= 0 || E <= 0 || D <= 0 || I <= 0) return 0;
  return LayerPlan(T, k, E, D, I).total;
}

int f16acc_layer(const void* x, int type, int64_t T, int64_t sr, int64_t sc, const void* router, int rtype, int64_t re,
                 int64_t rd, int E, int k, int sigmoid, const float* bias, int groups, int top, int renorm, float scale,
                 int64_t D, int64_t I, const uint8_t* w1, int64_t w1e, int64_t w1u, int64_t ld1, const float* s1,
                 int64_t s1e, int64_t s1u, int64_t s1n, int64_t s1k, const uint8_t* w2, int64_t w2e, int64_t ld2,
                 const float* s2, int64_t s2e, int64_t s2n, int64_t s2k, void* y, void* workspace, size_t ws_bytes,
                 void* stream_) {
  const ExpertWeights w{w1, w1e, w1u, ld1, s1, s1e, s1u, s1n, s1k, w2, w2e, ld2, s2, s2e, s2n, s2k};
  bool few = f16acc_layer_any_rows(T, k, D, I);
  int rc = experts_check(x, type, T, k, E, D, I, w, y, few);
  if (!rc) rc = quant_check(router, rtype, E, D);
  if (rc || T == 0) return rc;
  // (what is not there yet is not looked at)
  RouteArgs a{router, T, E, 1, E, k, sigmoid, bias, groups, top, renorm, scale, nullptr, (int*)router, nullptr, 0, 0, nullptr,
              false, 0, true};
  if ((rc = route_check(a, F16ACC_TYPE_F32)) || (rc = groups_check(a))) return rc;
  const LayerPlan plan(T, k, E, D, I);
  if (!workspace || (uintptr_t)workspace % 256 || ws_bytes < plan.total) return F16ACC_OPS_E_WORKSPACE;
  char* ws = (char*)workspace;
  float *logits = (float*)(ws + plan.logits), *weights = (float*)(ws + plan.weights);
  int* ids = (int*)(ws + plan.ids);
  const RouterArgs r{x, T, sr, sc, router, re, rd, E, D, false, logits};
  a.x = logits, a.weights = weights, a.ids = ids;
  // (the experts take any rows of the weights where they can load x wide)
  if (few && !layer_in_two(T * k, D, I) && f16acc_experts_any_rows(x, type, T, sr, sc, k)) few = false;
  if (few) {
    const int64_t Dp = up128(D), Ip = up128(I);
    LayerArgs l{};
    l.router = r, l.route = a, l.ytype = type, l.wide = wide_loads(x, type, sr, sc), l.sync = (LayerSync*)(ws + plan.sync);
    l.pieces = (int)cdiv(I, 16), l.claims = (Claim*)(ws + plan.claims);
    l.quant = QuantArgs{x, T, D, sr, sc, (uint8_t*)(ws + plan.xq), Dp, (float*)(ws + plan.xs), T, nullptr, 0, nullptr, 0};
    l.e = FewArgs{x,   sr,  (int)T, k,   E,   (int)(T * k), nullptr, nullptr, 0,   0,   D,   I, w1,          w1e, w1u,
                  ld1, s1,  s1e,    s1u, s1n, s1k,          w2,      w2e,     ld2, s2,  s2e, s2n, s2k, (float*)(ws + plan.h), Ip,
                  nullptr, y};
    rc = by_type(type, [&](auto* t) {
      using X = std::remove_pointer_t<decltype(t)>;
      return by_type(rtype, [&](auto* u) {
        using R = std::remove_pointer_t<decltype(u)>;
        router_wide<X, R>(l.router);
        const uint32_t grid = (uint32_t)(E + cdiv(T * (Dp / kBlock), 16));
        hipLaunchKernelGGL((layer_router_kernel<X, R>), dim3(grid), dim3(256), 0, (hipStream_t)stream_, l);
        return hip_status();
      });
    });
    return rc ? rc : by_experts<LaunchLayer>(E, F16ACC_TYPE_F32, l, (hipStream_t)stream_);
  }
  rc = by_type(type, [&](auto* t) {
    using X = std::remove_pointer_t<decltype(t)>;
    return by_type(rtype, [&](auto* u) {
      using R = std::remove_pointer_t<decltype(u)>;
      return launch_router<X, R>(r, (hipStream_t)stream_);
    });
  });
  if (rc) return rc;
  rc = by_experts<LaunchRoute>(E, F16ACC_TYPE_F32, a, (hipStream_t)stream_);
  if (rc) return rc;
  return f16acc_experts(x, type, T, sr, sc, weights, k, 1, ids, k, E, D, I, w1, w1e, w1u, ld1, s1, s1e, s1u, s1n, s1k, w2,
                        w2e, ld2, s2, s2e, s2n, s2k, y, ws + plan.experts, ws_bytes - plan.experts, stream_);
}

const char* f16acc_ops_strerror(int code) {
  switch (code) {
    case 0: return "f16acc: success";
    case F16ACC_OPS_E_ARG: return "f16acc: invalid argument";
    case F16ACC_OPS_E_UNSUPPORTED: return "f16acc: extent, stride or alignment not supported";
    case F16ACC_OPS_E_WORKSPACE: return "f16acc: workspace missing, misaligned or too small";
  }
  return code > 0 ? hipGetErrorString((hipError_t)code) : "f16acc: unknown error";
}

int f16acc_ops_abi_version(void) { return 1; }

}  // extern "C"

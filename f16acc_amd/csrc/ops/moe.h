// Mixture of experts around the products: routing and its gradient, the slots
// sorted by expert, the weighted sum of the experts' results.
#pragma once

#include "common.h"
#include "quant.h"

namespace f16ops {

struct RouteArgs {
  const void* x;  // [T][E] logits
  int64_t T, st, se;
  int E, k;
  int sigmoid;
  const float* bias;  // [E] or NULL
  int groups, top;
  int renorm;
  float scale;
  float* weights;  // [T][k]
  int* ids;        // [T][k]
  // gradient
  const float* dw;  // [T][k], stride dwt between tokens, dwk between experts
  int64_t dwt, dwk;
  void* dx;  // [T][E] contiguous
  bool wide;     // a lane's V logits are one load
  int lanes;     // lanes of a group where that is a power of two, else 0
  bool nan_id;   // a token with a NaN logit and no expert gets the first one, so what follows sees its NaN weight
};

// Order-preserving map of a float to an unsigned integer, -inf lowest; 0 is
// kept for "not available".
__device__ __forceinline__ uint32_t sortable(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = umax(v, dpp<0x111>(v));  // row_shr:1 .. 8: lane 15 of each row holds the row's
  v = umax(v, dpp<0x112>(v));
  v = umax(v, dpp<0x114>(v));
  v = umax(v, dpp<0x118>(v));
  v = umax(v, dpp<0x142>(v));  // row_bcast:15, row_bcast:31: lane 63 holds the wave's
  v = umax(v, dpp<0x143>(v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// The scores of a token, V experts a lane: lane l holds experts V l .. V l + V - 1.
// x: the logits as FP32, -inf past E; p: softmax or sigmoid.  `nan` tells
// whether any logit is NaN.
template <class T, int V>
__device__ __forceinline__ void scores(const RouteArgs& a, int64_t t, int lane, float (&x)[V], float (&p)[V],
                                       bool* nan) {
  const T* row = (const T*)a.x + t * a.st;
  bool bad = false;
  if (a.wide) {  // V divides E and rows are aligned to V elements
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = -INFINITY;
    if (lane * V < a.E) load_vec(row + lane * V, x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = lane * V + i < a.E ? (float)row[(lane * V + i) * a.se] : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) bad |= x[i] != x[i];
  *nan = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = 1.0f / (1.0f + expf(-x[i]));
  } else {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (m == -INFINITY) m = 0.0f;  // no expert available: every p is 0
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      p[i] = expf(x[i] - m);
      sum += p[i];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = sum > 0.0f || sum != sum ? p[i] / sum : 0.0f;
  }
}

// One wave a token.  Measured: 16384 tokens, 256 experts in 8 groups, FP32, 22 us
// (the scores' 16.8 MB are 3.4 at the copy rate) and 11 us for the gradient (33.6
// MB, 6.7).  Bound by instructions: exponentials and quotients of 256 scores, eight
// selections.  Selection: k times the wave's largest key (a DPP maximum),
// the lowest lane that holds it (ballot) and that lane's lowest expert, which
// is the lowest index since a lane's experts are consecutive.
// Lane j < k gets the j-th expert and its weight; `row` are 64 V floats of the wave's own.
template <class T, int V>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t t, int lane, float* row, int* expert,
                                            float* weight) {
  float x[V], p[V];
  bool nan;
  scores<T, V>(a, t, lane, x, p, &nan);
  uint32_t key[V];
  float keys[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    float f = x[i];
    if (a.sigmoid || a.bias) f = p[i] + (a.bias && e < a.E ? a.bias[e] : 0.0f);
    if (!(x[i] > -INFINITY) || !(f > -INFINITY) || e >= a.E) f = -INFINITY;
    key[i] = f > -INFINITY ? sortable(f + 0.0f) : 0u;  // (-0 and 0 are a tie)
    keys[i] = f;
  }
  if (a.lanes) {
    // groups of whole lanes: the best key, for sigmoid scores the best two's sum, by
    // exchanges within the group's lanes
    float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      b2 = fmaxf(b2, fminf(b1, keys[i]));
      b1 = fmaxf(b1, keys[i]);
    }
    for (int d = 1; d < a.lanes; d <<= 1) {
      const float o1 = __shfl_xor(b1, d), o2 = __shfl_xor(b2, d);
      b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
      b1 = fmaxf(b1, o1);
    }
    const float score = a.sigmoid && b2 > -INFINITY ? b1 + b2 : b1;
    const int mine = lane / a.lanes;
    int rank = 0;
    for (int j = 0; j < a.groups; ++j) {
      const float o = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(score), j * a.lanes));
      rank += o > score || (o == score && j < mine);
    }
    if (rank >= a.top) {
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = 0u;
    }
  } else if (a.groups > 1) {
    // a lane per group
#pragma unroll
    for (int i = 0; i < V; ++i) row[lane * V + i] = keys[i];
    wave_sync();
    const int size = a.E / a.groups;
    float b1 = -INFINITY, b2 = -INFINITY;
    if (lane < a.groups)
      for (int i = 0; i < size; ++i) {
        const float f = row[lane * size + i];
        b2 = fmaxf(b2, fminf(b1, f));
        b1 = fmaxf(b1, f);
      }
    const float score = a.sigmoid && b2 > -INFINITY ? b1 + b2 : b1;
    int rank = 0;
    for (int j = 0; j < a.groups; ++j) {
      const float o = __shfl(score, j);
      rank += o > score || (o == score && j < lane);
    }
    const uint64_t kept = __builtin_amdgcn_ballot_w64(lane < a.groups && rank < a.top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      if (e < a.E && !((kept >> (e / size)) & 1)) key[i] = 0u;
    }
  }
  float mine = 0.0f;  // lane j < k: the j-th selected score
  int id = -1;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = key[0];
    int at = 0;
    float pv = p[0];
#pragma unroll
    for (int i = 1; i < V; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
        pv = p[i];
      }
    const uint32_t top = wave_umax(best);
    if (top == 0u) break;
    const int src = __builtin_ctzll(__builtin_amdgcn_ballot_w64(best == top));
    const int e = src * V + __builtin_amdgcn_readlane(at, src);
    const float pe = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(pv), src));
    if (lane == j) {
      id = e;
      mine = pe;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane == src && i == at) key[i] = 0u;
  }
  if (a.renorm) mine = mine / (wave_sum(mine) + 1e-20f);
  if (nan) {
    mine = __uint_as_float(0x7fc00000u);
    if (a.nan_id && lane == 0 && id < 0) id = 0;
  }
  *expert = id;
  *weight = mine * a.scale;
}

template <class T, int V>
__global__ __launch_bounds__(256) void route_kernel(RouteArgs a) {
  __shared__ float lds[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  int id;
  float weight;
  route_token<T, V>(a, t, lane, lds[wave], &id, &weight);
  if (lane < a.k) {
    a.weights[t * a.k + lane] = weight;
    a.ids[t * a.k + lane] = id;
  }
}

// dlogits of a token from its scores, recomputed, and the selected experts.
//   renormalised: dp_j = g_j / S - (sum_i g_i p_i) / S^2, S = sum p + 1e-20
//   softmax: dx = p (dp - sum dp p); sigmoid: dx = dp p (1 - p)
template <class T, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteArgs a) {
  __shared__ float lds[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  float x[V], p[V];
  bool nan;
  scores<T, V>(a, t, lane, x, p, &nan);
#pragma unroll
  for (int i = 0; i < V; ++i) lds[wave][lane * V + i] = p[i];
  wave_sync();
  int id = -1;
  float g = 0.0f, sel = 0.0f;
  if (lane < a.k) {
    id = a.ids[t * a.k + lane];
    if (id >= 0 && id < a.E) {
      g = a.dw[t * a.dwt + lane * a.dwk] * a.scale;
      sel = lds[wave][id];
    } else {
      id = -1;
    }
  }
  if (a.renorm) {
    const float total = wave_sum(sel) + 1e-20f;
    g = g / total - wave_sum(g * sel) / (total * total);
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < V; ++i) lds[wave][lane * V + i] = 0.0f;
  wave_sync();
  if (id >= 0) lds[wave][id] = g;
  wave_sync();
  float dp[V], dot = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    dp[i] = lds[wave][lane * V + i];
    dot += dp[i] * p[i];
  }
  if (!a.sigmoid) dot = wave_sum(dot);
  T* out = (T*)a.dx + t * a.E + lane * V;
  struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Pack {
    T t[V];
  } o;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float d = a.sigmoid ? dp[i] * p[i] * (1.0f - p[i]) : p[i] * (dp[i] - dot);
    o.t[i] = (T)(nan ? __uint_as_float(0x7fc00000u) : d);
  }
  if (a.E % V == 0) {  // (the rows are aligned to V elements then: dx is contiguous)
    if (lane * V < a.E) *(Pack*)out = o;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane * V + i < a.E) out[i] = o.t[i];
  }
}

// Slots (token t's j-th expert is slot t k + j) sorted by expert, in slot order
// within one, without atomics on the order: every position is a count.
// Two launches: chunks of slots are counted by expert (beside the quantising of
// the tokens, which needs no sorting); then every chunk adds up the counts before
// its own and places its slots, and the first also writes the products' tiles.
struct SortArgs {
  const int* ids;
  int64_t slots;
  int E, k, bm;  // bm: tokens per tile of the products
  int* counts;   // [chunks][E]
  int* rows;     // [sorted position] -> token
  int* pos;      // [slot] -> sorted position, -1: none
  int4* tiles;   // (expert, first, end, 0)
  int* ntiles;
  int chunks;
};
constexpr int kSortChunk = 512;  // slots of one workgroup

__device__ __forceinline__ void count_chunk(const SortArgs& a, int chunk, int* hist) {
  for (int e = threadIdx.x; e < a.E; e += 256) hist[e] = 0;
  __syncthreads();
  const int64_t s0 = (int64_t)chunk * kSortChunk;
#pragma unroll
  for (int i = 0; i < kSortChunk; i += 256) {
    const int64_t s = s0 + i + threadIdx.x;
    const int e = s < a.slots ? a.ids[s] : -1;
    if (e >= 0 && e < a.E) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += 256) a.counts[(int64_t)chunk * a.E + e] = hist[e];
}

template <class T, bool WIDE>
__global__ __launch_bounds__(256) void quant_count_kernel(QuantArgs q, SortArgs a) {
  __shared__ int hist[kMaxExperts];
  if ((int)blockIdx.x < a.chunks)
    count_chunk(a, blockIdx.x, hist);
  else
    quant_rows<T, WIDE>(q, blockIdx.x - a.chunks, gridDim.x - a.chunks);
}

// The waves of a chunk take turns in slot order; within one, a slot's rank is
// the number of lower lanes with its expert.
__global__ __launch_bounds__(1024) void sort_place_kernel(SortArgs a) {
  __shared__ int next[kMaxExperts], sums[kMaxExperts], first[kMaxExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // per expert: all its slots, and those of earlier chunks; `per` threads an expert
  for (int e = tid; e < kMaxExperts; e += 1024) sums[e] = next[e] = 0;
  __syncthreads();
  int p2 = 1;
  while (p2 < a.E) p2 <<= 1;
  const int per = kMaxExperts / p2, e0 = tid & (p2 - 1), part = tid / p2;
  if (e0 < a.E) {
    int all = 0, before = 0;
#pragma unroll 4
    for (int c = part; c < a.chunks; c += per) {
      const int n = a.counts[(int64_t)c * a.E + e0];
      all += n;
      before += c < (int)blockIdx.x ? n : 0;
    }
    if (all) atomicAdd(&sums[e0], all);
    if (before) atomicAdd(&next[e0], before);
  }
  __syncthreads();
  const int total = sums[tid], tiles = (total + a.bm - 1) / a.bm;
  __syncthreads();
  // inclusive sums over the experts, of slots and of tiles
  int begin = total, tile = tiles;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(begin, d), v = __shfl_up(tile, d);
    if (lane >= d) begin += u, tile += v;
  }
  if (lane == 63) sums[wave] = begin, first[wave] = tile;
  __syncthreads();
  for (int w = 0; w < wave; ++w) begin += sums[w], tile += first[w];
  next[tid] += begin - total;
  if (blockIdx.x == 0) {
    if (tid == kMaxExperts - 1) *a.ntiles = tile;
    int at = begin - total;
    for (int t = tile - tiles; t < tile; ++t, at += a.bm)
      a.tiles[t] = int4{tid, at, at + a.bm < begin ? at + a.bm : begin, 0};
  }
  __syncthreads();
  const int64_t s = (int64_t)blockIdx.x * kSortChunk + tid;
  const bool mine = tid < kSortChunk && s < a.slots;
  const int e = mine ? a.ids[s] : -1;
  const bool in = e >= 0 && e < a.E;
  uint64_t same = __builtin_amdgcn_ballot_w64(in);
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    const uint64_t m = __builtin_amdgcn_ballot_w64((e >> b) & 1);
    same &= (e >> b) & 1 ? m : ~m;
  }
  const int rank = __popcll(same & ((1ull << lane) - 1)), n = __popcll(same);
  int p = -1;
#pragma unroll
  for (int w = 0; w < kSortChunk / 64; ++w) {
    if (w == wave && in) {
      p = next[e] + rank;
      if (rank == n - 1) next[e] = p + 1;
    }
    lds_barrier();
  }
  if (mine) a.pos[s] = p;
  if (in) a.rows[p] = (int)(s / a.k);
}

// y[t] = sum_j weights[t][j] * ys[pos[t][j]], j in order, FP32, rounded once.
// A thread takes eight columns; bound by reading ys.
struct CombineArgs {
  const float* ys;  // [slots][ld]
  int64_t ld;
  const float* weights;
  int64_t wt, wk;
  const int* pos;
  int64_t T, D;
  int k;
  void* y;  // [T][D]
};
template <class T>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  const int64_t t = blockIdx.x, n = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  if (n >= a.D) return;
  float sum[8] = {};
#pragma unroll 4
  for (int j = 0; j < a.k; ++j) {
    const int p = a.pos[t * a.k + j];
    if (p < 0) continue;
    const float w = a.weights[t * a.wt + j * a.wk];
    float v[8];
    load_vec(a.ys + p * a.ld + n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = __builtin_fmaf(w, v[i], sum[i]);
  }
  T* y = (T*)a.y + t * a.D + n;
  if (a.D % 8 == 0) {
    struct alignas(16) Pack {
      T t[8];
    } o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.t[i] = (T)sum[i];
    *(Pack*)y = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < a.D) y[i] = (T)sum[i];
  }
}

}  // namespace f16ops

// A whole mixture-of-experts layer: the router's product, and for a few tokens everything behind it in one
// more kernel.
#pragma once

#include "common.h"
#include "moe.h"
#include "quant.h"
#include "small.h"

namespace f16ops {

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct RouterArgs {
  const void* x;  // [T][D]
  int64_t T, sr, sc;  // element strides
  const void* r;  // [E][D]
  int64_t re, rd;
  int E;
  int64_t D;
  bool wide;      // rows of both are whole 16-byte units, eight elements a load
  float* logits;  // [T][E]
};

// Eight elements of a row from k, zero past the end.
template <class T>
__device__ __forceinline__ void load8(const T* p, int64_t stride, int64_t k, int64_t D, bool wide, float (&v)[8]) {
  if (wide && k + 8 <= D)
    load_vec(p + k, v);
  else
    load_clamped(p, k, D, stride, v);
}
// ... as they are.
template <class T>
__device__ __forceinline__ void fetch8(const T* p, int64_t stride, int64_t k, int64_t D, bool wide, T (&v)[8]) {
  if (wide && k + 8 <= D) {
    __builtin_memcpy(v, p + k, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[(k + i < D ? k + i : D - 1) * stride];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < D ? v[i] : (T)0.0f;
  }
}

// logits[t][e] = sum over d of x[t][d] r[e][d], summed in 64 bits and rounded once to FP32: products of 16-bit and
// FP32 values are exact there.  The three kernels (16 waves, 4 waves, 256 lanes
// of layer_router_kernel) add in different orders, so where a sum is not exact a token's logits, and with them the choice
// of its experts, can depend on the batch it comes in: if the sum lies within its rounding, 2^-53 of the magnitudes for each
// addition, of the middle between two FP32 values.  16 F tokens by 16 F experts a workgroup on v_mfma_f64_16x16x4_f64; the waves deal the
// chunks of 32 columns, a lane loads eight of a row, and their sums meet in LDS in wave order.  512 tokens of 64
// experts, 2048 wide: 11 us in 16 waves, two chunks ahead each (15 in eight, with one), of 8 MB and 2 us of matrix
// instructions: the launch, and two rounds of loads.  16384 tokens of 256 experts: 340 us with F = 2, of which
// the matrix instructions take 220 at their peak.
template <class T, class R, int W, int F>
__global__ __launch_bounds__(64 * W) void router_kernel(RouterArgs p) {
  __shared__ f64x4 sums[W][F * F][64];
  static_assert(F * F <= W, "a wave joins a fragment's sums");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int64_t t0 = (int64_t)blockIdx.x * 16 * F + l16;
  const int e0 = (int)blockIdx.y * 16 * F;
  const T* x[F];
  const R* r[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    x[f] = (const T*)p.x + (t0 + 16 * f < p.T ? t0 + 16 * f : p.T - 1) * p.sr;
    r[f] = (const R*)p.r + (e0 + 16 * f + l16 < p.E ? e0 + 16 * f + l16 : p.E - 1) * p.re;
  }
  constexpr int AHEAD = 2;  // chunks in flight
  f64x4 acc[F][F] = {};
  T a[AHEAD][F][8];
  R b[AHEAD][F][8];
  auto load = [&](int i, int64_t chunk) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      fetch8(x[f], p.sc, chunk + 8 * g, p.D, p.wide, a[i][f]);
      fetch8(r[f], p.rd, chunk + 8 * g, p.D, p.wide, b[i][f]);
    }
  };
  constexpr int64_t step = 32 * W;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(i, 32 * wave + i * step);
#pragma unroll 1
  for (int64_t c = 32 * wave; c < p.D; c += AHEAD * step) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {  // (past the end zeros)
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int m = 0; m < F; ++m)
#pragma unroll
          for (int n = 0; n < F; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)b[i][m][k], (double)(float)a[i][n][k],
                                                             acc[m][n], 0, 0, 0);
      if (c + AHEAD * step < p.D) load(i, c + (AHEAD + i) * step);
    }
  }
#pragma unroll
  for (int f = 0; f < F * F; ++f) sums[wave][f][lane] = acc[f / F][f % F];
  __syncthreads();
  const int64_t t = t0 + 16 * (wave % F);
  if (wave >= F * F || t >= p.T) return;
  f64x4 sum = sums[0][wave][lane];
#pragma unroll
  for (int i = 1; i < W; ++i) sum += sums[i][wave][lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = e0 + 16 * (wave / F) + g + 4 * i;
    if (row < p.E) p.logits[t * p.E + row] = (float)sum[i];
  }
}

// ---------------------------------------------------------------------------
// The layer of at most 4 tokens and 16 slots in two launches.  The first sums the logits, an expert a workgroup, and
// quantises the tokens beside it.  In the second every workgroup chooses the tokens' experts for itself (a
// wave a token); the first ones take 16 hidden columns of one expert, gate and up, the last ones 16 columns of
// the result each.  The latter load their weights, which depend on the choice alone, before they wait for
// the hidden values.
//
// The wait ends: a piece of hidden columns is claimed by who computes it, and who computes one waits for nobody.
// Before it waits, a workgroup sees that every piece is claimed and computes those that are not, so it
// takes neither a number of workgroups at once nor an order of theirs.  (An order of them is a matter of speed: with the
// result's workgroups first, those that fit beside none of the others raced for their pieces, 124 us instead of
// 48 for two tokens, 8 of 64 experts, 2048 x 1024, a size that is composed now.)
//
// Measured, in a graph, against the router's product, route and experts one after another, which take over where the
// slots' hidden columns are many (layer_in_two, with the figures), us: 64 experts, 2048 x 1024, one token, 2 of them
// 17 / 25, 6 (38 MB of weights, 7.6 us at the copy rate) 22 / 31, 8 32 / 35, two tokens, 6 40 / 43; 128 experts,
// 4096 x 1536, one token, 1 of them 23 / 36, 8 54 / 65; 32 experts, 7168 x 2048, one token, 8 of them 95 / 107.  Of 22
// us the logits take 4, the choice 3.5, gate and up 5
// to 7, at the rate of memory, and 9 pass from their last sums to the result: stores past the L2, a count, a
// poll, hidden values from memory, each a trip of a microsecond or two.
// ---------------------------------------------------------------------------

// The counters, in lines of their own: adds to one address follow each other at some 10 ns.
constexpr int kDoneLines = 16;
struct LayerSync {
  struct Line {
    int n, pad[31];
  } done[kDoneLines];  // pieces whose hidden values are written
};
struct Claim {
  int taken, pad[3];
};

struct LayerArgs {
  RouterArgs router;
  RouteArgs route;
  QuantArgs quant;  // the tokens: [T][Dp] and the scale of (token, block) at [block][T]
  bool wide;        // (16-byte loads of the tokens)
  FewArgs e;
  int ytype;
  int pieces;  // of an expert's hidden columns
  LayerSync* sync;
  Claim* claims;  // [slots][pieces]
};

template <class T, class R>
__global__ __launch_bounds__(256) void layer_router_kernel(LayerArgs a) {
  const RouterArgs& p = a.router;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)a.e.slots * a.pieces; i += (int64_t)gridDim.x * 256)
    a.claims[i].taken = 0;
  if ((int)blockIdx.x >= p.E) {
    if (a.wide)
      quant_rows<T, true>(a.quant, blockIdx.x - p.E, gridDim.x - p.E);
    else
      quant_rows<T, false>(a.quant, blockIdx.x - p.E, gridDim.x - p.E);
    return;
  }
  __shared__ double sums[4][kFewTokens];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = blockIdx.x;
  if (e == 0 && tid < kDoneLines) a.sync->done[tid].n = 0;
  const R* r = (const R*)p.r + e * p.re;
  double acc[kFewTokens] = {};
#pragma unroll 1
  for (int64_t k = 8 * tid; k < p.D; k += 2048) {
    float w[8], x[kFewTokens][8];
    load8(r, p.rd, k, p.D, p.wide, w);
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[t][i] = 0.0f;
      if (t < p.T) load8((const T*)p.x + t * p.sr, p.sc, k, p.D, p.wide, x[t]);
    }
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t)
      if (t < p.T) {
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[t] = __builtin_fma((double)x[t][i], (double)w[i], acc[t]);
      }
  }
#pragma unroll
  for (int t = 0; t < kFewTokens; ++t)
    if (t < p.T) {
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) acc[t] += __shfl_xor(acc[t], d);
      if (lane == 0) sums[wave][t] = acc[t];
    }
  __syncthreads();
  if (tid < p.T) p.logits[(int64_t)tid * p.E + e] = (float)(sums[0][tid] + sums[1][tid] + sums[2][tid] + sums[3][tid]);
}

// What the tokens chose: the distinct experts in order of their first slots, and each token's slot with each of them
// (-1: none) and its weight.
struct Choice {
  int ids[kFewSlots];
  float weights[kFewSlots];
  int count, expert[kFewSlots], taken, piece;
  int slot[kFewSlots][kFewTokens];
  float weight[kFewSlots][kFewTokens];
};

// By one wave, from ids and weights.
__device__ __forceinline__ void list_choice(Choice& c, int slots, int k, int E, int lane) {
  static_assert(kFewSlots * kFewTokens == 64, "a lane per entry");
  c.slot[0][lane] = -1;
  c.weight[0][lane] = 0.0f;
  if (lane < kFewSlots) c.expert[lane] = 0;
  wave_sync();
  const int e = lane < slots ? c.ids[lane] : -1;
  const bool is = e >= 0 && e < E;
  int first = lane;  // the lowest slot with this lane's expert
  for (int s = kFewSlots - 1; s >= 0; --s)
    if (__builtin_amdgcn_readlane(e, s) == e) first = s;
  const uint64_t mask = __builtin_amdgcn_ballot_w64(is && first == lane);
  const int d = __popcll(mask & ((1ull << first) - 1));
  if (is) {
    if (first == lane) c.expert[d] = e;
    c.slot[d][lane / k] = lane;  // (a token chooses an expert once)
    c.weight[d][lane / k] = c.weights[lane];
  }
  if (lane == 0) c.count = __popcll(mask);
}

struct LayerFew {
  static constexpr int W = 8;        // waves
  static constexpr int AHEAD = 6;    // pieces of the down weights that a wave has in flight
  static constexpr int GROUPS = 192; // blocks of hidden values that are held quantised at once
  static constexpr int GATE_UP = W * 2 * 64 * 16, DOWN = W * 64 * 16 + GROUPS * (kBlock + 4);
  static constexpr int SMEM = GATE_UP > DOWN ? GATE_UP : DOWN;

  __device__ static __forceinline__ i32x8 block_of(const uint8_t* w, int64_t k0, int64_t K, int g) {
    i32x4 lo, hi;
    if (k0 + kBlock <= K) {
      __builtin_memcpy(&lo, w + k0 + 16 * g, 16);
      __builtin_memcpy(&hi, w + k0 + 64 + 16 * g, 16);
    } else {
      lo = unit_of_row(w, k0 + 16 * g, K);
      hi = unit_of_row(w, k0 + 64 + 16 * g, K);
    }
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  // A lane's share of a block of D of a piece: gate's and up's rows and the token's values, and their scales.
  struct Block {
    i32x8 gate, up, x;
    float sg, su;
  };

  // 16 hidden columns of the d-th expert.
  __device__ static __forceinline__ void gate_up(const LayerArgs& a, const Choice& c, char* smem, int item, int tid) {
    const FewArgs& p = a.e;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), t16 = lane & 15, g = lane >> 4;
    const int d = item / a.pieces, e = c.expert[d], slot = t16 < kFewTokens ? c.slot[d][t16] : -1;
    f32x4(*sums)[2][64] = (f32x4(*)[2][64])smem;
    const int64_t n0 = (int64_t)(item - d * a.pieces) * 16, n = n0 + t16 < p.I ? n0 + t16 : p.I - 1;
    const uint8_t* w = p.w1 + e * p.w1e + n * p.ld1;
    const float* sw = p.s1 + e * p.s1e + n0 / kBlock * p.s1n;
    const int nk = (int)cdiv(p.D, kBlock), t = slot >= 0 ? t16 : 0;
    const uint8_t* xq = a.quant.q + t * a.quant.ldq + 16 * g;
    auto load = [&](Block& b, int kb) {
      const int64_t k0 = (int64_t)kb * kBlock;
      b.gate = block_of(w, k0, p.D, g);
      b.up = block_of(w + p.w1u, k0, p.D, g);
      const i32x4 lo = *(const i32x4*)(xq + k0), hi = *(const i32x4*)(xq + k0 + 64);
      b.x = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      const float s = a.quant.s[kb * a.quant.lds + t];
      b.sg = s * sw[kb * p.s1k];
      b.su = s * sw[p.s1u + kb * p.s1k];
    };
    f32x4 gate = {0.0f, 0.0f, 0.0f, 0.0f}, up = gate;
    Block b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (wave + i * W < nk) load(b[i], wave + i * W);
#pragma unroll 1
    for (int kb = wave; kb < nk; kb += 2 * W) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (kb + i * W < nk) {
          const Halves xh(b[i].x);
          gate += exact_product(b[i].gate, xh) * b[i].sg;
          __builtin_amdgcn_sched_barrier(0);  // (one operand's halves in registers at a time)
          up += exact_product(b[i].up, xh) * b[i].su;
          __builtin_amdgcn_sched_barrier(0);
          if (kb + (i + 2) * W < nk) load(b[i], kb + (i + 2) * W);
        }
    }
    sums[wave][0][lane] = gate;
    sums[wave][1][lane] = up;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 1; i < W; ++i) {
        gate += sums[i][0][lane];
        up += sums[i][1][lane];
      }
      if (slot >= 0) {
        // (stores of the agent's scope: past the XCD's own L2, where a release fence would write back all of it)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n0 + 4 * g + r < p.I)
            __hip_atomic_store(p.h + slot * p.ldh + n0 + 4 * g + r, silu_exact(gate[r]) * up[r], __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
      }
      wait_vm<0>();  // they are done before the count says so
      if (lane == 0)
        __hip_atomic_fetch_add(&a.sync->done[item % kDoneLines].n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }

  // A piece that nobody has claimed, claimed by this call, or -1.  By one wave.
  __device__ static __forceinline__ int unclaimed(const LayerArgs& a, int items, int lane) {
    constexpr int N = 8;  // loads in flight: each takes a microsecond
    for (int i0 = 0; i0 < items; i0 += 64 * N) {
      int taken[N];
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const int i = i0 + 64 * x + lane;
        taken[x] = 1;
        if (i < items) taken[x] = __hip_atomic_load(&a.claims[i].taken, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
#pragma unroll
      for (int x = 0; x < N; ++x)
        for (uint64_t open = __builtin_amdgcn_ballot_w64(taken[x] == 0); open; open &= open - 1) {
          const int at = i0 + 64 * x + __builtin_ctzll(open);
          int was = 1;
          if (lane == 0)
            was = __hip_atomic_exchange(&a.claims[at].taken, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (__builtin_amdgcn_readfirstlane(was) == 0) return at;
        }
    }
    return -1;
  }

  // The pieces of the down weights that a wave has in flight: unit u is block kb0 + u % nb of the (u / nb)-th expert.
  struct Ahead {
    i32x8 w[AHEAD];
    float s[AHEAD];
    __device__ __forceinline__ void load(const FewArgs& p, const Choice& c, int i, int u, int kb0, int nb, int64_t n0, int lane) {
      const int d = u / nb, kb = kb0 + u - d * nb;
      const int64_t e = c.expert[d], n = n0 + (lane & 15) < p.D ? n0 + (lane & 15) : p.D - 1;
      w[i] = block_of(p.w2 + e * p.w2e + n * p.ld2, (int64_t)kb * kBlock, p.I, lane >> 4);
      s[i] = p.s2[e * p.s2e + n0 / kBlock * p.s2n + kb * p.s2k];
    }
    __device__ __forceinline__ void load_all(const FewArgs& p, const Choice& c, int kb0, int nb, int64_t n0, int wave, int lane) {
      // (always all of them, the last unit again and again: an old value that stays would be held through what
      // comes before, a piece of gate and up perhaps)
      const int last = c.count * nb > 1 ? c.count * nb - 1 : 0;  // (without an expert the first one's)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) load(p, c, i, wave + i * W < last ? wave + i * W : last, kb0, nb, n0, lane);
    }
  };
  __device__ static __forceinline__ int blocks_at_once(const FewArgs& p) {
    const int nk = (int)cdiv(p.I, kBlock), most = GROUPS / p.slots;
    return nk < most ? nk : most;
  }

  // 16 columns of the result; `f` holds the first pieces.
  __device__ static __forceinline__ void down(const LayerArgs& a, const Choice& c, char* smem, Ahead& f, int64_t n0, int tid) {
    const FewArgs& p = a.e;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), t16 = lane & 15, g = lane >> 4;
    f32x4(*sums)[64] = (f32x4(*)[64])smem;
    uint8_t* hq = (uint8_t*)smem + W * 64 * 16;  // [group][128], a group: block of a slot
    float* hs = (float*)(hq + GROUPS * kBlock);
    const int nk = (int)cdiv(p.I, kBlock), count = c.count, most = blocks_at_once(p);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (wave == 0) {
      for (const int all = count * a.pieces;;) {
        int done = 0;
        if (lane < kDoneLines)
          done = __hip_atomic_load(&a.sync->done[lane].n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
        for (int x = kDoneLines / 2; x > 0; x >>= 1) done += __shfl_xor(done, x);
        if (__builtin_amdgcn_readfirstlane(done) >= all) break;
        __builtin_amdgcn_s_sleep(1);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // (the CU's L1, which the other waves share, and the L2)
    }
#pragma unroll 1
    for (int kb0 = 0; kb0 < nk; kb0 += most) {
      const int nb = nk - kb0 < most ? nk - kb0 : most, units = count * nb;
      if (kb0) f.load_all(p, c, kb0, nb, n0, wave, lane);
      __syncthreads();
      // the hidden values of these blocks, quantised, 16 lanes a block
      const int col = 8 * (lane & 15), groups = p.slots * nb;
      for (int i0 = tid >> 4; i0 < groups; i0 += 2 * 4 * W) {
        float v[2][8];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = i0 + x * 4 * W, slot = i / nb;
          const int64_t k = (int64_t)(kb0 + i - slot * nb) * kBlock + col;
          const bool in = i < groups && c.ids[slot] >= 0;
          const float* h = p.h + slot * p.ldh + k;
          if (in && k + 8 <= p.I) {
            load_vec(h, v[x]);
          } else {
#pragma unroll
            for (int r = 0; r < 8; ++r) v[x][r] = in && k + r < p.I ? h[r] : 0.0f;
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int i = i0 + x * 4 * W;
          uint32_t m = abs_bits(v[x][0]);
#pragma unroll
          for (int r = 1; r < 8; ++r) m = umax(m, abs_bits(v[x][r]));
          const BlockScale bs = block_scale(row_umax(m));
          if (i < groups) {
            i32x2 o;
            o[0] = pack_e4m3(v[x][0], v[x][1], v[x][2], v[x][3], bs.inv);
            o[1] = pack_e4m3(v[x][4], v[x][5], v[x][6], v[x][7], bs.inv);
            *(i32x2*)(hq + i * kBlock + col) = o;
            if (col == 0) hs[i] = bs.s;
          }
        }
      }
      __syncthreads();
#pragma unroll 1
      for (int u0 = wave; u0 < units; u0 += AHEAD * W) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          const int u = u0 + i * W;
          if (u >= units) break;
          const int d = u / nb, slot = t16 < kFewTokens ? c.slot[d][t16] : -1;
          const int at = slot >= 0 ? slot * nb + u - d * nb : 0;
          const uint8_t* q = hq + at * kBlock + 16 * g;
          const i32x4 lo = *(const i32x4*)q, hi = *(const i32x4*)(q + 64);
          const f32x4 part = mfma(f.w[i], __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
          if (slot >= 0) acc += part * (hs[at] * (f.s[i] * c.weight[d][t16]));
          if (u + AHEAD * W < units) f.load(p, c, i, u + AHEAD * W, kb0, nb, n0, lane);
        }
      }
      __syncthreads();
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || t16 >= p.T) return;
#pragma unroll
    for (int i = 1; i < W; ++i) acc += sums[i][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t col = n0 + 4 * g + r;
      if (col >= p.D) continue;
      const int64_t at = t16 * p.D + col;
      if (a.ytype == F16ACC_TYPE_F16)
        ((f16*)p.y)[at] = (f16)acc[r];
      else if (a.ytype == F16ACC_TYPE_BF16)
        ((bf16*)p.y)[at] = (bf16)acc[r];
      else
        ((float*)p.y)[at] = acc[r];
    }
  }
};

template <int V>
__global__ __launch_bounds__(64 * LayerFew::W, 4) void layer_few_kernel(LayerArgs a) {
  using L = LayerFew;
  __shared__ Choice c;
  __shared__ __align__(16) char smem[L::SMEM];  // (before its uses above: the rows of the routing)
  static_assert(kFewTokens * 64 * V * 4 <= L::SMEM, "the routing's rows");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hidden = a.e.slots * a.pieces, block = (int)blockIdx.x;
  if (tid == 0 && block < hidden)
    c.taken = __hip_atomic_exchange(&a.claims[block].taken, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (wave < a.e.T) {
    int id;
    float weight;
    route_token<float, V>(a.route, wave, lane, (float*)smem + wave * 64 * V, &id, &weight);
    if (lane < a.e.k) {
      c.ids[wave * a.e.k + lane] = id;
      c.weights[wave * a.e.k + lane] = weight;
    }
  }
  __syncthreads();
  if (wave == 0) list_choice(c, a.e.slots, a.e.k, a.e.E, lane);
  __syncthreads();
  const int items = c.count * a.pieces;
  if (block < hidden) {
    if (block < items && !c.taken) L::gate_up(a, c, smem, block, tid);
    return;
  }
  const int64_t n0 = (int64_t)(block - hidden) * 16;
  const int nb = L::blocks_at_once(a.e);
  L::Ahead f;
  f.load_all(a.e, c, 0, nb, n0, wave, lane);
  auto claim = [&] {
    if (wave == 0) {
      const int piece = L::unclaimed(a, items, lane);
      if (lane == 0) c.piece = piece;
    }
    __syncthreads();
    return c.piece;
  };
  int piece = claim();
  if (piece >= 0) {  // (what is in flight gives up its registers)
    do {
      L::gate_up(a, c, smem, piece, tid);
      __syncthreads();
      piece = claim();
    } while (piece >= 0);
    f.load_all(a.e, c, 0, nb, n0, wave, lane);
  }
  L::down(a, c, smem, f, n0, tid);
}

}  // namespace f16ops

// The products of at most 16 tokens: a decode step reads every weight byte once,
// and that is the whole cost, so nothing is staged.  A workgroup takes 16 weight
// rows; its waves deal the blocks of K among themselves and read the rows straight into
// the MFMA's registers (64 contiguous bytes a row and instruction, two of them a
// 128-byte line), one block ahead.  The tokens are quantised on the way, by each wave for the
// blocks it multiplies, so there is one launch and no quantised copy.  The waves'
// sums meet in LDS, in wave order.
//
// Measured (kernel time, weights cold): one token through 8960 x 1536 in 6.0 us, of
// which the weight's 13.8 MB are 2.8 at the copy rate and the rest the latency of a
// launch and of one load after another; through 8192 x 8192 in 16.9 us, 4.0 TB/s.
#pragma once

#include "common.h"
#include "mm.h"

namespace f16ops {

// A wave's block of 128 columns of up to 16 token rows, quantised on the way:
// 16 lanes take a token, 8 values each, four tokens at a time (a lane that
// quantised its own 32 operand values would spend as much on 15 absent tokens as
// on one), and the values pass through LDS into the MFMA's layout.
struct TokenBlock {
  static constexpr int ROW = kBlock + 16;  // bytes: rows on different banks
  uint8_t q[16 * ROW];
  float s[16];
};

// Rows row(t) of x (NULL: zeros) from k0, for t < tokens <= 4 G (row is asked for every
// t < 4 G); every group's loads are in flight together.
template <class T, int G, class Row>
__device__ __forceinline__ i32x8 quant_tokens(TokenBlock& b, Row row, int tokens, int64_t k0, int64_t K, int lane,
                                              float* s) {
  const int c = lane & 15;
  const int64_t k = k0 + 8 * c;
  float v[G][8];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int t = 4 * i + (lane >> 4);
    const T* x = row(t);  // (by every lane: it may exchange between lanes)
    if (t >= tokens) x = nullptr;
    if (x && k + 8 <= K) {
      load_vec(x + k, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = x && k + j < K ? (float)x[k + j] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int t = 4 * i + (lane >> 4);
    uint32_t m = abs_bits(v[i][0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) m = umax(m, abs_bits(v[i][j]));
    const BlockScale bs = block_scale(row_umax(m));
    i32x2 o;
    o[0] = pack_e4m3(v[i][0], v[i][1], v[i][2], v[i][3], bs.inv);
    o[1] = pack_e4m3(v[i][4], v[i][5], v[i][6], v[i][7], bs.inv);
    *(i32x2*)(b.q + t * TokenBlock::ROW + 8 * c) = o;
    if (c == 0) b.s[t] = bs.s;
  }
  wave_sync();
  const int t16 = lane & 15, g = lane >> 4;
  *s = b.s[t16];
  const uint8_t* q = b.q + t16 * TokenBlock::ROW + 16 * g;
  const i32x4 lo = *(const i32x4*)q, hi = *(const i32x4*)(q + 64);
  wave_sync();
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's share of block kb of a weight row, at any address (a 16-byte load goes
// from any, and costs the same from an aligned one).
__device__ __forceinline__ i32x4 load_unit(const uint8_t* w, int64_t k, int64_t K) {
  union {
    uint8_t b[16];
    i32x4 v;
  } u;
  u.v = i32x4{0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(u.b, w + k, 16);
  } else {
#pragma unroll 1
    for (int i = 0; k + i < K; ++i) {
      const int byte = w[k + i] << (8 * (i & 3));
      u.v[0] |= i < 4 ? byte : 0;
      u.v[1] |= i >= 4 && i < 8 ? byte : 0;
      u.v[2] |= i >= 8 && i < 12 ? byte : 0;
      u.v[3] |= i >= 12 ? byte : 0;
    }
  }
  return u.v;
}
__device__ __forceinline__ i32x8 load_weight(const uint8_t* w, int64_t k0, int64_t K, int g) {
  const i32x4 lo = load_unit(w, k0 + 16 * g, K), hi = load_unit(w, k0 + 64 + 16 * g, K);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

struct SmallArgs {
  const void* x;  // [M][ldx] elements
  int64_t ldx;
  const uint8_t* w;
  int64_t ldw;
  const float* sw;
  int64_t swn, swk;
  const void* bias;
  void* c;
  int64_t scm, scn;
  int64_t M, N, K;
};

template <class T, int W, int G>
__global__ __launch_bounds__(64 * W) void linear_small_kernel(SmallArgs p) {
  __shared__ f32x4 sums[W][64];
  __shared__ __align__(16) TokenBlock tokens[W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + t16 < p.N ? n0 + t16 : p.N - 1;
  const uint8_t* w = p.w + n * p.ldw;
  const float* sw = p.sw + n0 / kBlock * p.swn;
  const bool in = t16 < p.M;
  const int nk = (int)cdiv(p.K, kBlock);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  i32x8 next;
  if (wave < nk) next = load_weight(w, (int64_t)wave * kBlock, p.K, g);
#pragma unroll 1
  for (int kb = wave; kb < nk; kb += W) {
    const i32x8 wf = next;
    if (kb + W < nk) next = load_weight(w, (int64_t)(kb + W) * kBlock, p.K, g);
    const float sb = sw[kb * p.swk];
    float s;
    const i32x8 xf = quant_tokens<T, G>(tokens[wave], [&](int t) { return (const T*)p.x + t * p.ldx; }, (int)p.M,
                                     (int64_t)kb * kBlock, p.K, lane, &s);
    acc += mfma(wf, xf) * (s * sb);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 1; i < W; ++i) acc += sums[i][lane];
  const int64_t row = n0 + 4 * g;
  const int left = (int)(p.N - row < 4 ? p.N - row : 4);
  if (!in || left <= 0) return;
  if (p.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) acc[r] += (float)((const T*)p.bias)[row + r];
  }
  const bool wide = p.scn == 1 && p.scm % 4 == 0 && (uintptr_t)p.c % (4 * sizeof(T)) == 0;
  store4<T>((T*)p.c + (int64_t)t16 * p.scm + row * p.scn, p.scn, left, acc, wide);
}

// ---------------------------------------------------------------------------
// The experts' feed-forward for at most 4 tokens: no sorting.  Token t is column
// t of every expert's products, zero where the token does not go there, so the
// down kernel adds all experts of a token in one register, and the routing weight
// is a factor of the block's scale.
//
// The hidden values are quantised between the products, so the first product's sums
// are exact (binary16 operands, FP32 sums): what the 8-bit matrix instructions drop
// showed as 2e-3 of one token's result, and weights are what the kernels wait for.
//
// Measured: one token through 6 of 64 experts, 2048 x 1024, 38 MB of weights: 11.4 + 7.2
// us against 7.6 at the copy rate.  What is left is latency: a launch, the ids, the
// weights, one wait after another, on two launches.
// ---------------------------------------------------------------------------

__device__ __forceinline__ f32x4 exact_product(const i32x8& w, const Halves& x) {
  const Halves h(w);
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = mfma_f16(h.v[i], x.v[i], sum);
  return sum;
}

// At most 4 tokens and 16 slots.  Here and on the tiles, in us (bfloat16, in a graph; 8 tokens
// here with two groups of four):
//   64 experts of 2048 x 1024, 8 a token: 1 token 20 / 38, 2 32 / 40, 4 55 / 48, 8 100 / 72
//   16 of 4096 x 2048, 2 a token:         1 token 20 / 49, 4 39 / 55, 8 65 / 59
//   128 of 1024 x 512, 4 a token:         1 token 10 / 26, 4 15 / 26, 8 30 / 30
constexpr int kFewTokens = 4, kFewSlots = 16;

// What the down kernel reads of the routing: the distinct experts in order of their
// first slots, and each token's first slot with each of them (-1: none) and its weight.
struct FewMap {
  int count, expert[kFewSlots];
  int slot[kFewSlots][kFewTokens];
  float weight[kFewSlots][kFewTokens];
};

struct FewArgs {
  const void* x;
  int64_t ldx;
  int T, k, E, slots;
  const int* ids;
  const float* weights;
  int64_t wt, wk;
  int64_t D, I;
  const uint8_t* w1;
  int64_t w1e, w1u, ld1;
  const float* s1;
  int64_t s1e, s1u, s1n, s1k;
  const uint8_t* w2;
  int64_t w2e, ld2;
  const float* s2;
  int64_t s2e, s2n, s2k;
  float* h;  // [slots][ldh], at each (token, expert)'s first slot
  int64_t ldh;
  FewMap* map;
  void* y;
};

// Fills p.map, by one workgroup while the others multiply.
template <int THREADS>
__device__ __forceinline__ void few_map(const FewArgs& p) {
  __shared__ int ids[kFewSlots], index[kMaxExperts];
  __shared__ float weights[kFewSlots];
  static_assert(kFewSlots <= 64, "the first wave has a lane per slot");  // (and reads index before it writes it)
  const int tid = threadIdx.x, lane = tid & 63;
  // index[e]: the lowest slot with expert e, then the expert's place
  for (int i = tid; i < p.E; i += THREADS) index[i] = kFewSlots;
  int e = -1;
  if (tid < p.slots) {
    e = p.ids[tid];
    weights[tid] = p.weights[tid / p.k * p.wt + tid % p.k * p.wk];
    if (e >= p.E) e = -1;
    ids[tid] = e;
  }
  __syncthreads();
  if (e >= 0) atomicMin(&index[e], tid);
  __syncthreads();
  const bool first = e >= 0 && index[e] == tid;
  const uint64_t mask = __builtin_amdgcn_ballot_w64(first);
  if (first) {
    const int at = __popcll(mask & ((1ull << lane) - 1));
    p.map->expert[at] = e;
    index[e] = at;
  }
  if (tid == 0) p.map->count = __popcll(mask);
  if (tid < kFewSlots * kFewTokens) p.map->slot[0][tid] = -1;
  static_assert(THREADS >= kFewSlots * kFewTokens, "a thread per entry");
  __syncthreads();
  if (e < 0) return;
  // (a token may name an expert twice: its first slot has both weights)
  const int t = tid / p.k;
  float sum = weights[tid];
  for (int j = t * p.k; j < tid; ++j)
    if (ids[j] == e) return;
  for (int j = tid + 1; j < (t + 1) * p.k; ++j)
    if (ids[j] == e) sum += weights[j];
  p.map->slot[index[e]][t] = tid;
  p.map->weight[index[e]][t] = sum;
}

// h of 32 hidden columns of one expert, the one of slot blockIdx.y where that is its
// first.  The waves deal the blocks of D, the next one's weights in flight while one
// is multiplied.  All ids lie in the wave's registers: what the expert's tokens are
// is a ballot and no further load.
template <class T, int W, int G>
__global__ __launch_bounds__(64 * W) void few_gate_up_kernel(FewArgs p) {
  __shared__ f32x4 sums[W][4][64];
  __shared__ __align__(16) TokenBlock tokens[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t16 = lane & 15, g = lane >> 4, slot0 = blockIdx.y;
  if (slot0 == p.slots) {  // (the last row of workgroups)
    if (blockIdx.x == 0) few_map<64 * W>(p);
    return;
  }
  const int e = p.ids[slot0];
  const int id = lane < p.slots ? p.ids[lane] : -1;
  const uint64_t same = __builtin_amdgcn_ballot_w64(id == e);
  const bool earlier = (same & ((1ull << slot0) - 1)) != 0;
  if (e < 0 || e >= p.E || earlier) return;  // (the same in every wave)
  int slot = -1;  // the token's first slot with this expert
  if (t16 < p.T) {
    const int at = t16 * p.k;
    const uint64_t bits = (same >> at) & ((1ull << p.k) - 1);
    if (bits) slot = at + __builtin_ctzll(bits);
  }
  const int64_t n0 = (int64_t)blockIdx.x * 32;
  const int64_t na = n0 + t16 < p.I ? n0 + t16 : p.I - 1, nb = n0 + 16 + t16 < p.I ? n0 + 16 + t16 : p.I - 1;
  const uint8_t* w = p.w1 + e * p.w1e;
  const uint8_t *wa = w + na * p.ld1, *wb = w + nb * p.ld1;
  const float* sw = p.s1 + e * p.s1e + n0 / kBlock * p.s1n;
  const int nk = (int)cdiv(p.D, kBlock);
  f32x4 acc[4] = {};  // gate, gate, up, up
  const uint32_t here = (uint32_t)__builtin_amdgcn_ballot_w64(slot >= 0);  // bit t: token t goes there
  i32x8 next[4];
  auto load = [&](int kb) {
    const int64_t k0 = (int64_t)kb * kBlock;
    next[0] = load_weight(wa, k0, p.D, g);
    next[1] = load_weight(wb, k0, p.D, g);
    next[2] = load_weight(wa + p.w1u, k0, p.D, g);
    next[3] = load_weight(wb + p.w1u, k0, p.D, g);
  };
  if (wave < nk) load(wave);
#pragma unroll 1
  for (int kb = wave; kb < nk; kb += W) {
    const float sg = sw[kb * p.s1k], su = sw[p.s1u + kb * p.s1k];
    const i32x8 wf[4] = {next[0], next[1], next[2], next[3]};
    if (kb + W < nk) load(kb + W);
    float s;
    const Halves xh(quant_tokens<T, G>(
        tokens[wave], [&](int t) { return (here >> t) & 1 ? (const T*)p.x + t * p.ldx : nullptr; }, p.T,
        (int64_t)kb * kBlock, p.D, lane, &s));
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += exact_product(wf[i], xh) * (s * (i < 2 ? sg : su));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= 2 || slot < 0) return;  // wave 0: columns 0 .. 15, wave 1: 16 .. 31
  f32x4 gate = sums[0][wave][lane], up = sums[0][2 + wave][lane];
#pragma unroll
  for (int i = 1; i < W; ++i) {
    gate += sums[i][wave][lane];
    up += sums[i][2 + wave][lane];
  }
  const int64_t n = n0 + 16 * wave + 4 * g;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < p.I) p.h[slot * p.ldh + n + r] = silu_exact(gate[r]) * up[r];
}

// y of 16 columns: the waves deal the (expert, block of I) pairs, the next one's
// weights in flight while one is multiplied.
template <class T, int W, int G>
__global__ __launch_bounds__(64 * W) void few_down_kernel(FewArgs p) {
  __shared__ f32x4 sums[W][64];
  __shared__ __align__(16) TokenBlock tokens[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t16 = lane & 15, g = lane >> 4, t = t16 < kFewTokens ? t16 : kFewTokens - 1;
  const FewMap* map = p.map;
  const int64_t n0 = (int64_t)blockIdx.x * 16, n = n0 + t16 < p.D ? n0 + t16 : p.D - 1;
  const int nk = (int)cdiv(p.I, kBlock), units = map->count * nk;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  i32x8 next;
  float snext = 0.0f, wnext = 0.0f;
  int slots = -1, d = wave / nk, kb = wave - d * nk;  // slots: lane l holds token l's slot with the expert
  auto load = [&]() {
    const int64_t e = map->expert[d];
    next = load_weight(p.w2 + e * p.w2e + n * p.ld2, (int64_t)kb * kBlock, p.I, g);
    snext = p.s2[e * p.s2e + n0 / kBlock * p.s2n + kb * p.s2k];
    slots = map->slot[d][t];
    wnext = map->weight[d][t];
  };
  if (wave < units) load();
#pragma unroll 1
  for (int u = wave; u < units; u += W) {
    const i32x8 wf = next;
    const int here = t16 < p.T ? slots : -1, at = kb;
    const float f = here >= 0 ? snext * wnext : 0.0f;
    kb += W;
    while (kb >= nk) kb -= nk, ++d;
    if (u + W < units) load();
    float s;
    const i32x8 xf = quant_tokens<float, G>(
        tokens[wave],
        [&](int i) {
          const int slot = __shfl(here, i);
          return slot >= 0 ? p.h + slot * p.ldh : nullptr;
        },
        p.T, (int64_t)at * kBlock, p.I, lane, &s);
    const f32x4 part = mfma(wf, xf);
    if (here >= 0) acc += part * (s * f);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || t16 >= p.T) return;
#pragma unroll
  for (int i = 1; i < W; ++i) acc += sums[i][lane];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n0 + 4 * g + r < p.D) ((T*)p.y)[t16 * p.D + n0 + 4 * g + r] = (T)acc[r];
}

}  // namespace f16ops

// The products of at most 16 tokens: a decode step reads every weight byte
// once, and that is the whole cost, so nothing is staged.  A workgroup takes 16
// weight rows; its waves deal the blocks of K among themselves and read the
// rows straight into the MFMA's registers (64 contiguous bytes a row and
// instruction, two of them a 128-byte line).  The tokens are quantised on the way, by
// each wave for the blocks it multiplies: a lane's 32 values lie in its
// registers as the MFMA wants them, and a block's maximum is over four lanes.
// So there is one launch and no quantised copy.  The waves' sums meet in LDS,
// in wave order.
#pragma once

#include "common.h"
#include "mm.h"

namespace f16ops {

// A lane's share of block kb of a token row: k of units g and g + 4.
template <class T>
__device__ __forceinline__ void load_token(const T* x, int64_t k0, int64_t K, int g, bool in, float (&v)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t k = k0 + 64 * h + 16 * g;
    float t[16];
    if (in && k + 16 <= K) {
      load_vec(x + k, t);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) t[i] = in && k + i < K ? (float)x[k + i] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[16 * h + i] = t[i];
  }
}

// The lane's share quantised, and its block's scale.
__device__ __forceinline__ i32x8 quant_token(const float (&v)[32], float* s) {
  uint32_t m = abs_bits(v[0]);
#pragma unroll
  for (int i = 1; i < 32; ++i) m = umax(m, abs_bits(v[i]));
  m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
  m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
  const BlockScale bs = block_scale(m);
  *s = bs.s;
  i32x8 q;
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = pack_e4m3(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], bs.inv);
  return q;
}

// A lane's share of block kb of a weight row (zero from K to the next multiple
// of 16).
__device__ __forceinline__ i32x8 load_weight(const uint8_t* w, int64_t k0, int64_t K, int g) {
  i32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (k0 + 16 * g < K) lo = *(const i32x4*)(w + k0 + 16 * g);
  if (k0 + 64 + 16 * g < K) hi = *(const i32x4*)(w + k0 + 64 + 16 * g);
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

template <class T, int W>
__global__ __launch_bounds__(64 * W) void linear_small_kernel(SmallArgs p) {
  __shared__ f32x4 sums[W][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t16 = lane & 15, g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + t16 < p.N ? n0 + t16 : p.N - 1;
  const uint8_t* w = p.w + n * p.ldw;
  const float* sw = p.sw + n0 / kBlock * p.swn;
  const T* x = (const T*)p.x + (int64_t)t16 * p.ldx;
  const bool in = t16 < p.M;
  const int nk = (int)cdiv(p.K, kBlock);
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = wave; kb < nk; kb += W) {
    const i32x8 wf = load_weight(w, (int64_t)kb * kBlock, p.K, g);
    float v[32], s;
    load_token(x, (int64_t)kb * kBlock, p.K, g, in, v);
    const float sb = sw[kb * p.swk];
    const f32x4 part = mfma(wf, quant_token(v, &s));
    acc += part * (s * sb);
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

}  // namespace f16ops

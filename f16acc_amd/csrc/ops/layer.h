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
  if (wide && k + 8 <= D) {
    load_vec(p + k, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < D ? (float)p[(k + i) * stride] : 0.0f;
  }
}

// logits[t][e] = sum over d of x[t][d] r[e][d], summed in 64 bits and rounded once to FP32: products of 16-bit and
// FP32 values are exact there, so a token's logits, and with them the choice of its experts, do not depend
// on the batch it comes in.  16 tokens by 16 experts a workgroup on v_mfma_f64_16x16x4_f64; the waves deal the
// chunks of 32 columns, a lane loads eight of a row, and their sums meet in LDS in wave order.
template <class T, class R, int W>
__global__ __launch_bounds__(64 * W) void router_kernel(RouterArgs p) {
  __shared__ f64x4 sums[W][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g = lane >> 4;
  const int64_t t0 = (int64_t)blockIdx.x * 16;
  const int e0 = (int)blockIdx.y * 16;
  const int64_t t = t0 + l16 < p.T ? t0 + l16 : p.T - 1;
  const int e = e0 + l16 < p.E ? e0 + l16 : p.E - 1;
  const T* x = (const T*)p.x + t * p.sr;
  const R* r = (const R*)p.r + e * p.re;
  f64x4 acc = {0.0, 0.0, 0.0, 0.0};
  float a[8], b[8];
  const int64_t step = 32 * W;
  int64_t k = 32 * wave + 8 * g;
  load8(x, p.sc, k, p.D, p.wide, a);
  load8(r, p.rd, k, p.D, p.wide, b);
  for (int64_t c = 32 * wave; c < p.D; c += step) {
    float ca[8], cb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) ca[i] = a[i], cb[i] = b[i];
    k += step;
    load8(x, p.sc, k, p.D, p.wide, a);
    load8(r, p.rd, k, p.D, p.wide, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)cb[i], (double)ca[i], acc, 0, 0, 0);
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0 || t0 + l16 >= p.T) return;
#pragma unroll
  for (int i = 1; i < W; ++i) acc += sums[i][lane];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = e0 + g + 4 * i;
    if (row < p.E) p.logits[(t0 + l16) * p.E + row] = (float)acc[i];
  }
}

}  // namespace f16ops

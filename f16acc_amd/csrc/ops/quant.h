// Quantisation to e4m3 in blocks of 128: rows (1 x 128), columns (128 x 1, the
// result transposed), and squares (128 x 128), and the copy that gives stored
// 8-bit rows the alignment the products read.
#pragma once

#include "common.h"

namespace f16ops {

struct QuantArgs {
  const void* x;
  int64_t rows, cols, sr, sc;  // element strides
  uint8_t* q;                  // [rows][ldq], zero from cols to ldq
  int64_t ldq;
  float* s;  // scale of (row, block) at s[block * lds + row]; squares: s[rowblock * lds + block]
  int64_t lds;
  uint8_t* qt;  // [cols][ldqt], zero from rows to ldqt
  int64_t ldqt;
  float* st;  // scale of (column, rowblock) at st[rowblock * ldst + column]
  int64_t ldst;
};

// One row of a matrix in blocks of 1 x 128.  16 lanes take a block, 8 elements
// each: a wave reads four blocks with one 16-byte load a lane (16-bit types),
// finds each block's maximum with four row rotations and writes 8 bytes a
// lane.  Bound by memory, 2 bytes read and 1 written an element: 8192 x 8192
// bfloat16 in 41.6 us, 4.8 TB/s.
template <class T, bool WIDE>
__device__ __forceinline__ void quant_rows(const QuantArgs& p, uint32_t group, uint32_t groups) {
  const int64_t blocks = p.ldq / kBlock;
  const int64_t total = p.rows * blocks;
  const int lane = threadIdx.x & 15;
  for (int64_t b = (int64_t)group * 16 + (threadIdx.x >> 4); b < total; b += (int64_t)groups * 16) {
    // (64-bit division is a hundred instructions)
    const int64_t row = total >> 32 ? b / blocks : (int64_t)((uint32_t)b / (uint32_t)blocks), kb = b - row * blocks;
    const int64_t c0 = kb * kBlock + lane * 8;
    const T* x = (const T*)p.x + row * p.sr;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (WIDE && c0 + 8 <= p.cols) {
      load_vec(x + c0, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c0 + i < p.cols) v[i] = (float)x[(c0 + i) * p.sc];
    }
    uint32_t m = abs_bits(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = umax(m, abs_bits(v[i]));
    const BlockScale bs = block_scale(row_umax(m));
    i32x2 o;
    o[0] = pack_e4m3(v[0], v[1], v[2], v[3], bs.inv);
    o[1] = pack_e4m3(v[4], v[5], v[6], v[7], bs.inv);
    *(i32x2*)(p.q + row * p.ldq + c0) = o;
    if (lane == 0 && c0 < p.cols) p.s[kb * p.lds + row] = bs.s;  // (what pads a row has no scale)
  }
}
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs p) {
  quant_rows<T, WIDE>(p, blockIdx.x, gridDim.x);
}

// A 128 x 128 tile a workgroup: read once, quantised along its rows (ROWS), its
// columns (COLS, written transposed through LDS) or both, or as one square
// block (SQUARE, whose transpose has the same values and scales).
// Thread (r, c) holds rows 4 r .. 4 r + 3, columns 8 c .. 8 c + 7: a row's
// maximum is over the 16 lanes of a DPP row, a column's over the four DPP rows
// of a wave and then the eight waves.  4096 x 8960 in both directions: 36 us, 4.1 TB/s.
template <class T, bool WIDE, bool ROWS, bool COLS, bool SQUARE>
__global__ __launch_bounds__(512) void quant_tile_kernel(QuantArgs p) {
  // The transposed tile: 16-byte unit u of column col lies at u ^ (col / 8 % 8), so the
  // 64 four-byte writes of a wave (16 columns apart by 8, four row groups) fall on 32 banks.
  __shared__ __align__(16) uint8_t tile[COLS ? kBlock * kBlock : 16];
  __shared__ __align__(16) uint32_t part[SQUARE ? 32 : 8 * kBlock];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = tid >> 4, c = tid & 15;
  const int64_t kb = blockIdx.x, rb = blockIdx.y;
  const int64_t r0 = rb * kBlock + r * 4, c0 = kb * kBlock + c * 8;
  float v[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T* x = (const T*)p.x + (r0 + i) * p.sr;
    if (WIDE && r0 + i < p.rows && c0 + 8 <= p.cols) {
      load_vec(x + c0, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = r0 + i < p.rows && c0 + j < p.cols ? (float)x[(c0 + j) * p.sc] : 0.0f;
    }
  }
  auto store_rows = [&](int i, float inv) {
    i32x2 o;
    o[0] = pack_e4m3(v[i][0], v[i][1], v[i][2], v[i][3], inv);
    o[1] = pack_e4m3(v[i][4], v[i][5], v[i][6], v[i][7], inv);
    if (r0 + i < p.rows) *(i32x2*)(p.q + (r0 + i) * p.ldq + c0) = o;
  };
  auto stage_column = [&](int j, float inv) {
    *(int*)(tile + (c * 8 + j) * kBlock + (r ^ 4 * (c & 7)) * 4) = pack_e4m3(v[0][j], v[1][j], v[2][j], v[3][j], inv);
  };
  if (SQUARE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = umax(m, abs_bits(v[i][j]));
    m = row_umax(m);
    if (c == 0) part[r] = m;
    __syncthreads();
    const BlockScale bs = block_scale(umax(row_umax(part[c]), row_umax(part[16 + c])));
    if (tid == 0) p.s[rb * p.lds + kb] = bs.s;
#pragma unroll
    for (int i = 0; i < 4; ++i) store_rows(i, bs.inv);
    if (COLS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) stage_column(j, bs.inv);
    }
  } else {
    if (COLS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t m = umax(umax(abs_bits(v[0][j]), abs_bits(v[1][j])), umax(abs_bits(v[2][j]), abs_bits(v[3][j])));
        m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
        m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
        if (lane < 16) part[wave * kBlock + c * 8 + j] = m;
      }
    }
    if (ROWS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t m = abs_bits(v[i][0]);
#pragma unroll
        for (int j = 1; j < 8; ++j) m = umax(m, abs_bits(v[i][j]));
        const BlockScale bs = block_scale(row_umax(m));
        store_rows(i, bs.inv);
        if (c == 0 && r0 + i < p.rows) p.s[kb * p.lds + r0 + i] = bs.s;
      }
    }
    if (COLS) {
      __syncthreads();
      if (tid < kBlock) {  // a thread per column
        uint32_t m = part[tid];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = umax(m, part[i * kBlock + tid]);
        const BlockScale bs = block_scale(m);
        part[tid] = __float_as_uint(bs.inv);
        if (kb * kBlock + tid < p.cols) p.st[rb * p.ldst + kb * kBlock + tid] = bs.s;
      }
      __syncthreads();
      float inv[8];
      load_vec((const float*)part + c * 8, inv);
#pragma unroll
      for (int j = 0; j < 8; ++j) stage_column(j, inv[j]);
    }
  }
  if (COLS) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int col = k * 64 + (tid >> 3), u = tid & 7;
      if (kb * kBlock + col < p.cols)
        *(i32x4*)(p.qt + (kb * kBlock + col) * p.ldqt + rb * kBlock + u * 16) = 
            *(const i32x4*)(tile + col * kBlock + (u ^ (col >> 3 & 7)) * 16);
    }
  }
}

// dst[r][c] = src[r * s_r + c * s_c] for c < cols, zero up to ld (a multiple of
// 16): 8-bit rows of any strides laid out as the products read them.
struct Pack8Args {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, cols, s_r, s_c, ld;
};
__device__ __forceinline__ void pack8(const Pack8Args& p, uint32_t group, uint32_t groups) {
  const int64_t units = p.ld / 16, total = p.rows * units;
  for (int64_t i = (int64_t)group * 256 + threadIdx.x; i < total; i += (int64_t)groups * 256) {
    const int64_t r = total >> 32 ? i / units : (int64_t)((uint32_t)i / (uint32_t)units), c = (i - r * units) * 16;
    const uint8_t* s = p.src + r * p.s_r;
    union {
      uint8_t b[16];
      i32x4 v;
    } o;
    if (p.s_c == 1 && c + 16 <= p.cols) {
      __builtin_memcpy(o.b, s + c, 16);  // one 16-byte load: any alignment goes
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) o.b[k] = c + k < p.cols ? s[(c + k) * p.s_c] : 0;
    }
    *(i32x4*)(p.dst + r * p.ld + c) = o.v;
  }
}
__global__ __launch_bounds__(256) void pack8_kernel(Pack8Args p) { pack8(p, blockIdx.x, gridDim.x); }

// Both at once, for a product of new tokens with a weight whose rows are not aligned: the
// first `packs` workgroups copy.
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void quant_pack_kernel(QuantArgs q, Pack8Args p, uint32_t packs) {
  if (blockIdx.x < packs)
    pack8(p, blockIdx.x, packs);
  else
    quant_rows<T, WIDE>(q, blockIdx.x - packs, gridDim.x - packs);
}

}  // namespace f16ops

// Microscaled 4-bit operands: blocks of 32 e2m1 values with a power of two each (e8m0), two
// values a byte, the first in its low half.  Quantisation along the rows, along the
// columns (transposed) or both, the values back, the scales in the products' order.
//
//   m = max(|x|, 2^-100)   s = 2^e with 2^e <= m / 3.5 < 2^(e + 1)   q = e2m1(x / s), nearest, ties to even
//
// |x / s| stays below 7, the middle of 6 and the next power of two, so no value is cut off by
// more than its rounding.  A block that holds an infinity or a NaN has the scale NaN (255).
#pragma once

#include "common.h"
#include "quant.h"

namespace f16ops {

constexpr int kMx = 32;    // values of a block
constexpr int kQuad = 128; // values of four blocks, whose scales are one dword

// The e8m0 byte of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t mx_exponent(uint32_t bits) { return ((umax(bits, kTinyBits) + 0x200000u) >> 23) - 2; }
__device__ __forceinline__ uint32_t mx_byte(uint32_t bits) { return bits >= kInfBits ? 255u : mx_exponent(bits); }

// Eight consecutive values of a row as they are held, and what quantising takes of them: the bits of the largest
// magnitude (as FP32's, so NaN > infinity > finite) and the e2m1 values.  16-bit types stay in pairs: their
// magnitudes compare as integers, two at a time, and the conversion takes pairs.
template <class T>
struct Eight {
  static constexpr bool PAIRS = sizeof(T) == 2;
  static constexpr int N = PAIRS ? 4 : 8;
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef T Pair __attribute__((ext_vector_type(2)));
  uint32_t d[N];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) d[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(d, p, sizeof(d)); }  // (from any address)
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols, int64_t stride) {  // zero past cols
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = row[(c + i < cols ? c + i : cols - 1) * stride];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = c + i < cols ? t[i] : (T)0.0f;
    __builtin_memcpy(d, t, sizeof(d));
  }
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) {  // of magnitudes, element by element
    if constexpr (PAIRS)
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
    else
      return umax(a, b);
  }
  __device__ __forceinline__ static uint32_t magnitude(uint32_t v) { return v & (PAIRS ? 0x7fff7fffu : 0x7fffffffu); }
  // FP32's bits of a magnitude: of a 16-bit one in the low half.
  __device__ __forceinline__ static uint32_t bits(uint32_t m) {
    if constexpr (!PAIRS)
      return m;
    else if constexpr (std::is_same_v<T, bf16>)
      return m << 16;
    else
      return __float_as_uint((float)__builtin_bit_cast(f16, (uint16_t)m));
  }
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = magnitude(d[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = larger(m, magnitude(d[i]));
    if constexpr (PAIRS) m = umax(m >> 16, m & 0xffffu);
    return bits(m);
  }
  __device__ __forceinline__ uint32_t packed(uint32_t e) const {
    const float s = __uint_as_float(e << 23);  // (the conversion divides by it)
    uint32_t r = 0;
    if constexpr (!PAIRS) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(d[0]), __uint_as_float(d[1]), s, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(d[2]), __uint_as_float(d[3]), s, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(d[4]), __uint_as_float(d[5]), s, 2);
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(d[6]), __uint_as_float(d[7]), s, 3);
    } else if constexpr (std::is_same_v<T, bf16>) {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(Pair, d[0]), s, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(Pair, d[1]), s, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(Pair, d[2]), s, 2);
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(Pair, d[3]), s, 3);
    } else {
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(Pair, d[0]), s, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(Pair, d[1]), s, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(Pair, d[2]), s, 2);
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(Pair, d[3]), s, 3);
    }
  }
  // Column j of eight rows.
  __device__ __forceinline__ static Eight column(const Eight (&v)[8], int j) {
    Eight c;
    if constexpr (PAIRS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = v[2 * i].d[j / 2], b = v[2 * i + 1].d[j / 2];
        c.d[i] = j % 2 ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) c.d[i] = v[i].d[j];
    }
    return c;
  }
};

// Eight e2m1 values times 2^(e - 127); NaN where e is 255.
__device__ __forceinline__ void unpack_e2m1(uint32_t q, uint32_t e, float (&v)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
  const float t[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = e == 255u ? __uint_as_float(0x7fc00000u) : __builtin_ldexpf(t[i], (int)e - 127);
}

// Scale bytes: that of (row, block b) at s[row * row_stride + b / 4 * quad_stride + b % 4], both strides
// multiples of 4.  [rows][quads] has (4 quads, 4), [quads][rows] (4, 4 rows).
struct MxScales {
  uint8_t* s;
  int64_t row, quad;
};

struct MxQuantArgs {
  const void* x;
  int64_t rows, cols, sr, sc;  // element strides
  uint8_t* q;                  // [rows][ldq], zero from cols on; ldq: 64 for each 128 columns
  int64_t ldq;
  MxScales s;
  uint8_t* qt;  // [cols][ldqt], zero from rows on; ldqt: 64 for each 128 rows
  int64_t ldqt;
  MxScales st;
  // x held in 4 bits itself: bytes [rows][..], scale of (row, block) at xs + row * xsr + block * xsc
  const uint8_t* xs;
  int64_t xsr, xsc;
};

__device__ __forceinline__ uint32_t quad_umax(uint32_t v) {
  v = umax(v, dpp<0xb1>(v));  // quad_perm:[1,0,3,2], [2,3,0,1]
  return umax(v, dpp<0x4e>(v));
}

// The four bytes of a quad of blocks, held by 16 lanes, four alike for each block, as one dword.
__device__ __forceinline__ uint32_t quad_bytes(uint32_t byte, int lane) {
  uint32_t v = byte << (8 * (lane >> 2 & 3));
  v |= dpp<0x124>(v);  // row_ror:4, 8
  return v | dpp<0x128>(v);
}

// Rows of a matrix in blocks of 1 x 32.  16 lanes take 128 values of a row, 8 each: a 16-byte load a lane (16-bit
// types), the maximum of four lanes by two exchanges, 4 bytes a lane out.  A workgroup takes 16 quads of a
// row where a row's scales lie together, 16 rows of a quad where a quad's do: its scales are one piece
// of 64 bytes either way.  Bound by memory, 2 bytes read and 0.53 written a value: 8192 x 8192 bfloat16 in 34 us (scales by
// rows) or 36 (by quads), 5.0 TB/s, where a copy reaches 5.2.
template <class T, bool WIDE>
__device__ __forceinline__ void mx_quant_rows(const MxQuantArgs& p, uint32_t group, uint32_t groups) {
  const bool along = p.s.quad == 4;
  const int64_t quads = cdiv(p.cols, kQuad), total = along ? cdiv(p.rows * quads, 16) : cdiv(p.rows, 16) * quads;
  const int lane = threadIdx.x & 15, which = threadIdx.x >> 4;
  for (int64_t b = group; b < total; b += groups) {
    const int64_t i = along ? b * 16 + which : b;
    int64_t row = p.rows * quads >> 32 ? i / quads : (int64_t)((uint32_t)i / (uint32_t)quads);
    const int64_t kq = i - row * quads;
    if (!along) row = row * 16 + which;
    if (row >= p.rows) continue;
    const int64_t c0 = kq * kQuad + lane * 8;
    const T* x = (const T*)p.x + row * p.sr;
    Eight<T> v;
    if (WIDE && c0 + 8 <= p.cols)
      v.load(x + c0);
    else
      v.load(x, c0, p.cols, p.sc);
    const uint32_t m = quad_umax(v.largest());
    *(uint32_t*)(p.q + row * p.ldq + c0 / 2) = v.packed(mx_exponent(m));
    // (a block past the columns holds zeros: its byte is that of 2^-102, never NaN's)
    const uint32_t scales = quad_bytes(mx_byte(m), lane);
    if (lane == 0) *(uint32_t*)(p.s.s + row * p.s.row + kq * p.s.quad) = scales;
  }
}

// Scale bytes of any strides in the products' order, [quads][rows] dwords, zero past the blocks.
struct MxScaleArgs {
  const uint8_t* src;
  int64_t rows, blocks, s_r, s_b;
  uint32_t* dst;  // [quads][ld]
  int64_t ld;
};
// 16 rows by 16 quads a workgroup: pieces of 64 bytes on both sides.
__host__ __device__ inline int64_t mx_scales_tiles(const MxScaleArgs& p) {
  return cdiv(p.rows, 16) * cdiv(p.blocks, 64);
}
__device__ __forceinline__ void mx_scales(const MxScaleArgs& p, uint32_t group, uint32_t groups) {
  const int64_t tiles_q = cdiv(p.blocks, 64), tiles = mx_scales_tiles(p);
  for (int64_t i = group; i < tiles; i += groups) {
    const int64_t rb = i / tiles_q, r = rb * 16 + (threadIdx.x >> 4), kq = (i - rb * tiles_q) * 16 + (threadIdx.x & 15);
    if (r >= p.rows || 4 * kq >= p.blocks) continue;
    const uint8_t* s = p.src + r * p.s_r + 4 * kq * p.s_b;
    uint32_t v = 0;
    if (p.s_b == 1 && 4 * kq + 4 <= p.blocks) {
      __builtin_memcpy(&v, s, 4);
    } else {  // (inside the row, all in flight together: see load_clamped)
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = s[(4 * kq + j < p.blocks ? j : p.blocks - 1 - 4 * kq) * p.s_b];
#pragma unroll
      for (int j = 0; j < 4; ++j) v |= 4 * kq + j < p.blocks ? b[j] << (8 * j) : 0;
    }
    p.dst[kq * p.ld + r] = v;
  }
}

// What a product needs before it: the rows of two operands copied to an alignment, their scales in its
// order (any of it may be none).  ODD: an odd number of values, whose last byte holds one.
template <bool ODD>
__global__ __launch_bounds__(256) void mx_pack_kernel(Pack8Args x, Pack8Args w, MxScaleArgs a, MxScaleArgs b,
                                                      uint32_t nx, uint32_t nw, uint32_t na) {
  uint32_t group = blockIdx.x;
  if (group < nx) return pack8<ODD>(x, group, nx);
  group -= nx;
  if (group < nw) return pack8<ODD>(w, group, nw);
  group -= nw;
  if (group < na) return mx_scales(a, group, na);
  mx_scales(b, group - na, gridDim.x - nx - nw - na);
}

// Tokens quantised, beside a weight's scales reordered and its rows copied to an alignment (either
// may be none): what a product of new tokens with a stored weight needs before it.
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void mx_prepare_kernel(MxQuantArgs q, MxScaleArgs s, Pack8Args w, uint32_t packs,
                                                         uint32_t scales) {
  if (blockIdx.x < packs)
    pack8(w, blockIdx.x, packs);
  else if (blockIdx.x < packs + scales)
    mx_scales(s, blockIdx.x - packs, scales);
  else
    mx_quant_rows<T, WIDE>(q, blockIdx.x - packs - scales, gridDim.x - packs - scales);
}

struct Fp4Source {};  // x of MxQuantArgs held in 4 bits

// Eight values of a row from column c (a multiple of 8), as T.
template <class S, class T>
__device__ __forceinline__ Eight<T> mx_load(const MxQuantArgs& p, int64_t r, int64_t c) {
  Eight<T> v;
  v.zero();
  if (r >= p.rows || c >= p.cols) return v;
  if constexpr (std::is_same_v<S, Fp4Source>) {
    const uint8_t* q = (const uint8_t*)p.x + r * p.sr + c / 2 * p.sc;
    uint32_t u = 0, b[4];
    const int64_t last = (p.cols - 1 - c) / 2;  // (inside the row, all in flight together: see load_clamped)
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = q[(i < last ? i : last) * p.sc];
#pragma unroll
    for (int i = 0; i < 4; ++i) u |= i <= last ? b[i] << (8 * i) : 0;
    float f[8];
    unpack_e2m1(u, p.xs[r * p.xsr + c / kMx * p.xsc], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v.d[i] = c + i < p.cols ? __float_as_uint(f[i]) : 0;
  } else {
    v.load((const T*)p.x + r * p.sr, c, p.cols, p.sc);
  }
  return v;
}

// A 128 x 128 tile a workgroup, read once: quantised along its rows (q), its columns (qt, the
// result transposed) or both.  Thread (r, c) holds rows 8 r .. 8 r + 7, columns 8 c .. 8 c + 7: a row's block is four
// lanes, a column's block one wave's 32 rows, four DPP rows apart, so no maximum leaves a wave.
// 8192 x 8192 bfloat16 in both directions 44 us, 4.7 TB/s (as FP32 values, each load behind its own condition, 69).
template <class S, bool WIDE>
__device__ __forceinline__ void mx_quant_tile(const MxQuantArgs& p, uint32_t index) {
  typedef std::conditional_t<std::is_same_v<S, Fp4Source>, float, S> T;  // (4-bit values as FP32)
  typedef Eight<T> E;
  // The transposed tile, 64 bytes a column: 16-byte unit u (a wave's rows) of column col at u ^ (col / 8 % 4).
  __shared__ __align__(16) uint8_t tile[kQuad * 64];
  __shared__ __align__(4) uint8_t bytes[kQuad * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = tid >> 4, c = tid & 15;
  const uint32_t tiles_k = (uint32_t)cdiv(p.cols, kQuad);
  const int64_t rb = index / tiles_k, kb = index - rb * tiles_k, r0 = rb * kQuad + r * 8, c0 = kb * kQuad + c * 8;
  E v[8];
  if (WIDE && rb * kQuad + kQuad <= p.rows && kb * kQuad + kQuad <= p.cols) {  // (the tile's, for all threads)
    const T* x = (const T*)p.x + r0 * p.sr + c0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(x + i * p.sr);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_load<S, T>(p, r0 + i, c0);
  }
  if (p.q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = quad_umax(v[i].largest());
      const uint32_t q = v[i].packed(mx_exponent(m)), s = quad_bytes(mx_byte(m), lane);
      if (r0 + i < p.rows) {
        *(uint32_t*)(p.q + (r0 + i) * p.ldq + c0 / 2) = q;
        if (c == 0) *(uint32_t*)(p.s.s + (r0 + i) * p.s.row + kb * p.s.quad) = s;
      }
    }
  }
  if (!p.qt) return;
  uint32_t most[E::N];  // of the columns, as the values are held
#pragma unroll
  for (int d = 0; d < E::N; ++d) {
    uint32_t m = E::magnitude(v[0].d[d]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = E::larger(m, E::magnitude(v[i].d[d]));
    m = E::larger(m, (uint32_t)__shfl_xor((int)m, 16));
    most[d] = E::larger(m, (uint32_t)__shfl_xor((int)m, 32));
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t m = E::bits(E::PAIRS ? most[j * E::N / 8] >> 16 * (j % 2) & 0xffffu : most[j * E::N / 8]);
    *(uint32_t*)(tile + (c * 8 + j) * 64 + (wave ^ (c & 3)) * 16 + (r & 3) * 4) = E::column(v, j).packed(mx_exponent(m));
    if (lane < 16) bytes[(c * 8 + j) * 4 + wave] = (uint8_t)mx_byte(m);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int col = k * 64 + (tid >> 2), u = tid & 3;
    if (kb * kQuad + col < p.cols)
      *(i32x4*)(p.qt + (kb * kQuad + col) * p.ldqt + rb * 64 + u * 16) =
          *(const i32x4*)(tile + col * 64 + (u ^ (col >> 3 & 3)) * 16);
  }
  if (tid < kQuad && kb * kQuad + tid < p.cols)
    *(uint32_t*)(p.st.s + (kb * kQuad + tid) * p.st.row + rb * p.st.quad) = *(const uint32_t*)(bytes + tid * 4);
}

// One matrix or two: the first `first` workgroups have a's tiles.
template <class S, bool WIDE>
__global__ __launch_bounds__(256) void mx_quant_tile_kernel(MxQuantArgs a, MxQuantArgs b, uint32_t first) {
  const bool is_a = blockIdx.x < first;
  mx_quant_tile<S, WIDE>(is_a ? a : b, is_a ? blockIdx.x : blockIdx.x - first);
}

// The values of a 4-bit matrix, eight a thread: 8192 x 8192 to bfloat16 in 29 us, 5.9 TB/s of which 4.7 written.
struct MxValuesArgs {
  const uint8_t* q;
  int64_t q_r, q_c;  // byte strides
  const uint8_t* s;
  int64_t s_r, s_b;
  int64_t rows, cols;
  void* out;  // [rows][cols]
};
template <class T>
__global__ __launch_bounds__(256) void mx_values_kernel(MxValuesArgs p) {
  const int64_t units = cdiv(p.cols, 8), total = p.rows * units;
  struct alignas(8 * sizeof(T) < 16 ? 8 * sizeof(T) : 16) Pack {
    T t[8];
  };
  const bool wide = p.cols % 8 == 0, whole = p.q_c == 1;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = total >> 32 ? i / units : (int64_t)((uint32_t)i / (uint32_t)units), c = (i - r * units) * 8;
    const uint8_t* q = p.q + r * p.q_r + c / 2 * p.q_c;
    uint32_t u = 0;
    if (whole && c + 8 <= p.cols) {
      __builtin_memcpy(&u, q, 4);
    } else {
      uint32_t b[4];
      const int64_t last = (p.cols - 1 - c) / 2;  // (inside the row, all in flight together: see load_clamped)
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = q[(j < last ? j : last) * p.q_c];
#pragma unroll
      for (int j = 0; j < 4; ++j) u |= j <= last ? b[j] << (8 * j) : 0;
    }
    float v[8];
    unpack_e2m1(u, p.s[r * p.s_r + c / kMx * p.s_b], v);
    T* out = (T*)p.out + r * p.cols + c;
    if (wide) {
      Pack k;
#pragma unroll
      for (int j = 0; j < 8; ++j) k.t[j] = (T)v[j];
      *(Pack*)out = k;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.cols) out[j] = (T)v[j];
    }
  }
}

}  // namespace f16ops

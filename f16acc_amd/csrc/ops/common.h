// What the 8-bit products and the mixture-of-experts kernels share: types,
// wave reductions, e4m3 conversion and the global -> LDS copies.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "f16acc_ops.h"

namespace f16ops {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16;
typedef __bf16 bf16;
#define LDS_AS __attribute__((address_space(3)))

constexpr int kNumXcd = 8;       // workgroups are dealt round-robin over 8 XCDs
constexpr int kCus = 256;        // compute units of an MI355X
constexpr int kBlock = 128;      // quantisation block
constexpr int kMaxExperts = 1024;
constexpr int kOob = 0x7fffff00; // buffer offset past num_records: the load returns 0

// A block whose largest magnitude is below 2^-100 is scaled as if it were
// 2^-100, so 448 / m stays finite and an all-zero block needs no branch.
constexpr uint32_t kTinyBits = (127u - 100u) << 23;
constexpr uint32_t kInfBits = 0x7f800000u;

template <class T>
struct TypeId;
template <>
struct TypeId<f16> { static constexpr int id = F16ACC_TYPE_F16; };
template <>
struct TypeId<bf16> { static constexpr int id = F16ACC_TYPE_BF16; };
template <>
struct TypeId<float> { static constexpr int id = F16ACC_TYPE_F32; };

inline int type_size(int t) { return t == F16ACC_TYPE_F32 ? 4 : 2; }
__host__ __device__ inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// |x| as an integer: NaN > inf > finite in this order, so an integer maximum
// of it keeps a NaN, which a float maximum would drop.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}

// Maximum over the 16 lanes of a DPP row, in every lane of it (rotations).
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
  v = umax(v, dpp<0x121>(v));  // row_ror:1
  v = umax(v, dpp<0x122>(v));
  v = umax(v, dpp<0x124>(v));
  return umax(v, dpp<0x128>(v));
}

// Scale and reciprocal of a block from the bits of its largest magnitude: both
// correctly rounded FP32 quotients.  A block that holds an infinity or a NaN
// has the scale NaN.
//
// The quotients take 4 and 13 instructions here, 45 by `/`, which was half of what
// the quantising kernels issued.  m lies in [2^-100, 2^128), so neither quotient
// leaves the normal range and none of the operators' scaling steps are needed:
// m / 448 is a product with the reciprocal and one remainder step; 448 / m
// refines the hardware's reciprocal and the quotient by remainders.  Both equal `/` for every
// mantissa (all 2^23 compared, at the ends of the exponent range and between).
struct BlockScale {
  float s, inv;
};
__device__ __forceinline__ float over_448(float m) {
  constexpr float r = 1.0f / 448.0f;
  const float q = m * r;
  return __builtin_fmaf(__builtin_fmaf(-q, 448.0f, m), r, q);
}
__device__ __forceinline__ float div_448(float m) {
  const float down = m > 0x1p60f ? 0x1p-64f : 1.0f;  // (the reciprocal of a large m would be subnormal)
  m *= down;
  float r = __builtin_amdgcn_rcpf(m);
  r = __builtin_fmaf(__builtin_fmaf(-m, r, 1.0f), r, r);
  float q = 448.0f * r;
  q = __builtin_fmaf(__builtin_fmaf(-m, q, 448.0f), r, q);
  q = __builtin_fmaf(__builtin_fmaf(-m, q, 448.0f), r, q);
  return q * down;
}
__device__ __forceinline__ BlockScale block_scale(uint32_t bits) {
  const float m = __uint_as_float(umax(bits, kTinyBits));
  BlockScale r;
  r.s = bits >= kInfBits ? __uint_as_float(0x7fc00000u) : over_448(m);
  r.inv = div_448(m);
  return r;
}

// Four values times the block's reciprocal as e4m3, nearest even, in one
// dword.  Rounding can carry a product past 448 by a part in 2^23, which the
// conversion rounds back to 448, so nothing is clamped.
__device__ __forceinline__ int pack_e4m3(float a, float b, float c, float d, float inv) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, r, true);
}

// N consecutive elements from p as floats; wide loads where p is known to be
// aligned to them.
template <int N, class T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[N]) {
  struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Pack {
    T t[N];
  };
  const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (float)k.t[i];
}

// Up to N elements of a strided row from c on, zero past its end.  Every load reads inside the row, so all are in
// flight together: behind a branch each, the last columns of an odd width waited for one after another.
template <int N, class T>
__device__ __forceinline__ void load_clamped(const T* row, int64_t c, int64_t cols, int64_t stride, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (float)row[(c + i < cols ? c + i : cols - 1) * stride];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + i < cols ? v[i] : 0.0f;
}

// 16 bytes of a row of `bytes` >= 16 from k on, zero past its end: the last 16 before the end, moved down, in one load.
// (A loop over bytes there took 70 registers amid what was in flight, and a load each a wave's time.)
__device__ __forceinline__ i32x4 unit_of_row(const uint8_t* row, int64_t k, int64_t bytes) {
  const int over = k + 16 <= bytes ? 0 : k >= bytes ? 16 : (int)(k + 16 - bytes), bits = 8 * over;
  union {
    uint64_t d[2];
    i32x4 v;
  } u;
  __builtin_memcpy(&u, row + (over ? bytes - 16 : k), 16);
  const uint64_t lo = u.d[0], hi = u.d[1];
  u.d[0] = bits >= 64 ? hi >> (bits & 63) : bits ? lo >> bits | hi << (64 - bits) : lo;
  u.d[1] = bits >= 64 ? 0 : hi >> bits;
  if (over == 16) u.d[0] = 0;
  return u.v;
}

// SiLU with FP32's accuracy, behind sums of that accuracy: what is quantised from
// it should fall on the right side of a tie.
__device__ __forceinline__ float silu_exact(float g) { return g / (1.0f + expf(-g)); }
// SiLU, to a few units in the last place, behind 8-bit sums: the hardware's exponential
// and reciprocal (a correctly rounded quotient was a fifth of the gated product's time).
__device__ __forceinline__ float silu(float g) { return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// Raw buffer resource over `bytes` bytes at `base` (stride 0; reads past the
// end return 0).  Wave-uniform.
__device__ __forceinline__ i32x4 make_srd(const void* base, int64_t bytes) {
  const uint64_t a = (uint64_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  r[2] = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes < kOob ? bytes : kOob));
  r[3] = 0x00020000;
  return r;
}

// The resource moved up by `off` bytes (wave-uniform), its records lowered to match.
__device__ __forceinline__ i32x4 srd_at(const i32x4& r, int off) {
  i32x4 q = r;
  const uint64_t base = (((uint64_t)(uint32_t)r[1] << 32) | (uint32_t)r[0]) + (uint32_t)off;
  q[0] = (int)(uint32_t)base;
  q[1] = (int)(uint32_t)(base >> 32);
  q[2] = r[2] > off ? r[2] - off : 0;
  return q;
}

// One global -> LDS copy per lane of 16 bytes (4 bytes): lane i writes LDS
// bytes [lds + 16 i, + 16).  Issued as asm, so the compiler does not take it for a
// store to every LDS buffer; the K loops wait for it with wait_vm and a
// barrier.  M0 carries the LDS address, one wait state before the copy reads it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: the asm sets it itself
__device__ __forceinline__ void lds_dma16(const i32x4& rsrc, int lds, int voff) {
  i32x4 srd;
#pragma unroll
  for (int k = 0; k < 4; ++k) srd[k] = __builtin_amdgcn_readfirstlane(rsrc[k]);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voff), "s"(srd)
      : "memory", "m0");
}
__device__ __forceinline__ void lds_dma4(const i32x4& rsrc, int lds, int voff) {
  i32x4 srd;
#pragma unroll
  for (int k = 0; k < 4; ++k) srd[k] = __builtin_amdgcn_readfirstlane(rsrc[k]);
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dword %1, %2, 0 offen lds"
      :
      : "s"(lds), "v"(voff), "s"(srd)
      : "memory", "m0");
}
#pragma clang diagnostic pop

// s_waitcnt vmcnt(N), other counters left alone.
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N <= 63, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// LDS written by lanes of a wave and read by others of it: its accesses run in
// order, so only the compiler has to keep them apart.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A barrier for LDS alone: loads into registers stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  barrier();
}

// XCD-contiguous renumbering of a launch's workgroups: block b runs on XCD
// b % 8, and each XCD has its own L2, so every XCD gets one contiguous range.
__device__ __forceinline__ uint32_t xcd_order(uint32_t block, uint32_t total) {
  const uint32_t x = block % kNumXcd, l = block / kNumXcd, q = total / kNumXcd, r = total % kNumXcd;
  return x * q + (x < r ? x : r) + l;
}

inline int hip_status() { return (int)hipGetLastError(); }

}  // namespace f16ops

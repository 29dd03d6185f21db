// The product of microscaled 4-bit operands:
//
//   c[m][n] = sum_b sx[m][b] * sw[n][b] * sum_{k in b} x[m][k] * w[n][k],  blocks b of 32
//
// on v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies by the blocks' powers of two itself and adds in
// FP32: the products of e2m1 values are multiples of 1/4 up to 36, so a block's sum is exact.
// The weights are the MFMA's rows and the tokens its columns, so a lane holds groups of four consecutive n
// of one token.
//
// A workgroup stages 256 columns (128 bytes a row) of BM tokens and BN weight rows and their scales in LDS with
// global -> LDS copies, in a ring of NS stages; the next step's fragments and the next stage's copies go
// out one by one between the matrix instructions.
//
// Measured (bfloat16 result): 8192^3 on 256 x 256 tiles 257 to 270 us at best, 4.1 to 4.3 PFLOPS, and 277 to 343 in
// the median of calls one after another, by the card and the clock that their power leaves it (operands of zeros: 191 to 221);
// 254 with the operands in the caches.  Alone the matrix instructions would take 200 us (at the clock that they leave), the
// copies 207 (2.28 GB, 11.0 TB/s into LDS, whatever the depth of the ring), the fragment reads 121; they do not
// overlap all the time.  What did not help: stages of half lines (128 columns, four of them, 300 us
// where this took 280), four waves of 128 x 128 (the accumulators leave no registers), workgroups that go on to the next tile
// (286), touching the lines of later stages ahead (336).
#pragma once

#include "common.h"
#include "fp4.h"
#include "mm.h"

namespace f16ops {

struct Mx4Args {
  const uint8_t* x;  // [M][ldx] bytes, 16-byte aligned rows, zero from K to the next multiple of 32 values
  int64_t ldx;
  const uint8_t* sx;  // the dword of (row m, quad of blocks q) at m * sxm + q * sxq bytes
  int64_t sxm, sxq;
  const uint8_t* w;  // [N][ldw]
  int64_t ldw;
  const uint8_t* sw;
  int64_t swm, swq;
  const void* bias;  // [N] in the output's type, or NULL
  void* c;
  int64_t scm, scn;
  int64_t M, N, K;
  int ctype;
  // A split of K: workgroups (blockIdx.y) take ksplit stages each and write FP32
  // sums to parts[split][M][N]; 0: not split.
  int ksplit;
  float* parts;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int BM_, int BN_, int WM_, int WN_, int BK_, int NS_, int OCC_>
struct Mx4Cfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NS = NS_, OCC = OCC_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  static constexpr int UNITS = BK / 32, ROW = BK / 2;  // 16-byte units and bytes of a staged row
  static constexpr int QUADS = BK / kQuad, STEPS = BK / 64;
  static constexpr int LX = BM * UNITS / THREADS, LW = BN * UNITS / THREADS;  // 16-byte copies per lane and stage
  static constexpr int SX = (BM + 63) / 64 * 64, SROWS = SX + (BN + 63) / 64 * 64;  // scale dwords of a quad
  static constexpr int LS = (SROWS * QUADS + THREADS - 1) / THREADS, LOADS = LX + LW + LS;
  static constexpr int X_BYTES = BM * ROW, W_BYTES = BN * ROW, STAGE = X_BYTES + W_BYTES + LS * THREADS * 4;
  static_assert(LX * THREADS == BM * UNITS && LW * THREADS == BN * UNITS, "whole copies");
  static_assert(THREADS / UNITS % 16 == 0, "a lane's units keep the swizzle phase");
  static_assert(UNITS == 4 || UNITS == 8, "a quad or two of blocks a stage");
  static_assert(STAGE * NS <= 160 * 1024, "LDS of a CU");
  static_assert((NS - 1) * LOADS <= 63, "outstanding copies must fit vmcnt");
};

__device__ __forceinline__ f32x16 mfma_mx(const i32x4& w, const i32x4& x, const f32x16& sum, int sw, int sx, int step) {
  const i32x8 a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const i32x8 b = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  // 4: e2m1; the byte of the scale registers is a part of the instruction
  return step == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, sum, 4, 4, 0, sw, 0, sx)
                   : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, sum, 4, 4, 1, sw, 1, sx);
}

// T: the result's type (the parts of a split of K: FP32).
template <class C, class T>
struct Mx4Kernel {
  static constexpr int FP = C::FN < 2 ? C::FN : 2, COLS = 32 * FP;  // fragments and columns of a pass of the stores
  static constexpr int E = 16 / sizeof(T), OUT_ROW = COLS * sizeof(T) + 16;
  static_assert(C::WAVES * 32 * OUT_ROW <= C::STAGE * C::NS, "the stores' passes fit the ring");
  static_assert(C::FN % FP == 0, "whole passes");

  // Where a unit of a row lies: the 16 rows that a quarter of a fragment read touches fall on all banks.
  __device__ static __forceinline__ int swizzle(int row) { return C::UNITS == 4 ? row >> 2 & 3 : swz(row); }

  // Where the copies of the next stage read: resources whose bases move along K, and a lane's offsets.
  struct Loader {
    i32x4 xr, wr, sr[C::LS];
    int x_off[C::LX], w_off[C::LW], s_off[C::LS];
    int units;  // of a row, from the stage on
  };

  __device__ static __forceinline__ void moved(i32x4& r, int64_t bytes) {
    const uint64_t base = (((uint64_t)(uint32_t)r[1] << 32) | (uint32_t)r[0]) + (uint64_t)bytes;
    r[0] = (int)(uint32_t)base;
    r[1] = (int)(uint32_t)(base >> 32);
  }

  struct Tile;
  __device__ static __forceinline__ void init(Loader& l, const Mx4Args& p, const Tile& t, int k0, int tid) {
    const int row = tid / C::UNITS, u = (tid % C::UNITS) ^ swizzle(row), step = C::THREADS / C::UNITS;
    l.units = (int)cdiv(p.K, kMx) - k0 * C::UNITS;
#pragma unroll
    for (int j = 0; j < C::LX; ++j) l.x_off[j] = (int)((row + j * step) * p.ldx) + u * 16;
#pragma unroll
    for (int j = 0; j < C::LW; ++j) l.w_off[j] = (int)((row + j * step) * p.ldw) + u * 16;
    // (a row past the last one lies past the records, wherever along K the base is)
    l.xr = make_srd(p.x + t.m0 * p.ldx, t.m_left * p.ldx);
    l.wr = make_srd(p.w + t.n0 * p.ldw, t.n_left * p.ldw);
    moved(l.xr, (int64_t)k0 * C::ROW);
    moved(l.wr, (int64_t)k0 * C::ROW);
#pragma unroll
    for (int i = 0; i < C::LS; ++i) {
      const int at = i * C::THREADS + tid, q = __builtin_amdgcn_readfirstlane(at / C::SROWS), r = at % C::SROWS;
      const bool is_x = __builtin_amdgcn_readfirstlane(r < C::SX);  // (multiples of 64: the same in a wave)
      const int s_row = is_x ? r : r - C::SX, rows = is_x ? (t.m_left < C::BM ? t.m_left : C::BM) : (t.n_left < C::BN ? t.n_left : C::BN);
      l.s_off[i] = q < C::QUADS && s_row < rows ? (int)(s_row * (is_x ? p.sxm : p.swm)) : kOob;
      l.sr[i] = make_srd(is_x ? p.sx + t.m0 * p.sxm : p.sw + t.n0 * p.swm, kOob);
      moved(l.sr[i], ((int64_t)k0 * C::QUADS + q) * (is_x ? p.sxq : p.swq));
    }
  }

  // The copies of a stage into the one at `slot`, one by one.  With `any` false every unit reads zeros.
  struct Stage {
    i32x4 xr, wr, sr[C::LS];
    int x_off[C::LX], w_off[C::LW], s_off[C::LS], base, sbase;
    __device__ __forceinline__ void unit(int j) const {
      constexpr int STEP = C::THREADS * 16;
      if (j < C::LX)
        lds_dma16(xr, base + j * STEP, x_off[j]);
      else if (j < C::LX + C::LW)
        lds_dma16(wr, base + j * STEP, w_off[j - C::LX]);
      else
        lds_dma4(sr[j - C::LX - C::LW], sbase + (j - C::LX - C::LW) * C::THREADS * 4, s_off[j - C::LX - C::LW]);
    }
    __device__ __forceinline__ void all() const {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) unit(j);
    }
  };
  __device__ static __forceinline__ Stage stage(const Loader& l, bool any, int slot, int tid, int wave) {
    const int row = tid / C::UNITS, u = (tid % C::UNITS) ^ swizzle(row);
    Stage st;
    st.xr = l.xr, st.wr = l.wr;
    const bool in = any && u < l.units;
#pragma unroll
    for (int j = 0; j < C::LX; ++j) st.x_off[j] = in ? l.x_off[j] : kOob;
#pragma unroll
    for (int j = 0; j < C::LW; ++j) st.w_off[j] = in ? l.w_off[j] : kOob;
#pragma unroll
    for (int i = 0; i < C::LS; ++i) {
      const int q = __builtin_amdgcn_readfirstlane((i * C::THREADS + tid) / C::SROWS);
      st.sr[i] = l.sr[i];
      st.s_off[i] = any && 4 * q < l.units ? l.s_off[i] : kOob;
    }
    st.base = slot + wave * 1024;
    st.sbase = slot + C::X_BYTES + C::W_BYTES + wave * 256;
    return st;
  }
  __device__ static __forceinline__ void next_stage(Loader& l, const Mx4Args& p, int tid) {
    l.units -= C::UNITS;
    moved(l.xr, C::ROW);
    moved(l.wr, C::ROW);
#pragma unroll
    for (int i = 0; i < C::LS; ++i) {
      const bool is_x = __builtin_amdgcn_readfirstlane((i * C::THREADS + tid) % C::SROWS < C::SX);
      moved(l.sr[i], C::QUADS * (is_x ? p.sxq : p.swq));
    }
  }

  // Tile `id` of the launch: its first token and weight row.
  struct Tile {
    int64_t m0, n0;
    int m_left, n_left;
    __device__ __forceinline__ Tile(const Mx4Args& p, uint32_t at) {
      const uint32_t tiles_n = (uint32_t)cdiv(p.N, C::BN), tiles_m = (uint32_t)cdiv(p.M, C::BM);
      uint32_t id = xcd_order(at, tiles_m * tiles_n);
      // 8 tile rows at a time, column by column, so an XCD's tiles share operands
      const uint32_t width = 8 * tiles_n, first = tiles_m > 8 ? id / width * 8 : 0;
      const uint32_t gsz = tiles_m - first < 8 ? tiles_m - first : 8;
      id -= first * tiles_n;
      const uint32_t col = id / gsz;
      m0 = (int64_t)(first + (id - col * gsz)) * C::BM, n0 = (int64_t)col * C::BN;
      m_left = (int)(p.M - m0 < C::BM ? p.M - m0 : C::BM), n_left = (int)(p.N - n0 < C::BN ? p.N - n0 : C::BN);
    }
  };

  __device__ static __forceinline__ void run(const Mx4Args& p, char LDS_AS* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN, t32 = lane & 31, h = lane >> 5;
    const int lds0 = __builtin_amdgcn_readfirstlane((int)(uint32_t)(size_t)lds);
    int kb = 0, nk = (int)cdiv(p.K, C::BK);
    if (p.ksplit) {
      kb = (int)blockIdx.y * p.ksplit;
      nk = kb + p.ksplit < nk ? kb + p.ksplit : nk;
    }
    const Tile t(p, blockIdx.x);
    Loader l;
    init(l, p, t, kb, tid);
#pragma unroll
    for (int s = 0; s < C::NS; ++s) {
      stage(l, kb + s < nk, lds0 + s * C::STAGE, tid, wave).all();
      next_stage(l, p, tid);
    }
    f32x16 acc[C::FM][C::FN];
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    const int xa = (wm * C::TM + t32) * C::ROW, wa = C::X_BYTES + (wn * C::TN + t32) * C::ROW;
    const int sa = C::X_BYTES + C::W_BYTES + 2 * h, sxa = sa + (wm * C::TM + t32) * 4;
    const int swa = sa + (C::SX + wn * C::TN + t32) * 4, phase = swizzle(t32);
    i32x4 xf[2][C::FM], wf[2][C::FN];
    int sx[C::FM], sw[C::FN], nsx[C::FM], nsw[C::FN];  // a quad's scales, and the next one's
    // Step s multiplies unit 2 h + s % 2 of quad s / 2, with byte s % 2 of the half dword that holds its scales.
    // Fragment f (the tokens' first) of step s, and with an even step its scales.
    auto read = [&](int at, int s, int f) {
      const int u = ((4 * (s / 2) + 2 * h + s % 2) ^ phase) * 16, q = s / 2;
      if (f < C::FM) {
        xf[s % 2][f] = *(const i32x4 LDS_AS*)(lds + at + xa + 32 * f * C::ROW + u);
        if (s % 2 == 0) nsx[f] = *(const uint16_t LDS_AS*)(lds + at + sxa + (q * C::SROWS + 32 * f) * 4);
      } else {
        const int j = f - C::FM;
        wf[s % 2][j] = *(const i32x4 LDS_AS*)(lds + at + wa + 32 * j * C::ROW + u);
        if (s % 2 == 0) nsw[j] = *(const uint16_t LDS_AS*)(lds + at + swa + (q * C::SROWS + 32 * j) * 4);
      }
    };
    constexpr int R = C::FM + C::FN, S = C::FM * C::FN;
    int slot = 0;
    wait_vm<(C::NS - 1) * C::LOADS>();
    barrier();
#pragma unroll
    for (int f = 0; f < R; ++f) read(0, 0, f);

    do {
      const int at = slot * C::STAGE, nslot = slot + 1 == C::NS ? 0 : slot + 1, nat = nslot * C::STAGE;
      const Stage next = stage(l, kb + C::NS < nk, lds0 + at, tid, wave);
      next_stage(l, p, tid);
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        constexpr int LAST = C::STEPS - 1;
        if (s % 2 == 0) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i) sx[i] = nsx[i];
#pragma unroll
          for (int j = 0; j < C::FN; ++j) sw[j] = nsw[j];
        }
        if (s == LAST) {
          // This wave has read all of this stage: once every wave has, and the next
          // stage has landed, the copies of the stage after them may begin.
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          wait_vm<(C::NS - 2) * C::LOADS>();
          barrier();
        }
        // The next step's fragments and the copies go out one by one between the matrix instructions.
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int i = 0; i < C::FM; ++i) {
            const int t = j * C::FM + i;
            acc[i][j] = mfma_mx(wf[s % 2][j], xf[s % 2][i], acc[i][j], sw[j], sx[i], s % 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int f = t * R / S; f < (t + 1) * R / S; ++f) read(s == LAST ? nat : at, s == LAST ? 0 : s + 1, f);
            if (s == LAST) {
#pragma unroll
              for (int k = t * C::LOADS / S; k < (t + 1) * C::LOADS / S; ++k) next.unit(k);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      slot = nslot;
    } while (++kb < nk);
    // opaque, or the compiler forms the stores' addresses before the loop and holds them through it
    int ln = lane;
    asm volatile("" : "+v"(ln));
    wait_vm<0>();
    barrier();  // the stages are free
    store(p, lds + wave * 32 * OUT_ROW, acc, t, wm, wn, ln);
  }

  // The wave's sums plus the bias, rounded once; 32 tokens by 64 columns at a time pass through `area`, the
  // wave's share of the stages, and leave as 16-byte units of whole row pieces, at any alignment (columns apart: element
  // by element).
  __device__ static __forceinline__ void store(const Mx4Args& p, char LDS_AS* area, f32x16 (&acc)[C::FM][C::FN],
                                               const Tile& t, int wm, int wn, int lane) {
    const int t32 = lane & 31, h = lane >> 5;
    const int64_t nw = t.n0 + wn * C::TN;
    T* c = (T*)p.c + (p.ksplit ? (int64_t)blockIdx.y * p.M * p.N : 0);
    struct __attribute__((packed, aligned(sizeof(T)))) Unit {
      i32x4 v;
    };
    typedef int Four __attribute__((ext_vector_type(sizeof(T))));  // four values
    constexpr int UNITS = COLS / E;
#pragma unroll
    for (int jp = 0; jp < C::FN; jp += FP) {
      float b[FP][16] = {};
      if (p.bias) {
#pragma unroll
        for (int j = 0; j < FP; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int64_t n = nw + 32 * (jp + j) + 8 * (r / 4) + 4 * h + r % 4;
            b[j][r] = (float)((const T*)p.bias)[n < p.N ? n : p.N - 1];
          }
      }
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
#pragma unroll
        for (int j = 0; j < FP; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            union {
              T t[4];
              Four v;
            } f;
#pragma unroll
            for (int r = 0; r < 4; ++r) f.t[r] = (T)(acc[i][jp + j][4 * g + r] + b[j][4 * g + r]);
            *(Four LDS_AS*)(area + t32 * OUT_ROW + (32 * j + 8 * g + 4 * h) * (int)sizeof(T)) = f.v;
          }
        wave_sync();
#pragma unroll 1
        for (int k = 0; k < 32 * UNITS / 64; ++k) {
          const int row = (k * 64 + lane) / UNITS, u = (k * 64 + lane) % UNITS;
          const int m = wm * C::TM + 32 * i + row;
          const int64_t n = nw + 32 * jp + u * E;
          if (m >= t.m_left || n >= p.N) continue;
          T* to = c + (t.m0 + m) * p.scm + n * p.scn;
          union {
            i32x4 v;
            T t[E];
          } e;
          e.v = *(const i32x4 LDS_AS*)(area + row * OUT_ROW + u * 16);
          if (p.scn == 1 && n + E <= p.N) {
            ((Unit*)to)->v = e.v;
          } else {
#pragma unroll
            for (int r = 0; r < E; ++r)
              if (n + r < p.N) to[r * p.scn] = e.t[r];
          }
        }
        wave_sync();
        __builtin_amdgcn_sched_barrier(0);  // (one pass's values in registers at a time)
      }
    }
  }
};

template <class C, class T>
__global__ __launch_bounds__(C::THREADS, C::OCC) void mm_fp4_kernel(Mx4Args p) {
  __shared__ __align__(1024) char smem[C::STAGE * C::NS];
  Mx4Kernel<C, T>::run(p, (char LDS_AS*)smem);
}

template <class C>
int launch_mm_fp4(Mx4Args p, hipStream_t stream, int splits) {
  const dim3 grid((uint32_t)(cdiv(p.M, C::BM) * cdiv(p.N, C::BN)), (uint32_t)splits);
  if (p.ksplit) p.c = p.parts, p.scm = p.N, p.scn = 1, p.bias = nullptr, p.ctype = F16ACC_TYPE_F32;
  switch (p.ctype) {
    case F16ACC_TYPE_F16: hipLaunchKernelGGL((mm_fp4_kernel<C, f16>), grid, dim3(C::THREADS), 0, stream, p); break;
    case F16ACC_TYPE_BF16: hipLaunchKernelGGL((mm_fp4_kernel<C, bf16>), grid, dim3(C::THREADS), 0, stream, p); break;
    default: hipLaunchKernelGGL((mm_fp4_kernel<C, float>), grid, dim3(C::THREADS), 0, stream, p);
  }
  return hip_status();
}

}  // namespace f16ops

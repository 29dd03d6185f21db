// The product of microscaled 4-bit operands:
//
//   c[m][n] = sum_b sx[m][b] * sw[n][b] * sum_{k in b} x[m][k] * w[n][k],  blocks b of 32
//
// on v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies by the blocks' powers of two itself and adds in
// FP32: the products of e2m1 values are multiples of 1/4 up to 36, so a block's sum is exact.
// The weights are the MFMA's rows and the tokens its columns, so a lane holds groups of four consecutive n
// of one token.
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

template <class C>
struct Mx4Kernel {
  // Where a unit of a row lies: the 16 rows that a quarter of a fragment read touches fall on all banks.
  __device__ static __forceinline__ int swizzle(int row) { return C::UNITS == 4 ? row >> 2 & 3 : swz(row); }

  struct Loader {
    i32x4 xr, wr;
    int x_off, w_off, x_step, w_step, u;
    int s_off[C::LS];
    i32x4 sr[C::LS];
    int s_quad[C::LS];  // the quad of a stage that a scale copy belongs to
    int64_t s_step[C::LS];
    int quads, units;  // of a row
    int k0, nk;        // the stages of this workgroup
  };

  __device__ static __forceinline__ void init(Loader& l, const Mx4Args& p, int64_t m0, int m_left, int64_t n0, int n_left,
                                              int tid) {
    const int row = tid / C::UNITS, u = (tid % C::UNITS) ^ swizzle(row);
    l.u = u;
    l.units = (int)cdiv(p.K, kMx);
    l.quads = (int)cdiv(p.K, kQuad);
    l.k0 = 0;
    l.nk = (int)cdiv(p.K, C::BK);
    if (p.ksplit) {
      l.k0 = (int)blockIdx.y * p.ksplit;
      l.nk = l.k0 + p.ksplit < l.nk ? l.k0 + p.ksplit : l.nk;
    }
    l.x_step = (int)(C::THREADS / C::UNITS * p.ldx);
    l.w_step = (int)(C::THREADS / C::UNITS * p.ldw);
    l.x_off = (int)(row * p.ldx) + u * 16;
    l.w_off = (int)(row * p.ldw) + u * 16;
    l.xr = make_srd(p.x + m0 * p.ldx, m_left * p.ldx);
    l.wr = make_srd(p.w + n0 * p.ldw, n_left * p.ldw);
#pragma unroll
    for (int i = 0; i < C::LS; ++i) {
      const int at = i * C::THREADS + tid, q = at / C::SROWS, r = at % C::SROWS;
      const bool is_x = __builtin_amdgcn_readfirstlane(r < C::SX);  // (multiples of 64: the same in a wave)
      const int s_row = is_x ? r : r - C::SX;
      const bool in = q < C::QUADS && s_row < (is_x ? (m_left < C::BM ? m_left : C::BM) : (n_left < C::BN ? n_left : C::BN));
      l.s_off[i] = in ? (int)(s_row * (is_x ? p.sxm : p.swm)) : kOob;
      l.s_quad[i] = __builtin_amdgcn_readfirstlane(q);
      l.s_step[i] = is_x ? p.sxq : p.swq;
      l.sr[i] = make_srd(is_x ? p.sx + m0 * p.sxm : p.sw + n0 * p.swm, kOob);
    }
  }

  __device__ static __forceinline__ i32x4 advanced(const i32x4& r, int64_t bytes) {
    i32x4 q = r;
    const uint64_t base = (((uint64_t)(uint32_t)r[1] << 32) | (uint32_t)r[0]) + (uint64_t)bytes;
    q[0] = (int)(uint32_t)base;
    q[1] = (int)(uint32_t)(base >> 32);
    return q;
  }

  // The copies of stage kb into the one at `slot`, one by one.  Past the last stage every unit reads zeros.
  struct Stage {
    i32x4 xr, wr;
    int x_off, w_off, base, sbase, kb;
    bool any;
    const Loader* l;
    __device__ __forceinline__ void unit(int j) const {
      constexpr int STEP = C::THREADS * 16;
      if (j < C::LX) {
        lds_dma16(srd_at(xr, j * l->x_step), base + j * STEP, x_off);
      } else if (j < C::LX + C::LW) {
        lds_dma16(srd_at(wr, (j - C::LX) * l->w_step), base + j * STEP, w_off);
      } else {
        const int i = j - C::LX - C::LW, q = kb * C::QUADS + l->s_quad[i];
        lds_dma4(advanced(l->sr[i], q * l->s_step[i]), sbase + i * C::THREADS * 4, any && q < l->quads ? l->s_off[i] : kOob);
      }
    }
    __device__ __forceinline__ void all() const {
#pragma unroll
      for (int j = 0; j < C::LOADS; ++j) unit(j);
    }
  };
  __device__ static __forceinline__ Stage stage(const Loader& l, int kb, int slot, int wave) {
    Stage st;
    st.any = kb < l.nk;
    const bool in = st.any && kb * C::UNITS + l.u < l.units;
    st.xr = advanced(l.xr, (int64_t)kb * C::ROW);
    st.wr = advanced(l.wr, (int64_t)kb * C::ROW);
    st.x_off = in ? l.x_off : kOob;
    st.w_off = in ? l.w_off : kOob;
    st.base = slot + wave * 1024;
    st.sbase = slot + C::X_BYTES + C::W_BYTES + wave * 256;
    st.kb = kb;
    st.l = &l;
    return st;
  }

  __device__ static __forceinline__ void run(const Mx4Args& p, char LDS_AS* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN, t32 = lane & 31, h = lane >> 5;
    const uint32_t tiles_n = (uint32_t)cdiv(p.N, C::BN), tiles_m = (uint32_t)cdiv(p.M, C::BM);
    uint32_t id = xcd_order(blockIdx.x, tiles_m * tiles_n);
    // 8 tile rows at a time, column by column, so an XCD's tiles share operands
    const uint32_t width = 8 * tiles_n, first = tiles_m > 8 ? id / width * 8 : 0;
    const uint32_t gsz = tiles_m - first < 8 ? tiles_m - first : 8;
    id -= first * tiles_n;
    const uint32_t col = id / gsz;
    const int64_t m0 = (int64_t)(first + (id - col * gsz)) * C::BM, n0 = (int64_t)col * C::BN;
    const int m_left = (int)(p.M - m0 < C::BM ? p.M - m0 : C::BM), n_left = (int)(p.N - n0 < C::BN ? p.N - n0 : C::BN);
    Loader l;
    init(l, p, m0, m_left, n0, n_left, tid);
    const int lds0 = __builtin_amdgcn_readfirstlane((int)(uint32_t)(size_t)lds);

    f32x16 acc[C::FM][C::FN];
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

#pragma unroll
    for (int s = 0; s < C::NS; ++s) stage(l, l.k0 + s, lds0 + s * C::STAGE, wave).all();

    const int xa = (wm * C::TM + t32) * C::ROW, wa = C::X_BYTES + (wn * C::TN + t32) * C::ROW;
    const int sa = C::X_BYTES + C::W_BYTES + 2 * h, sxa = sa + (wm * C::TM + t32) * 4;
    const int swa = sa + (C::SX + wn * C::TN + t32) * 4, phase = swizzle(t32);
    i32x4 xf[2][C::FM], wf[2][C::FN];
    int sx[C::FM], sw[C::FN], nsx[C::FM], nsw[C::FN];  // a quad's scales, and the next one's
    // Step s multiplies unit 2 h + s % 2 of quad s / 2, with byte s % 2 of the half dword that holds its scales.
    auto read = [&](int at, int s) {
      const int u = ((4 * (s / 2) + 2 * h + s % 2) ^ phase) * 16;
#pragma unroll
      for (int i = 0; i < C::FM; ++i) xf[s % 2][i] = *(const i32x4 LDS_AS*)(lds + at + xa + 32 * i * C::ROW + u);
#pragma unroll
      for (int j = 0; j < C::FN; ++j) wf[s % 2][j] = *(const i32x4 LDS_AS*)(lds + at + wa + 32 * j * C::ROW + u);
      if (s % 2) return;
      const int q = s / 2;
#pragma unroll
      for (int i = 0; i < C::FM; ++i)
        nsx[i] = *(const uint16_t LDS_AS*)(lds + at + sxa + (q * C::SROWS + 32 * i) * 4);
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
        nsw[j] = *(const uint16_t LDS_AS*)(lds + at + swa + (q * C::SROWS + 32 * j) * 4);
    };
    int slot = 0, kb = l.k0;
    wait_vm<(C::NS - 1) * C::LOADS>();
    barrier();
    read(0, 0);
    do {
      const int at = slot * C::STAGE, nslot = slot + 1 == C::NS ? 0 : slot + 1, nat = nslot * C::STAGE;
      const Stage next = stage(l, kb + C::NS, lds0 + at, wave);
#pragma unroll
      for (int s = 0; s < C::STEPS; ++s) {
        if (s % 2 == 0) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i) sx[i] = nsx[i];
#pragma unroll
          for (int j = 0; j < C::FN; ++j) sw[j] = nsw[j];
        }
        if (s == C::STEPS - 1) {
          // This wave has read all of this stage: once every wave has, and the next
          // stage has landed, the copies of the stage after them may begin.
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          wait_vm<(C::NS - 2) * C::LOADS>();
          barrier();
          read(nat, 0);
          next.all();
        } else {
          read(at, s + 1);
        }
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int i = 0; i < C::FM; ++i)
            acc[i][j] = mfma_mx(wf[s % 2][j], xf[s % 2][i], acc[i][j], sw[j], sx[i], s % 2);
      }
      slot = nslot;
    } while (++kb < l.nk);
    wait_vm<0>();
    // opaque, or the compiler forms the stores' addresses before the loop and holds them through it
    int ln = lane;
    asm volatile("" : "+v"(ln));
    store_all(p, lds, acc, m0, m_left, n0, wave, wm, wn, ln);
  }

  __device__ static __forceinline__ void store_all(const Mx4Args& p, char LDS_AS* lds, f32x16 (&acc)[C::FM][C::FN],
                                                   int64_t m0, int m_left, int64_t n0, int wave, int wm, int wn,
                                                   int lane) {
    if (p.ksplit) {
      Mx4Args q = p;
      q.c = p.parts + (int64_t)blockIdx.y * p.M * p.N;
      q.scm = p.N, q.scn = 1, q.bias = nullptr;
      store<float>(q, lds, acc, m0, m_left, n0, wave, wm, wn, lane);
    } else if (p.ctype == F16ACC_TYPE_F16)
      store<f16>(p, lds, acc, m0, m_left, n0, wave, wm, wn, lane);
    else if (p.ctype == F16ACC_TYPE_BF16)
      store<bf16>(p, lds, acc, m0, m_left, n0, wave, wm, wn, lane);
    else
      store<float>(p, lds, acc, m0, m_left, n0, wave, wm, wn, lane);
  }

  // The wave's sums plus the bias, rounded once; 32 tokens by 64 columns at a time pass through LDS and leave
  // as 16-byte units of whole row pieces, at any alignment.
  template <class T>
  __device__ static __forceinline__ void store(const Mx4Args& p, char LDS_AS* lds, f32x16 (&acc)[C::FM][C::FN],
                                               int64_t m0, int m_left, int64_t n0, int wave, int wm, int wn, int lane) {
    const int t32 = lane & 31, h = lane >> 5;
    const int64_t nw = n0 + wn * C::TN;
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int64_t n = nw + 32 * j + 8 * (r / 4) + 4 * h + r % 4;
          const float b = n < p.N ? (float)((const T*)p.bias)[n] : 0.0f;
#pragma unroll
          for (int i = 0; i < C::FM; ++i) acc[i][j][r] += b;
        }
    }
    if (p.scn != 1) {
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        const int m = wm * C::TM + 32 * i + t32;
#pragma unroll
        for (int j = 0; j < C::FN; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int64_t n = nw + 32 * j + 8 * (r / 4) + 4 * h + r % 4;
            if (m < m_left && n < p.N) ((T*)p.c)[(m0 + m) * p.scm + n * p.scn] = (T)acc[i][j][r];
          }
      }
      return;
    }
    constexpr int FP = C::FN < 2 ? C::FN : 2, COLS = 32 * FP;  // fragments of a pass
    constexpr int E = 16 / sizeof(T), UNITS = COLS / E, ROW = COLS * sizeof(T) + 16;
    static_assert(C::WAVES * 32 * (COLS * 4 + 16) <= C::STAGE * C::NS, "staging fits the ring");
    static_assert(C::FN % FP == 0, "whole passes");
    struct __attribute__((packed, aligned(sizeof(T)))) Unit {
      i32x4 v;
    };
    typedef int Four __attribute__((ext_vector_type(sizeof(T))));  // four values
    char LDS_AS* area = lds + wave * 32 * ROW;
    barrier();  // every wave has read its last stage
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int jp = 0; jp < C::FN; jp += FP) {
#pragma unroll
        for (int j = 0; j < FP; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            union {
              T t[4];
              Four v;
            } f;
#pragma unroll
            for (int r = 0; r < 4; ++r) f.t[r] = (T)acc[i][jp + j][4 * g + r];
            *(Four LDS_AS*)(area + t32 * ROW + (32 * j + 8 * g + 4 * h) * (int)sizeof(T)) = f.v;
          }
        wave_sync();
#pragma unroll
        for (int k = 0; k < 32 * UNITS / 64; ++k) {
          const int row = (k * 64 + lane) / UNITS, u = (k * 64 + lane) % UNITS;
          const int m = wm * C::TM + 32 * i + row;
          const int64_t n = nw + 32 * jp + u * E;
          if (m >= m_left || n >= p.N) continue;
          T* c = (T*)p.c + (m0 + m) * p.scm + n;
          const i32x4 v = *(const i32x4 LDS_AS*)(area + row * ROW + u * 16);
          if (n + E <= p.N) {
            ((Unit*)c)->v = v;
          } else {
            union {
              i32x4 v;
              T t[E];
            } e;
            e.v = v;
#pragma unroll
            for (int r = 0; r < E; ++r)
              if (n + r < p.N) c[r] = e.t[r];
          }
        }
        wave_sync();
      }
  }
};

template <class C>
__global__ __launch_bounds__(C::THREADS, C::OCC) void mm_fp4_kernel(Mx4Args p) {
  __shared__ __align__(1024) char smem[C::STAGE * C::NS];
  Mx4Kernel<C>::run(p, (char LDS_AS*)smem);
}

template <class C>
int launch_mm_fp4(const Mx4Args& p, hipStream_t stream, int splits) {
  const int64_t tiles = cdiv(p.M, C::BM) * cdiv(p.N, C::BN);
  if (tiles > 0x7fffffff) return F16ACC_OPS_E_UNSUPPORTED;
  hipLaunchKernelGGL((mm_fp4_kernel<C>), dim3((uint32_t)tiles, (uint32_t)splits), dim3(C::THREADS), 0, stream, p);
  return hip_status();
}

}  // namespace f16ops

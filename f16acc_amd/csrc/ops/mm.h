// The block-scaled product of e4m3 operands, as one product and as the products
// of a set of experts:
//
//   c[m][n] = sum_kb sx[m][kb] * sw[n][kb] * sum_{k in kb} x[m][k] * w[n][k]
//
// x holds tokens (rows), w weight rows; kb are the blocks of 128 along K.  The
// inner sum is one v_mfma_f32_16x16x128_f8f6f4 (K = 128, one block) into zero,
// the outer one an FP32 multiply-add per element: 32 matrix cycles against 16
// of the vector unit per 16 x 16 block step, which run side by side.  The
// weights are the MFMA's rows and the tokens its columns, so a lane holds four
// consecutive n of ONE token: its scale is one register per 16 tokens, already
// multiplied by the weight block's scale.
//
// A workgroup stages BM tokens and BN weight rows by 128 K in LDS with 16-byte
// global -> LDS copies, in a ring of NS stages; unit u of a row lies at u ^ swz(row),
// which spreads the 16 rows of a fragment read over the banks.  Units past K,
// rows past M or N and tokens of other experts read zeros.
//
// The K loop is one stream of matrix steps: a step's FP32 multiply-adds follow two
// steps later, weight fragments are read two ahead, the next stage's token fragments
// into the registers that the last steps free, and the copies go out one by one behind
// the barrier.  The sums stay in vector registers (128 a lane on 256 x 256, eight
// waves): in accumulation registers every multiply-add would move them out and back.
//
// The 8-bit matrix instructions (16x16x128 here; 32x32x64 and 16x16x32 lose as much) add eight products at a
// time (consecutive k), each cut towards zero to a multiple of 2^-13 of two to the group's
// largest sum of exponents (a subnormal's is -6), and the groups in FP32.  The result is off by
// 1.5e-5 of the 2-norm on normal values, by 7e-5 on positive ones over 18 binades; one element of a few
// products by 2.1e-4 and 2.6e-3 of the sum of their magnitudes at most (measured, 2 million
// elements each).  Everything past one block's sum is FP32.
//
// Gate and up may take the other way (kGatedExact): their result is quantised, and a sum
// that is off by 1e-5 falls on the other side of an e4m3 tie once in some hundred
// values.  Then both operands are converted to binary16, which is exact, and the
// block is four v_mfma_f32_16x16x32_f16 in FP32: twice the matrix cycles and, on
// 64 x 64 sums a wave, two conversions for each MFMA, which bound it (dealing them one by
// one between the MFMAs gained 2 %).  4096 tokens, 8 of 64 experts, 2048 x 1024: 419 us
// on 128 x 256 tiles against 212 in 8 bits on 256 x 256 (profiled; 256 x 256 spills
// with the halves).
//
// Measured (bfloat16 result): 8192^3 450 us, 2440 TFLOPS, where a library's product with
// one scale for everything reaches 2770; 4096^3 64 us, 2150; with a scale for each
// weight row 531 us.  On 8192^3 the matrix unit is busy 61 % of the cycles, at
// about 1.9 GHz; without the copies the same loop ran at 4600 TFLOPS, so what is left
// is the operands' way into LDS: 64 KB a stage and CU, one stage ahead.
#pragma once

#include "common.h"

namespace f16ops {

struct MmArgs {
  const uint8_t* x;  // [M][ldx] bytes, 16-byte aligned rows
  int64_t ldx;
  const float* sx;  // element (m, kb) at m * sxm + kb * sxk
  int64_t sxm, sxk;
  const uint8_t* w;  // [N][ldw]
  int64_t ldw;
  const float* sw;  // element (n or n / 128, kb) at i * swn + kb * swk
  int64_t swn, swk;
  const void* bias;  // [N] in the output's type, or NULL
  void* c;
  int64_t scm, scn;
  int64_t M, N, K;
  int ctype;
  // A split of K: workgroups (blockIdx.y) take ksplit blocks each and write FP32
  // sums to parts[split][M][N]; 0: not split.
  int ksplit;
  float* parts;
  // Experts: the tile list (expert, first slot, end slot, -) and its length, the
  // token row of each slot (NULL: the slot itself), the strides between experts.
  const int4* tiles;
  const int* ntiles;
  const int* rows;
  int64_t xrows;  // rows of x
  int64_t we, swe;
  int tile_rows;  // tokens per entry of the tile list, a multiple of the kernel's
  // Gate and up (kGatedQuant): w holds the gate's N rows, then (at up bytes, its scales at
  // sup elements) the up's; the result goes to q and its scales, quantised.
  int64_t up, sup;
  uint8_t* q;
  int64_t ldq;
  float* sq;
  int64_t ldsq;
};

enum Epilogue { kStore = 0, kGatedQuant = 1, kGatedExact = 2 };

template <int BM_, int BN_, int WM_, int WN_, int NS_, int OCC_>
struct MmCfg {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_, OCC = OCC_;
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr int LX = BM * 8 / THREADS, LW = BN * 8 / THREADS;  // 16-byte copies per lane and stage
  static constexpr int X_BYTES = BM * kBlock, W_BYTES = BN * kBlock, S_BYTES = THREADS * 4;
  static_assert(LX * THREADS == BM * 8 && LW * THREADS == BN * 8, "whole copies");
  static_assert(BM <= THREADS, "one scale copy per stage covers the tokens");
  static_assert(THREADS / 8 % 16 == 0, "a lane's units keep the swizzle phase");
  static constexpr int stage_bytes(bool row_scales) {
    return X_BYTES + W_BYTES + S_BYTES * (row_scales ? 1 + (BN + THREADS - 1) / THREADS : 1);
  }
};

// Spreads the 16 rows that a fragment read touches over the LDS banks.
__device__ __forceinline__ int swz(int row) { return ((row >> 1) ^ ((row & 1) << 2)) & 7; }

__device__ __forceinline__ f32x4 mfma(const i32x8& w, const i32x8& x) {
  const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

// 8 e4m3 values as binary16.
__device__ __forceinline__ f16x8 halves(int lo, int hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
struct Halves {
  f16x8 v[4];
  Halves() = default;
  __device__ __forceinline__ explicit Halves(const i32x8& q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = halves(q[2 * i], q[2 * i + 1]);
  }
};

__device__ __forceinline__ f32x4 mfma_f16(const f16x8& w, const f16x8& x, const f32x4& sum) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(w, x, sum, 0, 0, 0);
}

// Four consecutive outputs of one token from FP32, rounded once.
template <class T>
__device__ __forceinline__ void store4(T* p, int64_t scn, int left, const f32x4& v, bool wide) {
  if (wide && left >= 4) {
    struct alignas(4 * sizeof(T)) Pack {
      T t[4];
    } k;
#pragma unroll
    for (int i = 0; i < 4; ++i) k.t[i] = (T)v[i];
    *(Pack*)p = k;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i * scn] = (T)v[i];
  }
}

template <class C, bool ROW_SCALES, bool EXPERTS, int EPI>
struct MmKernel {
  static constexpr int STAGE = C::stage_bytes(ROW_SCALES);
  static constexpr int LSW = ROW_SCALES ? (C::BN + C::THREADS - 1) / C::THREADS : 0;
  static constexpr int LOADS = C::LX + C::LW + 1 + LSW;
  static constexpr bool EXACT = EPI == kGatedExact, GATED = EPI == kGatedQuant || EXACT;
  static_assert(GATED || kBlock % C::TN == 0, "a wave's weight rows lie in one block");
  static constexpr int BN_OUT = GATED ? C::BN / 2 : C::BN;  // columns of the result
  static_assert((C::NS - 1) * LOADS <= 63, "outstanding copies must fit vmcnt");

  // Where a lane's copies read.
  struct Loader {
    int x_off[EXPERTS ? C::LX : 1], x_step;
    int w_off, w_step, u;  // u: the first k of the lane's units
    int s_off;             // token scale
    int sw_off[ROW_SCALES ? LSW : 1];
    i32x4 xr, wr, ur, sr, swr;
    int64_t sxk, swk;
    int k0, nk, last, krest;  // blocks k0 .. nk - 1 of K; the last block and its length
  };

  __device__ static __forceinline__ void init(Loader& l, const MmArgs& p, int64_t m0, int m_left, int64_t n0,
                                              const uint8_t* w, const float* sw, int tid) {
    const int row = tid >> 3, u = (tid & 7) ^ swz(row);
    l.u = u * 16;
    l.last = (int)cdiv(p.K, kBlock) - 1;
    l.krest = (int)(p.K - (int64_t)l.last * kBlock);
    l.k0 = 0;
    l.nk = l.last + 1;
    if (!EXPERTS && p.ksplit) {
      l.k0 = (int)blockIdx.y * p.ksplit;
      l.nk = l.k0 + p.ksplit < l.nk ? l.k0 + p.ksplit : l.nk;
    }
    l.x_step = (int)(C::THREADS / 8 * p.ldx);
    l.w_step = (int)(C::THREADS / 8 * p.ldw);
    l.w_off = (int)(row * p.ldw) + l.u;
    if (EXPERTS) {
#pragma unroll
      for (int j = 0; j < C::LX; ++j) {
        const int r = row + j * (C::THREADS / 8);
        l.x_off[j] = kOob;
        if (r < m_left) l.x_off[j] = (int)((p.rows ? p.rows[m0 + r] : (int)m0 + r) * p.ldx) + l.u;
      }
      l.xr = make_srd(p.x, p.xrows * p.ldx);
      l.s_off = kOob;
      if (tid < m_left) l.s_off = (int)((p.rows ? p.rows[m0 + tid] : (int)m0 + tid) * p.sxm * 4);
      l.sr = make_srd(p.sx, kOob);
    } else {
      l.x_off[0] = (int)(row * p.ldx) + l.u;
      l.xr = make_srd(p.x + m0 * p.ldx, m_left * p.ldx);
      l.s_off = tid < m_left ? (int)(tid * p.sxm * 4) : kOob;
      l.sr = make_srd(p.sx + m0 * p.sxm, kOob);
    }
    if (C::BM < C::THREADS && tid >= C::BM) l.s_off = kOob;
    const int64_t n_left = p.N - n0;
    l.wr = make_srd(w + n0 * p.ldw, n_left * p.ldw);
    if (GATED) l.ur = make_srd(w + p.up + n0 * p.ldw, n_left * p.ldw);
    if (ROW_SCALES) {
      l.swr = make_srd(sw + n0 * p.swn, kOob);
#pragma unroll
      for (int j = 0; j < LSW; ++j) {
        const int n = tid + j * C::THREADS;
        l.sw_off[j] = n < C::BN && n < n_left ? (int)(n * p.swn * 4) : kOob;
      }
    }
    l.sxk = p.sxk * 4;
    l.swk = p.swk * 4;
  }

  __device__ static __forceinline__ i32x4 advanced(const i32x4& r, int64_t bytes) {
    i32x4 q = r;
    const uint64_t base = (((uint64_t)(uint32_t)r[1] << 32) | (uint32_t)r[0]) + (uint64_t)bytes;
    q[0] = (int)(uint32_t)base;
    q[1] = (int)(uint32_t)(base >> 32);
    return q;
  }

  // The copies of K block kb into the stage at `slot`, one by one: unit(0) .. unit(LOADS - 1).
  // Past the last block every unit reads zeros.
  struct Stage {
    i32x4 xr, wr, ur, sr, swr;
    int x_off, w_off, s_off;  // this lane's offsets, kOob past K
    bool in, any;
    int base, sbase;
    const Loader* l;
    __device__ __forceinline__ void unit(int j) const {
      constexpr int STEP = C::THREADS * 16;
      if (j < C::LX) {
        if (EXPERTS)
          lds_dma16(xr, base + j * STEP, in ? l->x_off[j] : kOob);
        else
          lds_dma16(srd_at(xr, j * l->x_step), base + j * STEP, x_off);
      } else if (j < C::LX + C::LW) {
        const int k = j - C::LX;
        if (GATED && k >= C::LW / 2)
          lds_dma16(srd_at(ur, (k - C::LW / 2) * l->w_step), base + C::X_BYTES + k * STEP, w_off);
        else
          lds_dma16(srd_at(wr, k * l->w_step), base + C::X_BYTES + k * STEP, w_off);
      } else if (j == C::LX + C::LW) {
        lds_dma4(sr, sbase, s_off);
      } else if (ROW_SCALES) {
        const int k = j - C::LX - C::LW - 1;
        lds_dma4(swr, sbase + C::S_BYTES * (1 + k), any ? l->sw_off[k] : kOob);
      }
    }
    __device__ __forceinline__ void all() const {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) unit(j);
    }
  };
  __device__ static __forceinline__ Stage stage(const Loader& l, int kb, int slot, int wave) {
    const int left = kb >= l.nk ? 0 : kb == l.last ? l.krest : kBlock;
    Stage st;
    st.in = l.u < left;
    st.any = left != 0;
    st.xr = advanced(l.xr, (int64_t)kb * kBlock);
    st.wr = advanced(l.wr, (int64_t)kb * kBlock);
    if (GATED) st.ur = advanced(l.ur, (int64_t)kb * kBlock);
    st.sr = advanced(l.sr, kb * l.sxk);
    if (ROW_SCALES) st.swr = advanced(l.swr, kb * l.swk);
    st.x_off = st.in ? l.x_off[0] : kOob;
    st.w_off = st.in ? l.w_off : kOob;
    st.s_off = st.any ? l.s_off : kOob;
    st.base = slot + wave * 1024;
    st.sbase = slot + C::X_BYTES + C::W_BYTES + wave * 256;
    st.l = &l;
    return st;
  }

  // Row of fragment j of the wave's weights in the staged tile.  Gated: the
  // first half of the fragments are gate rows, the second the same up rows.
  __device__ static __forceinline__ int w_row(int wn, int j) {
    if (!GATED) return wn * C::TN + 16 * j;
    return j < C::FN / 2 ? wn * (C::TN / 2) + 16 * j : C::BN / 2 + wn * (C::TN / 2) + 16 * (j - C::FN / 2);
  }

  __device__ static __forceinline__ void run(const MmArgs& p, char LDS_AS* lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN, t16 = lane & 15, g = lane >> 4;
    int64_t m0, n0;
    int m_left;
    const uint8_t* w = p.w;
    const float* sw = p.sw;
    const uint32_t tiles_n = (uint32_t)cdiv(p.N, BN_OUT);
    if (EXPERTS) {
      const uint32_t parts = (uint32_t)p.tile_rows / C::BM, total = (uint32_t)*p.ntiles * parts * tiles_n;
      if (blockIdx.x >= total) return;
      const uint32_t id = xcd_order(blockIdx.x, total), t = id / tiles_n;
      const int4 tile = p.tiles[t / parts];
      const int first = tile.y + (int)(t % parts) * C::BM;
      if (first >= tile.z) return;
      m0 = first;
      m_left = tile.z - first < C::BM ? tile.z - first : C::BM;
      n0 = (int64_t)(id - t * tiles_n) * BN_OUT;
      w += tile.x * p.we;
      sw += tile.x * p.swe;
    } else {
      const uint32_t tiles_m = (uint32_t)cdiv(p.M, C::BM);
      uint32_t id = xcd_order(blockIdx.x, tiles_m * tiles_n);
      // 8 tile rows at a time, column by column, so an XCD's tiles share operands
      const uint32_t width = 8 * tiles_n, first = tiles_m > 8 ? id / width * 8 : 0;
      const uint32_t gsz = tiles_m - first < 8 ? tiles_m - first : 8;
      id -= first * tiles_n;
      const uint32_t col = id / gsz;
      m0 = (int64_t)(first + (id - col * gsz)) * C::BM;
      n0 = (int64_t)col * C::BN;
      m_left = (int)(p.M - m0 < C::BM ? p.M - m0 : C::BM);
    }
    Loader l;
    init(l, p, m0, m_left, n0, w, sw, tid);
    const int lds0 = __builtin_amdgcn_readfirstlane((int)(uint32_t)(size_t)lds);

    f32x4 acc[C::FM][C::FN];
#pragma unroll
    for (int i = 0; i < C::FM; ++i)
#pragma unroll
      for (int j = 0; j < C::FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
    for (int s = 0; s < C::NS; ++s) stage(l, l.k0 + s, lds0 + s * STAGE, wave).all();

    // The weight block's scale, one value a wave (gated: the gate's and the up's), read
    // through the scalar cache: a vector load among the copies would make the
    // compiler wait for all of them.
    const int64_t nb = GATED ? n0 / kBlock : (n0 + wn * C::TN) / kBlock;
    const int64_t nb_last = cdiv(p.N, kBlock) - 1;
    typedef const float __attribute__((address_space(4)))* Scalar;
    const Scalar swp = (Scalar)(uintptr_t)(sw + (nb < nb_last ? nb : nb_last) * p.swn);

    // A wave's addresses in a stage; the fragments of an operand lie 16 rows apart.  Lane group g
    // holds units g and g + 4 of a row's eight.  (The order of k inside a block is the same for both
    // operands, so any will do.)
    const int frag = t16 * kBlock, lo = (g ^ swz(t16)) << 4, hi = ((g + 4) ^ swz(t16)) << 4;
    const int xa = wm * C::TM * kBlock + frag, wa = C::X_BYTES + frag;
    const int sa = C::X_BYTES + C::W_BYTES + (wm * C::TM + t16) * 4;

    auto read = [&](int at) {
      const i32x4 a = *(const i32x4 LDS_AS*)(lds + at + lo), b = *(const i32x4 LDS_AS*)(lds + at + hi);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    constexpr int AHEAD = C::FN > 2 ? 2 : 1, RING = AHEAD == 1 ? 2 : 4;  // fragments of w read ahead
    static_assert(C::FN % RING == 0, "a stage starts with the ring's first slot");
    static_assert(!ROW_SCALES || (RING == 4 && C::FM >= 2), "row scales are read AHEAD of their last use");
    i32x8 xf[C::FM], wf[RING];
    float s[C::FM], sb = 0.0f, sb2 = 0.0f;
    f32x4 sr[4];

    int slot = 0, kb = l.k0;
    wait_vm<(C::NS - 1) * LOADS>();
    barrier();
    // A wave without a token (the last tile of an expert or of M) copies its share
    // and leaves the matrix unit to the others: a half-empty tile takes little over
    // half the time.
    if (wm * C::TM >= m_left) {
      do {
        wait_vm<(C::NS - 2) * LOADS>();
        barrier();
        stage(l, kb + C::NS, lds0 + slot * STAGE, wave).all();
        slot = slot + 1 == C::NS ? 0 : slot + 1;
      } while (++kb < l.nk);
      wait_vm<0>();
      store_all(p, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
      return;
    }
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
      xf[i] = read(xa + 16 * i * kBlock);
      s[i] = *(const float LDS_AS*)(lds + sa + 64 * i);
    }
    auto read_w = [&](int base, int j) {
      wf[j % RING] = read(base + wa + w_row(wn, j) * kBlock);
      if (ROW_SCALES)
        sr[j % 4] =
            *(const f32x4 LDS_AS*)(lds + base + C::X_BYTES + C::W_BYTES + C::S_BYTES + (w_row(wn, j) + 4 * g) * 4);
    };
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) read_w(0, j);
    if (!ROW_SCALES) {
      sb = swp[l.k0 * p.swk];
      if (GATED) sb2 = swp[p.sup + l.k0 * p.swk];
    }

    do {
      const int at = slot * STAGE, nslot = slot + 1 == C::NS ? 0 : slot + 1, nat = nslot * STAGE;
      // products of the two scales
      float sc[C::FM], sc2[GATED ? C::FM : 1];
#pragma unroll
      for (int i = 0; i < C::FM; ++i) {
        sc[i] = ROW_SCALES ? s[i] : s[i] * sb;
        if (GATED) sc2[i] = s[i] * sb2;
      }
      if (!ROW_SCALES && kb + 1 < l.nk) {
        sb = swp[(kb + 1) * p.swk];
        if (GATED) sb2 = swp[p.sup + (kb + 1) * p.swk];
      }
      const Stage next = stage(l, kb + C::NS, lds0 + at, wave);
      auto turn = [&](int j) {
        if (j != C::FN - AHEAD) return;
        // This wave has read all of this stage: once every wave has, and the next
        // stage has landed, the copies of the stage after them may begin.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vm<(C::NS - 2) * LOADS>();
        barrier();
      };
      if constexpr (EXACT) {  // the block's sums on the 16-bit instructions
        f32x4 part[2][C::FM];  // a weight fragment's sums are added while the next one's form
        auto finish = [&](int j) {
#pragma unroll
          for (int i = 0; i < C::FM; ++i) {
            const float f = j >= C::FN / 2 ? sc2[i] : sc[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(part[j % 2][i][r], f, acc[i][j][r]);
          }
        };
        Halves xh[C::FM];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) xh[i] = Halves(xf[i]);
#pragma unroll
        for (int j = 0; j < C::FN; ++j) {
          turn(j);
          const Halves wh(wf[j % RING]);
          read_w(j < C::FN - AHEAD ? at : nat, (j + AHEAD) % C::FN);
          f32x4(&sum)[C::FM] = part[j % 2];
#pragma unroll
          for (int i = 0; i < C::FM; ++i) sum[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int i = 0; i < C::FM; ++i) sum[i] = mfma_f16(wh.v[k], xh[i].v[k], sum[i]);
          if (j == C::FN - 1) {
#pragma unroll
            for (int i = 0; i < C::FM; ++i) {
              xf[i] = read(nat + xa + 16 * i * kBlock);
              s[i] = *(const float LDS_AS*)(lds + nat + sa + 64 * i);
            }
          }
          if (j >= C::FN - AHEAD) {
            const int u = j - (C::FN - AHEAD);
#pragma unroll
            for (int k = u * LOADS / AHEAD; k < (u + 1) * LOADS / AHEAD; ++k) next.unit(k);
          }
          if (j) finish(j - 1);
        }
        finish(C::FN - 1);
      } else {
        f32x4 part[3];
        auto finish = [&](int t) {
          const int i = t % C::FM, j = t / C::FM;
          const f32x4& v = part[t % 3];
          if (ROW_SCALES) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(v[r], sc[i] * sr[j % 4][r], acc[i][j][r]);
          } else {
            const float f = GATED && j >= C::FN / 2 ? sc2[i] : sc[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(v[r], f, acc[i][j][r]);
          }
        };
#pragma unroll
        for (int j = 0; j < C::FN; ++j) {
          turn(j);
#pragma unroll
          for (int i = 0; i < C::FM; ++i) {
            const int t = j * C::FM + i;
            part[t % 3] = mfma(wf[j % RING], xf[i]);
            __builtin_amdgcn_sched_barrier(0);
            if (i == 0) read_w(j < C::FN - AHEAD ? at : nat, (j + AHEAD) % C::FN);
            if (j == C::FN - 1) {  // the next stage's tokens, each as soon as its register is free
              xf[i] = read(nat + xa + 16 * i * kBlock);
              s[i] = *(const float LDS_AS*)(lds + nat + sa + 64 * i);
            }
            if (j >= C::FN - AHEAD) {  // the copies, spread over the steps after the barrier
              constexpr int STEPS = AHEAD * C::FM;
              const int u = t - (C::FN - AHEAD) * C::FM;
#pragma unroll
              for (int k = u * LOADS / STEPS; k < (u + 1) * LOADS / STEPS; ++k) next.unit(k);
            }
            if (t >= 2) finish(t - 2);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        constexpr int T = C::FM * C::FN;
        if (T >= 2) finish(T - 2);
        finish(T - 1);
      }
      slot = nslot;
    } while (++kb < l.nk);
    wait_vm<0>();
    // opaque, or the compiler forms the stores' addresses before the loop and
    // holds (256 x 256: spills) them through it
    int ln = lane;
    asm volatile("" : "+v"(ln));
    store_all(p, lds, acc, m0, m_left, n0, wave, wm, wn, ln & 15, ln >> 4);
  }

  __device__ static __forceinline__ void store_all(const MmArgs& p, char LDS_AS* lds, f32x4 (&acc)[C::FM][C::FN],
                                                   int64_t m0, int m_left, int64_t n0, int wave, int wm, int wn,
                                                   int t16, int g) {
    if (GATED) {
      store_gated(p, lds, acc, m0, m_left, n0, wm, wn, t16, g);
    } else if (EXPERTS) {
      // A slot's results wait in memory for the sum over its token's experts, in FP32: they are
      // parts of that sum.  (As binary16 over a power of two for each wave tile's columns they are
      // half the bytes, and what lay 2^14 below the largest column lost its bits; 4096
      // tokens of 8 experts each, width 2048, took 355 us, 358 to 375 now.)
      store<float>(p, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
    } else if (p.ksplit) {
      MmArgs q = p;
      q.c = p.parts + (int64_t)blockIdx.y * p.M * p.N;
      q.scm = p.N, q.scn = 1, q.bias = nullptr;
      store<float>(q, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
    } else if (p.ctype == F16ACC_TYPE_F16)
      store<f16>(p, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
    else if (p.ctype == F16ACC_TYPE_BF16)
      store<bf16>(p, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
    else
      store<float>(p, lds, acc, m0, m_left, n0, wave, wm, wn, t16, g);
  }

  // The wave's sums plus the bias, rounded once.  A lane's four consecutive
  // columns of one token would go out as 8 bytes in every row of 16: 4096 x 4096 x
  // 128 in bfloat16 took 30 us that way.  So 16 tokens at a time pass through LDS and
  // leave as 16-byte units of whole row pieces (TN columns), at any alignment.
  template <class T>
  __device__ static __forceinline__ void store(const MmArgs& p, char LDS_AS* lds, f32x4 (&acc)[C::FM][C::FN],
                                               int64_t m0, int m_left, int64_t n0, int wave, int wm, int wn, int t16,
                                               int g) {
    const int64_t nw = n0 + wn * C::TN;
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j) {
        const int64_t n = nw + 16 * j + 4 * g;
        f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < p.N) b[r] = (float)((const T*)p.bias)[n + r];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) acc[i][j] += b;
      }
    }
    if (p.scn != 1) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j) {
        const int64_t n = nw + 16 * j + 4 * g;
        const int left = (int)(p.N - n < 4 ? p.N - n : 4);
#pragma unroll
        for (int i = 0; i < C::FM; ++i) {
          const int m = wm * C::TM + 16 * i + t16;
          if (m < m_left) store4<T>((T*)p.c + (m0 + m) * p.scm + n * p.scn, p.scn, left, acc[i][j], false);
        }
      }
      return;
    }
    constexpr int E = 16 / sizeof(T), UNITS = C::TN / E, ROW = C::TN * sizeof(T) + 16;
    static_assert(C::WAVES * 16 * (C::TN * 4 + 16) <= STAGE * C::NS, "staging fits the ring");
    struct __attribute__((packed, aligned(sizeof(T)))) Unit {
      i32x4 v;
    };
    typedef int Four __attribute__((ext_vector_type(sizeof(T))));  // four values
    char LDS_AS* area = lds + wave * 16 * ROW;
    barrier();  // every wave has read its last stage
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
#pragma unroll
      for (int j = 0; j < C::FN; ++j) {
        union {
          T t[4];
          Four v;
        } f;
#pragma unroll
        for (int r = 0; r < 4; ++r) f.t[r] = (T)acc[i][j][r];
        *(Four LDS_AS*)(area + t16 * ROW + (16 * j + 4 * g) * (int)sizeof(T)) = f.v;
      }
      wave_sync();
      const int lane = g * 16 + t16;
#pragma unroll
      for (int k = 0; k < 16 * UNITS / 64; ++k) {
        const int row = (k * 64 + lane) / UNITS, u = (k * 64 + lane) % UNITS;
        const int m = wm * C::TM + 16 * i + row;
        const int64_t n = nw + u * E;
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

  // h = silu(gate) * up of the tile's 128 columns, quantised: they are one block
  // of each token, whose maximum is over the lane groups and the waves beside
  // each other.
  __device__ static __forceinline__ void store_gated(const MmArgs& p, char LDS_AS* lds, f32x4 (&acc)[C::FM][C::FN],
                                                     int64_t m0, int m_left, int64_t n0, int wm, int wn, int t16,
                                                     int g) {
    static_assert(!GATED || C::BN == 2 * kBlock, "a tile is one block of h");
    barrier();  // the stages are free
    uint32_t LDS_AS* most = (uint32_t LDS_AS*)lds;  // [WN][BM]
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < C::FN / 2; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float h = (EXACT ? silu_exact(acc[i][j][r]) : silu(acc[i][j][r])) * acc[i][j + C::FN / 2][r];
          acc[i][j][r] = h;
          m = umax(m, abs_bits(h));
        }
      m = umax(m, (uint32_t)__shfl_xor((int)m, 16));
      m = umax(m, (uint32_t)__shfl_xor((int)m, 32));
      if (g == 0) most[wn * C::BM + wm * C::TM + 16 * i + t16] = m;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < C::FM; ++i) {
      const int m = wm * C::TM + 16 * i + t16;
      uint32_t bits = most[m];
#pragma unroll
      for (int k = 1; k < C::WN; ++k) bits = umax(bits, most[k * C::BM + m]);
      const BlockScale bs = block_scale(bits);
      if (m < m_left) {
#pragma unroll
        for (int j = 0; j < C::FN / 2; ++j)
          *(int*)(p.q + (m0 + m) * p.ldq + n0 + wn * (C::TN / 2) + 16 * j + 4 * g) =
              pack_e4m3(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], bs.inv);
        if (wn == 0 && g == 0) p.sq[n0 / kBlock * p.ldsq + m0 + m] = bs.s;
      }
    }
  }
};

// The splits' sums, in split order, plus the bias, rounded once.
struct FinishArgs {
  const float* parts;
  int64_t M, N, scm, scn;
  int splits;
  const void* bias;
  void* c;
};
template <class T>
__global__ __launch_bounds__(256) void mm_finish_kernel(FinishArgs p) {
  const int64_t size = p.M * p.N;
  if (p.N % 4 == 0) {
    const bool wide = p.scn == 1 && p.scm % 4 == 0 && (uintptr_t)p.c % (4 * sizeof(T)) == 0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 1024) {
      const int64_t m = i / p.N, n = i - m * p.N;
      f32x4 v = *(const f32x4*)(p.parts + i);
      for (int s = 1; s < p.splits; ++s) v += *(const f32x4*)(p.parts + s * size + i);
      if (p.bias) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] += (float)((const T*)p.bias)[n + r];
      }
      store4<T>((T*)p.c + m * p.scm + n * p.scn, p.scn, 4, v, wide);
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256) {
      const int64_t m = i / p.N, n = i - m * p.N;
      float v = p.parts[i];
      for (int s = 1; s < p.splits; ++s) v += p.parts[s * size + i];
      if (p.bias) v += (float)((const T*)p.bias)[n];
      ((T*)p.c)[m * p.scm + n * p.scn] = (T)v;
    }
  }
}

template <class C, bool ROW_SCALES, bool EXPERTS, int EPI>
__global__ __launch_bounds__(C::THREADS, C::OCC) void mm_kernel(MmArgs p) {
  using K = MmKernel<C, ROW_SCALES, EXPERTS, EPI>;
  static_assert(K::STAGE * C::NS <= 160 * 1024, "LDS of a CU");
  __shared__ __align__(1024) char smem[K::STAGE * C::NS];
  K::run(p, (char LDS_AS*)smem);
}

template <class C, bool ROW_SCALES, bool EXPERTS, int EPI>
int launch_mm(const MmArgs& p, int64_t max_tiles_m, hipStream_t stream, int splits = 1) {
  using K = MmKernel<C, ROW_SCALES, EXPERTS, EPI>;
  const int64_t tiles = max_tiles_m * cdiv(p.N, K::BN_OUT);
  if (tiles > 0x7fffffff) return F16ACC_OPS_E_UNSUPPORTED;
  hipLaunchKernelGGL((mm_kernel<C, ROW_SCALES, EXPERTS, EPI>), dim3((uint32_t)tiles, (uint32_t)splits), dim3(C::THREADS),
                     0, stream, p);
  return hip_status();
}

}  // namespace f16ops

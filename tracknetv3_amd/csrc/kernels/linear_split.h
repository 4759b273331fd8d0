// linear_split.h -- fp32 products on the bf16 matrix pipe.
//
// x = x0 + x1 + x2 with x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1), round to nearest even: both differences are exact in fp32 (16 and
// 7 significant bits are left), so the three planes hold x exactly unless a part falls below bf16's 2^-133 (an element is then off by at most 2^-134:
// fp32's relative accuracy holds down to |x| of about 2^-110, measured 9e-6 at 2^-118).  Of the nine products x_p y_q the six
// with p + q <= 2 are summed (fp32 accumulators).  |x1| <= 2^-8 |x| and |x2| <= 2^-16 |x|, so what is left out, x1 y2 + x2 y1 + x2 y2, is at most 2^-23
// of the term and of either sign -- two half steps of fp32 at worst, a tenth of that on average.  Six products at 2.5 PFLOP/s are 417 TFLOP/s against
// the fp32 pipe's 157.
//
// Infinities: inf * (the other's zero low planes) is NaN, and a value beyond bf16's largest rounds to inf.  So if any sum of the workgroup's tile is
// not finite the tile is computed a second time (CAREFUL) with such values kept apart: x0 = the value, truncated instead of rounded if rounding
// overflows, x1 = x2 = 0 for inf / NaN, and inf / NaN taken out of the cross products.  The result is then what fp32 gives.
//
// Layout of a step (32 of the contraction, two fragment halves): the elements pass through registers, because a plane is 11 vector instructions per
// pair to make.  Those stand between the first half's products: while they are issued, the next step's elements are split and stored to the other LDS stage,
// and each register's load for the step after is issued as soon as it is free.  (They add their time to the products' all the same: two register sets
// or a finer interleave changed nothing.)  The barrier lies between the halves: the second half's fragments are in registers by then, the next step's
// first fragments are read under the second half's products.
#pragma once
#include "linear_common.h"

namespace tnv3 {

template <int TM_, int TN_, int WM_, int WN_>
struct LinSplitCfg {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr int NW = WM * WN, NT = NW * 64, BI = TM * 32 * WM, BJ = TN * 32 * WN, BK = 32;
  static constexpr int A_PLANE = BI * BK, B_PLANE = BJ * BK, STAGE = 3 * (A_PLANE + B_PLANE);      // 16-bit elements
  static constexpr int SLABS = NW * kLinSlabFloats * 2;
  static constexpr int LDS = 2 * STAGE > SLABS ? 2 * STAGE : SLABS;
};

__device__ __forceinline__ bool lin_finite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u; }

// two fp32 values -> their packed halves of the three planes
template <bool CAREFUL>
__device__ __forceinline__ void lin_split2(float a, float b, unsigned (&o)[3]) {
  unsigned h = lin_pack2(a, b, LinBf16{});
  if (CAREFUL) {
    const unsigned ua = __builtin_bit_cast(unsigned, a), ub = __builtin_bit_cast(unsigned, b);
    if (lin_finite(a) && (h & 0x7fffu) == 0x7f80u) h = (h & 0xffff0000u) | (ua >> 16);
    if (lin_finite(b) && ((h >> 16) & 0x7fffu) == 0x7f80u) h = (h & 0xffffu) | (ub & 0xffff0000u);
  }
  float ra = a - lin_bits(h << 16), rb = b - lin_bits(h & 0xffff0000u);
  if (CAREFUL) {
    ra = lin_finite(a) ? ra : 0.0f;
    rb = lin_finite(b) ? rb : 0.0f;
  }
  const unsigned m = lin_pack2(ra, rb, LinBf16{});
  o[0] = h;
  o[1] = m;
  o[2] = lin_pack2(ra - lin_bits(m << 16), rb - lin_bits(m & 0xffff0000u), LinBf16{});
}
// a fragment without its infinities and NaNs
__device__ __forceinline__ lin_s8 lin_drop_nonfinite(lin_s8 f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (f[i] & 0x7f80) == 0x7f80 ? (short)0 : f[i];
  return f;
}

// One operand's share of a step in registers: N pieces of 8 consecutive elements per work-item, loaded through a buffer descriptor that ends
// with the operand (beyond it: zeros; a raw buffer's 16-byte access needs 4-byte alignment only and is checked per element).
template <bool KS, int ROWS, int NT>
struct LinSplitLoader {
  static constexpr int BK = 32, N = ROWS * BK / 8 / NT;
  static_assert(N * NT * 8 == ROWS * BK, "whole pieces per work-item");
  float v[N][8];
  unsigned off[N];          // bytes from the operand's first element of the step
  int kpos;                 // k-contiguous: k of the piece's first element within the step
  const char* base;
  long left, step;
  template <class RowOf>
  __device__ __forceinline__ void init(const void* src, long base_el, long end_el, long ld, RowOf row_of, int tid) {
    base = static_cast<const char*>(src) + 4 * base_el;
    left = 4 * (end_el - base_el);
    step = KS ? 4 * BK * ld : 4 * BK;
    kpos = (tid % (BK / 8)) * 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * NT;
      off[i] = KS ? (unsigned)((id / (ROWS / 8)) * (int)(4 * ld) + (id % (ROWS / 8)) * 32) : row_of(id / (BK / 8)) + (unsigned)kpos * 4u;
    }
  }
  __device__ __forceinline__ tnv3_rsrc_t rsrc() const {
    return tnv3_make_rsrc(base, lin_range(left));
  }
  __device__ __forceinline__ void load(tnv3_rsrc_t r, int i) {
    const f32x4 a = lin_buf_load4(r, off[i], 0), b = lin_buf_load4(r, off[i], 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[i][e] = a[e]; v[i][4 + e] = b[e]; }
  }
  __device__ __forceinline__ void advance() { base += step; left -= step; }
  // the step's last elements of the contraction end inside it: what follows them in memory is the next row
  __device__ __forceinline__ void mask(int valid) {
    if (KS) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = kpos + e < valid ? v[i][e] : 0.0f;
  }
  __device__ __forceinline__ unsigned short* slot(unsigned short* tile, int i, int tid) const {
    const int id = tid + i * NT;
    return tile + (KS ? lin_pos_ks(id / (ROWS / 8), id % (ROWS / 8), ROWS) : lin_pos_kc<BK>(id / (BK / 8), id % (BK / 8)));
  }
};

template <class Cfg, bool KSA, bool KSB, bool GATED>
__device__ __forceinline__ void lin_split_product(const LinGemmArgs& p, int block, unsigned short* lds, int& redo) {
  constexpr int TM = Cfg::TM, TN = Cfg::TN, BI = Cfg::BI, BJ = Cfg::BJ, BK = Cfg::BK, NT = Cfg::NT, STAGE = Cfg::STAGE;
  constexpr int A_PLANE = Cfg::A_PLANE, B_PLANE = Cfg::B_PLANE;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / Cfg::WN, wj = wave % Cfg::WN;
  int ti, tj, sp;
  if (!lin_tile(p, block, ti, tj, sp)) return;
  const long i0 = (long)ti * BI, j0 = (long)tj * (GATED ? BJ / 2 : BJ);
  const long kbeg = (long)sp * p.k_per_split, kend = kbeg + p.k_per_split < p.kk ? kbeg + p.k_per_split : p.kk;
  const int steps = kend > kbeg ? (int)((kend - kbeg + BK - 1) / BK) : 0;
  const int tail = (int)((kend - kbeg) - (long)(steps - 1) * BK);           // elements of the last step, 1 .. BK

  f32x16 acc[TM][TN];
  auto pass = [&](auto careful_tag) {
    constexpr bool CAREFUL = decltype(careful_tag)::value;
    LinSplitLoader<KSA, BI, NT> la;
    LinSplitLoader<KSB, BJ, NT> lb;
    constexpr int NA = LinSplitLoader<KSA, BI, NT>::N, NB = LinSplitLoader<KSB, BJ, NT>::N, PAIRS = 4 * (NA + NB), GROUPS = 6;
    la.init(p.a, KSA ? kbeg * p.lda + i0 : i0 * p.lda + kbeg, KSA ? p.kk * p.lda : p.rows_i * p.lda, p.lda,
            [&](int r) { return (unsigned)r * (unsigned)(4 * p.lda); }, tid);
    if (GATED) {
      // tile row r holds weight row (r / H odd ? f : 0) + j0 + (r / 2H) H + r % H, H = TN 16; a wave's 16 rows per piece lie in one half, the
      // same for all its pieces (NT / 4 rows apart), so the jump is in its base
      constexpr int H = TN * 16;
      static_assert(H % 16 == 0 && (NT / 4) % (2 * H) == 0, "a wave's pieces stay within one half");
      lb.init(p.b, (j0 + ((wave * 16 / H) & 1 ? p.f : 0)) * p.ldb + kbeg, p.rows_j * p.ldb, p.ldb,
              [&](int r) { return (unsigned)((r / (2 * H)) * H + r % H) * (unsigned)(4 * p.ldb); }, tid);
    } else {
      lb.init(p.b, KSB ? kbeg * p.ldb + j0 : j0 * p.ldb + kbeg, KSB ? p.kk * p.ldb : p.rows_j * p.ldb, p.ldb,
              [&](int r) { return (unsigned)r * (unsigned)(4 * p.ldb); }, tid);
    }
#pragma unroll
    for (int x = 0; x < TM; ++x)
#pragma unroll
      for (int y = 0; y < TN; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;

    lin_s8 fa[2][3][TM], fb[2][3][TN];
    auto read = [&](const unsigned short* t, int q, int set) {
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) {
#pragma unroll
        for (int x = 0; x < TM; ++x) fa[set][pl][x] = lin_frag<KSA, BK, BI>(t + pl * A_PLANE, wi * TM * 32, x, q, lane);
#pragma unroll
        for (int y = 0; y < TN; ++y) fb[set][pl][y] = lin_frag<KSB, BK, BJ>(t + 3 * A_PLANE + pl * B_PLANE, wj * TN * 32, y, q, lane);
      }
    };
    // group g of six: plane products in the order of their size, smallest first
    auto products = [&](int set, int g) {
      const int pa = g == 0 ? 2 : (g == 2 || g == 3 ? 1 : 0), pb = g == 1 ? 2 : (g == 2 || g == 4 ? 1 : 0);
#pragma unroll
      for (int x = 0; x < TM; ++x)
#pragma unroll
        for (int y = 0; y < TN; ++y) {
          lin_s8 a = fa[set][pa][x], b = fb[set][pb][y];
          if (CAREFUL && g < 5) { a = lin_drop_nonfinite(a); b = lin_drop_nonfinite(b); }
          acc[x][y] = lin_mfma(a, b, acc[x][y], LinBf16{});
        }
    };
    // piece i of the step in registers -> planes in stage t, then its load for the step after
    lin_u4 o[3];
    auto pair = [&](unsigned short* t, int k, tnv3_rsrc_t ra, tnv3_rsrc_t rb) {
      const int i = k >> 2, e = k & 3;
      const bool is_a = i < NA;
      const int ii = is_a ? i : i - NA;
      float x, y;
      if (is_a) { x = la.v[ii < NA ? ii : 0][2 * e]; y = la.v[ii < NA ? ii : 0][2 * e + 1]; }
      else { x = lb.v[ii < NB ? ii : 0][2 * e]; y = lb.v[ii < NB ? ii : 0][2 * e + 1]; }
      unsigned h[3];
      lin_split2<CAREFUL>(x, y, h);
#pragma unroll
      for (int pl = 0; pl < 3; ++pl) o[pl][e] = h[pl];
      if (e == 3) {
        unsigned short* d = is_a ? la.slot(t, ii, tid) : lb.slot(t + 3 * A_PLANE, ii, tid);
#pragma unroll
        for (int pl = 0; pl < 3; ++pl) *reinterpret_cast<lin_u4*>(d + pl * (is_a ? A_PLANE : B_PLANE)) = o[pl];
        if (is_a) la.load(ra, ii < NA ? ii : 0); else lb.load(rb, ii < NB ? ii : 0);
      }
    };
    auto sync = [&]() {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xc07f);            // lgkmcnt(0): this wave's planes are stored, its fragments are in registers
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    };

    {
      const tnv3_rsrc_t ra = la.rsrc(), rb = lb.rsrc();
#pragma unroll
      for (int i = 0; i < NA; ++i) la.load(ra, i);
#pragma unroll
      for (int i = 0; i < NB; ++i) lb.load(rb, i);
      la.advance();
      lb.advance();
      if (steps == 1) { la.mask(tail); lb.mask(tail); }
      const tnv3_rsrc_t na = la.rsrc(), nb = lb.rsrc();
#pragma unroll
      for (int k = 0; k < PAIRS; ++k) pair(lds, k, na, nb);
      la.advance();
      lb.advance();
    }
    sync();
    read(lds, 0, 0);
    for (int s = 0; s < steps; ++s) {
      const unsigned short* t = lds + (s & 1) * STAGE;
      unsigned short* n = lds + (~s & 1) * STAGE;
      // (the last steps store and load as the others do: the stage is not read, the loads end with the operand)
      if (s + 2 == steps) { la.mask(tail); lb.mask(tail); }
      const tnv3_rsrc_t ra = la.rsrc(), rb = lb.rsrc();
      read(t, 1, 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        products(0, g);
#pragma unroll
        for (int k = g * PAIRS / GROUPS; k < (g + 1) * PAIRS / GROUPS; ++k) pair(n, k, ra, rb);
        __builtin_amdgcn_sched_barrier(0);
      }
      la.advance();
      lb.advance();
      sync();
      read(n, 0, 0);                                  // (behind the last step: a stage of this launch, unused)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) products(1, g);
      __builtin_amdgcn_sched_barrier(0);
    }
    sync();
  };
  if (steps > 0) {
    pass(LinFlag<false>{});
    bool bad = false;
#pragma unroll
    for (int x = 0; x < TM; ++x)
#pragma unroll
      for (int y = 0; y < TN; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad |= !lin_finite(acc[x][y][r]);
    if (tid == 0) redo = 0;
    __syncthreads();
    if (bad) redo = 1;
    __syncthreads();
    if (redo) pass(LinFlag<true>{});
  }
  auto put = [&](float* slab, int tm, int left, int right) { lin_put32(acc, slab, tm, left, right, lane); };
  lin_write_out<float, TM, TN, GATED, KSB>(p, put, reinterpret_cast<float*>(lds) + wave * kLinSlabFloats, lane, i0 + wi * TM * 32,
                                      j0 + (long)wj * TN * (GATED ? 16 : 32), sp);
}

template <class Cfg, bool GATED>
__global__ void __launch_bounds__(Cfg::NT, 2) lin_split_kernel(const LinGemmArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned short lds[Cfg::LDS];
  __shared__ int redo;
  lin_split_product<Cfg, false, false, GATED>(p, blockIdx.x, lds, redo);
}
template <class Cfg>
__global__ void __launch_bounds__(Cfg::NT, 2) lin_split_pair_kernel(const LinPairArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned short lds[Cfg::LDS];
  __shared__ int redo;
  const int b = blockIdx.x, c = b - p.blocks_dx, d = c - p.blocks_dw;
  if (c < 0) lin_split_product<Cfg, false, true, false>(p.dx, b, lds, redo);
  else if (d < 0) lin_split_product<Cfg, true, true, false>(p.dw, c, lds, redo);
  else lin_colsum<float, Cfg::NT>(p.sums, static_cast<float*>(p.db), p.sum_rows, p.sum_cols, d, reinterpret_cast<float*>(lds));
}

}  // namespace tnv3

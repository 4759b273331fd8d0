// linear_staged.h -- the products of 16-bit operands whose rows or bases no 16-byte load fits: elements pass through registers on their way to LDS.
// Also the LDS layouts and fragment reads that all the wide products share.
#pragma once
#include "linear_common.h"

namespace tnv3 {

template <int TM_, int TN_, int WM_, int WN_>
struct LinStagedCfg {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;   // 32x32 tiles per wave, waves
  static constexpr int NT = WM * WN * 64, BI = TM * 32 * WM, BJ = TN * 32 * WN, BK = 32;
};

// Position (in 16-bit elements) of 8-element chunk c of row r in an LDS tile.  k-contiguous rows of BK elements: rows 8 apart would share
// their banks, so the chunk index is exchanged with row bits -- a fragment read's eight lanes then cover all banks once.  k-strided tiles are rows of `ld`
// elements; the transposing read takes 4 rows x 32 bytes at a time: row bits move the 32-byte piece.
template <int BK> __device__ __forceinline__ int lin_pos_kc(int r, int c) { return r * BK + ((c ^ (BK == 64 ? (r & 7) : ((r >> 1) & 3))) << 3); }
__device__ __forceinline__ int lin_pos_ks(int k, int c, int ld) { return k * ld + ((c ^ ((k & 3) << 1)) << 3); }

// fragments of one operand: rows base + 32 t + (l & 31), k = 16 s + 8 (l >> 5) + 0..7
template <bool KS, int BK, int ROWS>
__device__ __forceinline__ lin_s8 lin_frag(const unsigned short* tile, int base, int t, int s, int lane) {
  if (!KS) return *reinterpret_cast<const lin_s8*>(tile + lin_pos_kc<BK>(base + 32 * t + (lane & 31), 2 * s + (lane >> 5)));
  const int q = lane & 15, c = ((base + 32 * t) >> 3) + ((lane >> 4) & 1) * 2 + ((q & 3) >> 1);
  const int k = 16 * s + 8 * (lane >> 5) + (q >> 2);
  const unsigned short* p = tile + lin_pos_ks(k, c, ROWS) + (q & 1) * 4;
  const lin_s4 lo = lin_lds_tr4(p), hi = lin_lds_tr4(p + 4 * ROWS);
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One operand's part of a stage: rows base.. of the tile, BK of k, in 8-element chunks held in registers until the buffer is free.
template <class T, bool KS, int ROWS, int NT>
struct LinLoader {
  static constexpr int BK = 32, CHUNKS = ROWS * BK / 8, N = CHUNKS / NT;
  static_assert(CHUNKS % NT == 0, "whole chunks per work-item");
  lin_u4 raw[N];
  template <class RowOf>
  __device__ __forceinline__ void load(const T* src, RowOf row_of, long rows, long ld, long k0, long kend, bool vec, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * NT;
      const int r = KS ? (id % (ROWS / 8)) * 8 : id / (BK / 8), c = KS ? id / (ROWS / 8) : (id % (BK / 8)) * 8;
      const long row = row_of(r), k = k0 + c;
      const long left = KS ? rows - row : kend - k;
      int n = left < 8 ? (left < 0 ? 0 : (int)left) : 8;
      if (KS ? k >= kend : row >= rows) n = 0;
      const unsigned short* h = reinterpret_cast<const unsigned short*>(src + (KS ? k * ld + row : row * ld + k));
      lin_u4 q = {0u, 0u, 0u, 0u};
      if (vec && n == 8) {
        q = *reinterpret_cast<const lin_u4*>(h);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) q[e >> 1] |= (unsigned)h[e] << (16 * (e & 1));
      }
      raw[i] = q;
    }
  }
  __device__ __forceinline__ void store(unsigned short* tile, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * NT;
      *reinterpret_cast<lin_u4*>(tile + (KS ? lin_pos_ks(id / (ROWS / 8), id % (ROWS / 8), ROWS) : lin_pos_kc<BK>(id / (BK / 8), id % (BK / 8)))) = raw[i];
    }
  }
};

template <class Cfg, class T, bool KSA, bool KSB, bool GATED>
__global__ void __launch_bounds__(Cfg::NT) lin_staged_kernel(const LinGemmArgs p) {
  constexpr int TM = Cfg::TM, TN = Cfg::TN, BI = Cfg::BI, BJ = Cfg::BJ, BK = Cfg::BK, NT = Cfg::NT;
  constexpr int STAGE = (BI + BJ) * BK;
  constexpr int SLABS = NT / 64 * kLinSlabFloats * 2;                           // in 16-bit elements
  constexpr int LDS = 2 * STAGE > SLABS ? 2 * STAGE : SLABS;
  __shared__ __attribute__((aligned(16))) unsigned short lds[LDS];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wi = wave / Cfg::WN, wj = wave % Cfg::WN;
  int ti, tj, sp;
  lin_tile(p, ti, tj, sp);
  const long i0 = (long)ti * BI, j0 = (long)tj * (GATED ? BJ / 2 : BJ);
  const long kbeg = (long)sp * p.k_per_split, kend = kbeg + p.k_per_split < p.kk ? kbeg + p.k_per_split : p.kk;
  const int steps = kend > kbeg ? (int)((kend - kbeg + BK - 1) / BK) : 0;
  const T* a = static_cast<const T*>(p.a);
  const T* b = static_cast<const T*>(p.b);

  LinLoader<T, KSA, BI, NT> la;
  LinLoader<T, KSB, BJ, NT> lb;
  auto row_a = [&](int r) -> long { return i0 + r; };
  auto row_b = [&](int r) -> long {
    if (!GATED) return j0 + r;
    constexpr int W = TN * 32, H = TN * 16;              // a wave's columns: H of the gate, then H of the other factor
    const long j = j0 + (long)(r / W) * H + r % H;
    return (r / H) & 1 ? (j < p.f ? p.f + j : p.rows_j) : (j < p.f ? j : p.rows_j);
  };
  auto load = [&](int s) {
    la.load(a, row_a, p.rows_i, p.lda, kbeg + (long)s * BK, kend, p.vec & kLinVecA, tid);
    lb.load(b, row_b, p.rows_j, p.ldb, kbeg + (long)s * BK, kend, p.vec & kLinVecB, tid);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int x = 0; x < TM; ++x)
#pragma unroll
    for (int y = 0; y < TN; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
  if (steps > 0) load(0);
  for (int s = 0; s < steps; ++s) {
    // two stage buffers, one barrier a step: buffer s & 1 was last read in step s - 2, and the barrier of step s - 1 lies in between
    unsigned short* ta = lds + (s & 1) * STAGE;
    unsigned short* tb = ta + BI * BK;
    la.store(ta, tid);
    lb.store(tb, tid);
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
#pragma unroll
    for (int q = 0; q < BK / 16; ++q) {
      lin_s8 fa[TM], fb[TN];
#pragma unroll
      for (int x = 0; x < TM; ++x) fa[x] = lin_frag<KSA, BK, BI>(ta, wi * TM * 32, x, q, lane);
#pragma unroll
      for (int y = 0; y < TN; ++y) fb[y] = lin_frag<KSB, BK, BJ>(tb, wj * TN * 32, y, q, lane);
#pragma unroll
      for (int x = 0; x < TM; ++x)
#pragma unroll
        for (int y = 0; y < TN; ++y) acc[x][y] = lin_mfma(fa[x], fb[y], acc[x][y], T{});
    }
  }
  __syncthreads();
  lin_write_out<T, TM, TN, GATED>(p, acc, reinterpret_cast<float*>(lds) + wave * kLinSlabFloats, lane, i0 + wi * TM * 32,
                                  j0 + (long)wj * TN * (GATED ? 16 : 32), sp);
}

}  // namespace tnv3

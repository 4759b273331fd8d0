// linear_staged.h -- the products whose operands pass through registers on their way to LDS: fp32 (where an element becomes three bf16 planes)
// and 16-bit operands whose rows or bases no 16-byte load fits.
//
// fp32 on the bf16 matrix pipe.  x = x0 + x1 + x2 with x0 = bf16(x), x1 = bf16(x - x0), x2 = bf16(x - x0 - x1), round to nearest even: both
// differences are exact in fp32 (16 and 7 significant bits are left), so the three planes hold x exactly unless a part falls below bf16's
// 2^-133.  Of the nine products x_p y_q the six with p + q <= 2 are summed (fp32 accumulators).  |x1| <= 2^-8 |x| and |x2| <= 2^-16 |x|, so what is
// left out, x1 y2 + x2 y1 + x2 y2, is at most 2^-23 of the term and of either sign -- two half steps of fp32 at worst, a tenth of that on average.
// Six products at 2.5 PFLOP/s are 417 TFLOP/s against the fp32 pipe's 157.
// Infinities: inf * (the other's zero low planes) is NaN, and a value beyond bf16's largest rounds to inf.  So if any sum of the workgroup's tile is
// not finite the tile is computed a second time with the planes of such values kept apart (`careful`): x0 = the value, truncated instead of rounded
// if rounding overflows, x1 = x2 = 0 for inf / NaN, and inf / NaN taken out of the cross products.  The result is then what fp32 gives.
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

__device__ __forceinline__ bool lin_finite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u; }

// eight fp32 values -> their three planes
__device__ __forceinline__ void lin_split8(const float (&x)[8], lin_u4 (&o)[3], bool careful) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
    unsigned h = lin_pack2(a, b, LinBf16{});
    if (careful) {
      const unsigned ua = __builtin_bit_cast(unsigned, a), ub = __builtin_bit_cast(unsigned, b);
      if (lin_finite(a) && (h & 0x7fffu) == 0x7f80u) h = (h & 0xffff0000u) | (ua >> 16);
      if (lin_finite(b) && ((h >> 16) & 0x7fffu) == 0x7f80u) h = (h & 0xffffu) | (ub & 0xffff0000u);
    }
    float ra = a - lin_bits(h << 16), rb = b - lin_bits(h & 0xffff0000u);
    if (careful) {
      ra = lin_finite(a) ? ra : 0.0f;
      rb = lin_finite(b) ? rb : 0.0f;
    }
    const unsigned m = lin_pack2(ra, rb, LinBf16{});
    o[0][i] = h;
    o[1][i] = m;
    o[2][i] = lin_pack2(ra - lin_bits(m << 16), rb - lin_bits(m & 0xffff0000u), LinBf16{});
  }
}
// a fragment without its infinities and NaNs
__device__ __forceinline__ lin_s8 lin_drop_nonfinite(lin_s8 f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (f[i] & 0x7f80) == 0x7f80 ? (short)0 : f[i];
  return f;
}

template <class T> struct LinStage { static constexpr int P = 1; typedef T mfma_t; };
template <> struct LinStage<float> { static constexpr int P = 3; typedef LinBf16 mfma_t; };

// One operand's part of a stage: rows base.. of the tile, BK of k, in 8-element chunks held in registers until the buffer is free.
template <class T, bool KS, int ROWS, int NT>
struct LinLoader {
  static constexpr int BK = 32, CHUNKS = ROWS * BK / 8, N = CHUNKS / NT;
  static_assert(CHUNKS % NT == 0, "whole chunks per work-item");
  float v[sizeof(T) == 4 ? N : 1][8];
  lin_u4 raw[sizeof(T) == 4 ? 1 : N];
  // src: element (0, 0) of the operand; row0: first row, f_jump: rows of the upper half of a wave's columns lie f_jump further on (gated)
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
      const T* p = src + (KS ? k * ld + row : row * ld + k);
      if (sizeof(T) == 4) {
        if (n == 0) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        } else {
          lin_load8<float>(reinterpret_cast<const float*>(p), v[i], vec && n == 8, n);
        }
      } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
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
  }
  __device__ __forceinline__ void store(unsigned short* tile, int plane, bool careful, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * NT;
      unsigned short* d = tile + (KS ? lin_pos_ks(id / (ROWS / 8), id % (ROWS / 8), ROWS) : lin_pos_kc<BK>(id / (BK / 8), id % (BK / 8)));
      if (sizeof(T) == 4) {
        lin_u4 o[3];
        lin_split8(v[i], o, careful);
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<lin_u4*>(d + q * plane) = o[q];
      } else {
        *reinterpret_cast<lin_u4*>(d) = raw[i];
      }
    }
  }
};

template <class Cfg, class T, bool KSA, bool KSB, bool GATED>
__global__ void __launch_bounds__(Cfg::NT) lin_staged_kernel(const LinGemmArgs p) {
  constexpr int TM = Cfg::TM, TN = Cfg::TN, BI = Cfg::BI, BJ = Cfg::BJ, BK = Cfg::BK, NT = Cfg::NT, P = LinStage<T>::P;
  constexpr int A_PLANE = BI * BK, B_PLANE = BJ * BK, STAGE = P * (A_PLANE + B_PLANE);
  constexpr int SLABS = NT / 64 * kLinSlabFloats * 2;                           // in 16-bit elements
  constexpr int LDS = 2 * STAGE > SLABS ? 2 * STAGE : SLABS;
  typedef typename LinStage<T>::mfma_t M;
  __shared__ __attribute__((aligned(16))) unsigned short lds[LDS];
  __shared__ int redo;

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
  bool careful = false;
  for (;;) {
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
      unsigned short* tb = ta + P * A_PLANE;
      la.store(ta, A_PLANE, careful, tid);
      lb.store(tb, B_PLANE, careful, tid);
      __syncthreads();
      if (s + 1 < steps) load(s + 1);
#pragma unroll
      for (int q = 0; q < BK / 16; ++q) {
        lin_s8 fa[P][TM], fb[P][TN];
#pragma unroll
        for (int pl = 0; pl < P; ++pl) {
#pragma unroll
          for (int x = 0; x < TM; ++x) fa[pl][x] = lin_frag<KSA, BK, BI>(ta + pl * A_PLANE, wi * TM * 32, x, q, lane);
#pragma unroll
          for (int y = 0; y < TN; ++y) fb[pl][y] = lin_frag<KSB, BK, BJ>(tb + pl * B_PLANE, wj * TN * 32, y, q, lane);
        }
        if (P == 3) {
          // smallest products first; planes (0, 0) last
          auto mm = [&](int pa, int pb) {
#pragma unroll
            for (int x = 0; x < TM; ++x)
#pragma unroll
              for (int y = 0; y < TN; ++y) acc[x][y] = lin_mfma(fa[pa][x], fb[pb][y], acc[x][y], M{});
          };
          if (careful) {
            lin_s8 ka[TM], kb[TN];
#pragma unroll
            for (int x = 0; x < TM; ++x) { ka[x] = fa[0][x]; fa[0][x] = lin_drop_nonfinite(ka[x]); }
#pragma unroll
            for (int y = 0; y < TN; ++y) { kb[y] = fb[0][y]; fb[0][y] = lin_drop_nonfinite(kb[y]); }
            mm(2 % P, 0); mm(0, 2 % P); mm(1 % P, 1 % P); mm(1 % P, 0); mm(0, 1 % P);
#pragma unroll
            for (int x = 0; x < TM; ++x) fa[0][x] = ka[x];
#pragma unroll
            for (int y = 0; y < TN; ++y) fb[0][y] = kb[y];
          } else {
            mm(2 % P, 0); mm(0, 2 % P); mm(1 % P, 1 % P); mm(1 % P, 0); mm(0, 1 % P);
          }
          mm(0, 0);
        } else {
#pragma unroll
          for (int x = 0; x < TM; ++x)
#pragma unroll
            for (int y = 0; y < TN; ++y) acc[x][y] = lin_mfma(fa[0][x], fb[0][y], acc[x][y], M{});
        }
      }
    }
    __syncthreads();
    if (P == 1 || careful) break;
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
    if (!redo) break;
    careful = true;
    __syncthreads();
  }
  lin_write_out<T, TM, TN, GATED>(p, acc, reinterpret_cast<float*>(lds) + wave * kLinSlabFloats, lane, i0 + wi * TM * 32,
                                  j0 + (long)wj * TN * (GATED ? 16 : 32), sp);
}

}  // namespace tnv3

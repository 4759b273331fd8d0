// linear_rows.h -- forward products of few rows (single positions of a stream, small batches): bound by reading the weight once.
//
// A workgroup takes 16 weight rows (gated: 16 of the gate and the same 16 of the other factor) against all rows of x; its NW waves share the
// contraction, 128 bytes of every row per wave in turn, and join their sums through LDS in a fixed order.  Operands go from memory straight into MFMA
// fragments (16x16x32 for 16-bit types, 16x16x4 for fp32): each weight element is used once, so there is nothing for LDS to share, and x is small
// enough to stay in L2.  Each lane's 16-byte loads need no alignment beyond the element's: odd widths run at the same speed.  fp32 stays on the fp32
// matrix pipe -- its 157 TFLOP/s are far above what the weight's bytes allow here.
// Four blocks of loads are issued before the first is used (96 of the 128 registers that 16 waves per CU leave each), so that a CU has
// 64 KB and more in flight.
#pragma once
#include "linear_common.h"

namespace tnv3 {

#ifndef TNV3_EMU
typedef unsigned lin_u4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, LinBf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf8, a), __builtin_bit_cast(lin_bf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, LinF16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_h8, a), __builtin_bit_cast(lin_h8, b), c, 0, 0, 0);
}
#else
typedef unsigned lin_u4_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, LinBf16) {
  return emu_mfma_16x16x32(__builtin_bit_cast(lin_s8, a), __builtin_bit_cast(lin_s8, b), c, emu_bf16_up);
}
__device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, LinF16) {
  return emu_mfma_16x16x32(__builtin_bit_cast(lin_s8, a), __builtin_bit_cast(lin_s8, b), c, emu_f16_up);
}
#endif
// fp32: lane l's four k values are 4 (l >> 4) + 0..3 of 16; product e takes k = e, 4 + e, 8 + e, 12 + e of both operands
__device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, float) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(lin_bits(a[e]), lin_bits(b[e]), c, 0, 0, 0);
  return c;
}

// 16 bytes' elements at p: those from `from` on are kept, the others become 0
template <class T> __device__ __forceinline__ lin_u4 lin_keep_from(lin_u4 q, int from) {
  if (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = e >= from ? q[e] : 0u;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] &= (2 * e >= from ? 0xffffu : 0u) | (2 * e + 1 >= from ? 0xffff0000u : 0u);
  }
  return q;
}
// the first n of 16 bytes' elements, the others 0; one by one, `row` being an address that may be read in any case
template <class T> __device__ __forceinline__ lin_u4 lin_load_first(const T* row, const T* p, int n) {
  constexpr int EL = 16 / (int)sizeof(T);
  lin_u4 q = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < EL; ++e) {
    const T* at = e < n ? p + e : row;
    const unsigned v = sizeof(T) == 4 ? *reinterpret_cast<const unsigned*>(at) : (unsigned)*reinterpret_cast<const unsigned short*>(at);
    if (sizeof(T) == 4) q[e % 4] = e < n ? v : 0u;
    else q[e / 2] |= (e < n ? v : 0u) << (16 * (e & 1));
  }
  return q;
}

template <class T, int MT, int NW, bool GATED>
__global__ void __launch_bounds__(NW * 64) lin_rows_kernel(const LinGemmArgs p) {
  constexpr int EL = 16 / (int)sizeof(T), BLK = 8 * EL, G = GATED ? 2 : 1, U = MT * G >= 4 ? 1 : (MT * G == 2 ? 2 : 4);
  __shared__ __attribute__((aligned(16))) float red[NW][G][MT][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kq = (lane >> 4) * EL;
  const long n0 = (long)blockIdx.x * 16, nout = GATED ? p.f : p.rows_j;

  const T* wp[G];
  const T* xp[MT];
  // rows beyond the last repeat it: their results are not written
  const long wr = n0 + r16 < nout ? n0 + r16 : nout - 1;
#pragma unroll
  for (int g = 0; g < G; ++g) wp[g] = static_cast<const T*>(p.b) + (wr + (g ? p.f : 0)) * p.ldb + kq;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const long xr = 16 * m + r16 < p.rows_i ? 16 * m + r16 : p.rows_i - 1;
    xp[m] = static_cast<const T*>(p.a) + xr * p.lda + kq;
  }
  f32x4 acc[G][MT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  const int nfull = (int)(p.kk / BLK), tail = (int)(p.kk % BLK);
  auto run = [&](int b, auto count) {
    constexpr int C = decltype(count)::value;
    lin_u4 w[C][2][G], x[C][2][MT];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long k = (long)(b + c * NW) * BLK + h * 4 * EL;
#pragma unroll
        for (int g = 0; g < G; ++g) w[c][h][g] = *reinterpret_cast<const lin_u4_any*>(wp[g] + k);
#pragma unroll
        for (int m = 0; m < MT; ++m) x[c][h][m] = *reinterpret_cast<const lin_u4_any*>(xp[m] + k);
      }
    __builtin_amdgcn_sched_barrier(0);           // all loads of the blocks are issued before the first product
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[g][m] = lin_mfma16(w[c][h][g], x[c][h][m], acc[g][m], T{});
  };
  int b = wave;
  for (; b + (U - 1) * NW < nfull; b += U * NW) run(b, LinCount<U>{});
  for (; b < nfull; b += NW) run(b, LinCount<1>{});
  if (tail && nfull % NW == wave) {
    // what whole blocks leave over: the row's last block, without the elements that were summed already; rows shorter than a block: one by one
    const int skip = (int)p.kk - BLK;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      auto part = [&](const T* lane_row) -> lin_u4 {
        if (nfull) return lin_keep_from<T>(*reinterpret_cast<const lin_u4_any*>(lane_row + skip + h * 4 * EL), BLK - tail - h * 4 * EL - kq);
        return lin_load_first<T>(lane_row - kq, lane_row + h * 4 * EL, tail - h * 4 * EL - kq);
      };
      lin_u4 x[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m] = part(xp[m]);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const lin_u4 w = part(wp[g]);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[g][m] = lin_mfma16(w, x[m], acc[g][m], T{});
      }
    }
  }
  // D register r: weight row 4 (lane >> 4) + r, x row lane & 15
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<f32x4*>(&red[wave][g][m][r16 * 16 + (lane >> 4) * 4]) = acc[g][m];
  __syncthreads();
  for (int idx = tid; idx < MT * 256; idx += NW * 64) {
    const long i = idx >> 4, j = n0 + (idx & 15);
    if (i >= p.rows_i || j >= nout) continue;
    float v = 0.0f, u = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += (&red[w][0][0][0])[idx];
    if (GATED) {
#pragma unroll
      for (int w = 0; w < NW; ++w) u += (&red[w][G - 1][0][0])[idx];
    }
    const T* bias = static_cast<const T*>(p.bias);
    constexpr bool FAST = sizeof(T) == 2;
    if (bias) {
      v += lin_up(bias[j]);
      if (GATED) u += lin_up(bias[p.f + j]);
    }
    if (GATED) {
      if (p.pre) {
        static_cast<float*>(p.pre)[i * p.rows_j + j] = v;
        static_cast<float*>(p.pre)[i * p.rows_j + p.f + j] = u;
      }
      lin_down(lin_act1<FAST>(v, p.act) * u, static_cast<T*>(p.out)[i * p.f + j]);
    } else {
      const long o = i * p.rows_j + j;
      if (p.pre) lin_down(v, static_cast<T*>(p.pre)[o]);
      v = lin_act1<FAST>(v, p.act);
      if (p.res) v += lin_up(static_cast<const T*>(p.res)[o]);
      lin_down(v, static_cast<T*>(p.out)[o]);
    }
  }
}

}  // namespace tnv3

// linear_rows.h -- forward products of few rows (single positions of a stream, small batches): bound by reading the weight once, beyond about 32 rows by
// reading x once per 16 weight rows.
//
// A workgroup takes 16 weight rows (gated: 16 of the gate and the same 16 of the other factor) against all rows of x; its NW waves share the
// contraction, one block of 128 bytes per row each in turn, and join their sums through LDS in a fixed order.  A block goes through registers and a
// piece of LDS of the wave's own (no barrier): 8 lanes load a row's 128 bytes, which the fragment reads (16x16x32 MFMA for 16-bit types, 16x16x4 for
// fp32) then take apart.  Loaded straight into fragments, 16 neighbouring lanes would name 16 different cache lines and the CU's address path would
// be the bound (16 bytes per clock: 1 x 4096 -> 8192 in bf16 14.0 us, 64 rows 37.9 us).  The 16-byte loads need no alignment beyond the element's: odd
// widths take the same path.  fp32 stays on the fp32 matrix pipe, whose rate is far above what the weight's bytes allow here.
// U blocks of loads are issued before the first is used, and a block's registers are loaded again as soon as they are free.
#pragma once
#include "linear_common.h"

namespace tnv3 {

template <class T> __device__ __forceinline__ f32x4 lin_mfma16(lin_u4 a, lin_u4 b, f32x4 c, T) {
  return lin_mfma16(__builtin_bit_cast(lin_s8, a), __builtin_bit_cast(lin_s8, b), c, T{});
}
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
  constexpr int EL = 16 / (int)sizeof(T), BLK = 8 * EL, G = GATED ? 2 : 1, U = MT * G == 1 ? 4 : (MT * G < 8 ? 2 : 1);
  constexpr int WROWS = 16 * G, ROWS = WROWS + 16 * MT, NWL = WROWS / 8, NL = ROWS / 8;        // staged rows; loads (8 rows each) per block
  constexpr int STAGE = NW * ROWS * 32, RED = NW * G * MT * 256;                               // floats
  __shared__ __attribute__((aligned(1024))) float lds[STAGE > RED ? STAGE : RED];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15;
  const int lr = lane >> 3, piece = lane & 7;
  const long n0 = (long)blockIdx.x * 16, nout = GATED ? p.f : p.rows_j;
  float* stage = lds + wave * ROWS * 32;

  // the lane's 16 bytes of each load: row 8 i + lane / 8 (weight rows, then x rows; beyond the last: the last again, results not written), piece
  // lane & 7.  Groups of 8 x rows that do not exist are not loaded at all.
  unsigned off[NL];                                   // bytes from the uniform base of the row group (below 64 rows x 2^20 x 4)
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int r = (i < NWL ? i & 1 : i - NWL) * 8 + lr;
    const long last = (i < NWL ? nout - n0 : p.rows_i) - 1;
    off[i] = (unsigned)(r < last ? r : last) * (unsigned)(sizeof(T) * (i < NWL ? p.ldb : p.lda)) + piece * 16;
  }
  const char* base[3] = {reinterpret_cast<const char*>(static_cast<const T*>(p.b) + n0 * p.ldb),
                         reinterpret_cast<const char*>(static_cast<const T*>(p.b) + (n0 + p.f) * p.ldb), static_cast<const char*>(p.a)};
  auto src = [&](int i) -> const char* { return base[i < NWL ? i >> 1 : 2]; };
  const int xgroups = (int)((p.rows_i + 7) / 8);
  f32x4 acc[G][MT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[g][m] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  lin_u4 v[U][NL];
  auto load = [&](int c, int t) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (i < NWL || i - NWL < xgroups) v[c][i] = *reinterpret_cast<const lin_u4_any*>(src(i) + (long)t * 128 + off[i]);
  };
  auto put = [&](int c) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (i < NWL || i - NWL < xgroups) *reinterpret_cast<lin_u4*>(stage + (8 * i + lr) * 32 + ((piece ^ lr) << 2)) = v[c][i];
  };
  auto use = [&]() {
    lin_wave_sync();
    lin_u4 f[2][ROWS / 16];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < ROWS / 16; ++q)
        f[h][q] = *reinterpret_cast<const lin_u4*>(stage + (16 * q + r16) * 32 + ((((lane >> 4) + 4 * h) ^ (r16 & 7)) << 2));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[g][m] = lin_mfma16(f[h][g], f[h][G + m], acc[g][m], T{});
    lin_wave_sync();
  };
  const int nfull = (int)(p.kk / BLK), tail = (int)(p.kk % BLK);
  const int mine = nfull > wave ? (nfull - wave + NW - 1) / NW : 0;        // this wave's whole blocks: wave, wave + NW, ..
  int t = wave, left = mine;
  if (left >= U) {
#pragma unroll
    for (int c = 0; c < U; ++c) load(c, t + c * NW);
    t += U * NW;
    left -= U;
    for (; left >= U; left -= U, t += U * NW) {
#pragma unroll
      for (int c = 0; c < U; ++c) {
        put(c);
        load(c, t + c * NW);
        use();
      }
    }
#pragma unroll
    for (int c = 0; c < U; ++c) {
      put(c);
      use();
    }
  }
  if (left > 0) {                                     // fewer than U blocks: all their loads first
#pragma unroll
    for (int c = 0; c < U - 1; ++c)
      if (c < left) load(c, t + c * NW);
#pragma unroll
    for (int c = 0; c < U - 1; ++c)
      if (c < left) {
        put(c);
        use();
      }
  }
  if (tail && nfull % NW == wave) {
    // what whole blocks leave over: the row's last block, without the elements that were summed already; rows shorter than a block: one by one
    const long skip = (p.kk - BLK) * (long)sizeof(T);
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (i < NWL || i - NWL < xgroups)
        v[0][i] = nfull ? lin_keep_from<T>(*reinterpret_cast<const lin_u4_any*>(src(i) + skip + off[i]), BLK - tail - piece * EL)
                        : lin_load_first<T>(reinterpret_cast<const T*>(src(i) + (off[i] - piece * 16)), reinterpret_cast<const T*>(src(i) + off[i]),
                                            tail - piece * EL);
    put(0);
    use();
  }
  __syncthreads();                                    // every wave is done with its stage: the sums take the same LDS
  float(*red)[G][MT][256] = reinterpret_cast<float(*)[G][MT][256]>(lds);
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
      if (p.pre) lin_down(lin_keep_positive<T>(v), static_cast<T*>(p.pre)[o]);
      v = lin_act1<FAST>(v, p.act);
      if (p.res) v += lin_up(static_cast<const T*>(p.res)[o]);
      lin_down(v, static_cast<T*>(p.out)[o]);
    }
  }
}

}  // namespace tnv3

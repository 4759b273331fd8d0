// linear_grad.h -- the element-wise part of the position-wise layers' backward passes.
//   linear  dz = dy act'(z)                                       gated  dz = [dh u act'(g) | dh act(g)],  z = [g | u]
// The gated layer's z is kept in fp32: rounded to 16 bits, its two factors' errors enter both halves of dz and double the gradients' distance from the
// exact ones behind a chain of layers (measured: 3.4e-3 of the weight gradient's norm in bf16, a single rounding being 1.7e-3).  The linear layer's z is
// kept in the type: it enters through act' alone and takes the weight gradient from 2.35e-3 to 2.41e-3 off (bf16, any of the smooth activations, dz's and
// the result's rounding included), where fp32 would write and read 2 more bytes per element.  dz is rounded to the type, once: it is an operand of both
// products on the matrix pipe, and a second plane for what the rounding drops would double them (1570 of the 1720 us of a training step of an
// 8192 x 2048 -> 2 x 5504 -> 2048 block).
// And the bias gradient, the column sums of dz.  Bound by memory: dy and z are read and dz is written once, in 16-byte pieces.  A workgroup takes 256
// columns (32 work-items of 8) and every 8th row of its row block per work-item; its column sums are joined through LDS and written as
// partial sums [row block][columns], which lin_colsum adds in order: no atomics, the same bits from run to run.
#pragma once
#include "linear_common.h"

namespace tnv3 {

struct LinDzArgs {
  const void* dy;        // [rows][n]
  const void* pre;       // [rows][n], gated [rows][2 n] in fp32; null: no activation, only the column sums are wanted
  void* dz;              // [rows][ld_dz] of which n / 2 n columns hold dz and the others become 0; null with pre
  int ld_dz;
  float* part;           // [row blocks][n] / [..][2 n], or null: no bias
  long rows;
  int n, act, rows_per_block;
};

template <class T, bool GATED>
__global__ void __launch_bounds__(256) lin_dz_kernel(const LinDzArgs p) {
  constexpr bool FAST = sizeof(T) == 2;
  __shared__ float red[GATED ? 2 : 1][8][256 + 8];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int jt = (p.n + 255) / 256, jb = blockIdx.x % jt;
  const long rb = blockIdx.x / jt;
  const int j = jb * 256 + tx * 8, n = p.n - j < 8 ? p.n - j : 8;
  const bool vec = n == 8;
  const long r0 = rb * p.rows_per_block, r1 = r0 + p.rows_per_block < p.rows ? r0 + p.rows_per_block : p.rows;
  const int ldz = GATED ? 2 * p.n : p.n;
  float s0[8], s1[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s0[e] = s1[e] = 0.0f;
  if (n > 0) {
    for (long r = r0 + ty; r < r1; r += 8) {
      float d[8], g[8], u[8];
      lin_load8<T>(static_cast<const T*>(p.dy) + r * p.n + j, d, vec, n);
      if (p.pre) {
        T* o = static_cast<T*>(p.dz) + r * p.ld_dz + j;
        if (GATED) {
          const float* z = static_cast<const float*>(p.pre) + r * ldz + j;
          lin_load8<float>(z, g, vec, n);
          lin_load8<float>(z + p.n, u, vec, n);
        } else {
          lin_load8<T>(static_cast<const T*>(p.pre) + r * ldz + j, g, vec, n);
        }
        // the switch outside of the eight elements' loop; the column sums take dz before it is rounded to T
#define TNV3_LIN_DZ_CASE(A)                                              \
  case A:                                                                \
    _Pragma("unroll") for (int e = 0; e < 8; ++e) {                      \
      float av, dv;                                                      \
      lin_act_grad1<FAST>(g[e], A, av, dv);                              \
      if (GATED) { g[e] = d[e] * u[e] * dv; u[e] = d[e] * av; }          \
      else g[e] = d[e] * dv;                                             \
    }                                                                    \
    break;
        switch (p.act) {
          TNV3_LIN_DZ_CASE(kActLeaky) TNV3_LIN_DZ_CASE(kActSigmoid) TNV3_LIN_DZ_CASE(kActRelu) TNV3_LIN_DZ_CASE(kActSilu)
          TNV3_LIN_DZ_CASE(kActGelu) TNV3_LIN_DZ_CASE(kActGeluTanh)
          default:
            TNV3_LIN_DZ_CASE(kActNone)
        }
#undef TNV3_LIN_DZ_CASE
        lin_store8<T>(o, g, vec, n);
        if (GATED) lin_store8<T>(o + p.n, u, vec, n);
        if (j + 8 >= p.n) {                                // the last columns' work-item clears what the row is padded with
          T* end = static_cast<T*>(p.dz) + r * p.ld_dz;
          for (int c = ldz; c < p.ld_dz; ++c) end[c] = T{};
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) { s0[e] += g[e]; if (GATED) s1[e] += u[e]; }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) s0[e] += d[e];
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    red[0][ty][tx * 8 + e] = s0[e];
    if (GATED) red[GATED ? 1 : 0][ty][tx * 8 + e] = s1[e];
  }
  __syncthreads();
  const int c = threadIdx.x, col = jb * 256 + c;
  if (col >= p.n) return;
#pragma unroll
  for (int h = 0; h < (GATED ? 2 : 1); ++h) {
    float s = 0.0f;
#pragma unroll
    for (int y = 0; y < 8; ++y) s += red[h][y][c];
    p.part[rb * ldz + h * p.n + col] = s;
  }
}

}  // namespace tnv3

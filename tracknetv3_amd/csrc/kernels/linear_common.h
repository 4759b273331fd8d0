// linear_common.h -- what the position-wise products share (linear, gated_linear and their backward passes): element types, the
// MFMA fragments, the activations with their derivatives, and the write-out of a workgroup's tile.
//
// Every product is C(i, j) = sum_k A(i, k) B(j, k) with fp32 accumulators:
//   forward          i = row m of x,      j = output column n,  k = input column:  A = x,   B = W        both k-contiguous
//   gradient of x    i = row m,           j = input column,     k = output column: A = dz,  B = W^T      B strided in k
//   gradient of W    i = output column,   j = input column,     k = row m:         A = dz^T, B = x^T     both strided in k
// MFMA 32x32x16 (the fp32 products' planes): lane l supplies A[l & 31][8 (l >> 5) + 0..7] and B[l & 31][the same k]; accumulator register r of lane l
// is C[(r & 3) + 8 (r >> 2) + 4 (l >> 5)][l & 31].  16x16x32 (16-bit tensors): A[l & 15][8 (l >> 4) + 0..7], B likewise; register r of lane l is
// C[4 (l >> 4) + r][l & 15].
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "conv3x3_mfma.h"

namespace tnv3 {

typedef short lin_s8 __attribute__((ext_vector_type(8)));
typedef short lin_s4 __attribute__((ext_vector_type(4)));
typedef unsigned lin_u4 __attribute__((ext_vector_type(4)));
// in memory: rows of odd widths start anywhere, and the hardware's 16-byte global accesses need no alignment beyond the element's
typedef unsigned lin_u4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef float lin_f4_any __attribute__((ext_vector_type(4), aligned(4)));

template <bool V> struct LinFlag { static constexpr bool value = V; };

struct LinBf16 { unsigned short v; };
struct LinF16 { unsigned short v; };

enum { kLinF32 = 0, kLinBf16 = 1, kLinF16 = 2 };
enum { kActNone = 0, kActLeaky = 1, kActSigmoid = 2, kActRelu = 3, kActSilu = 4, kActGelu = 5, kActGeluTanh = 6, kActCount = 7 };

#ifndef TNV3_EMU
typedef __bf16 lin_bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 lin_h8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x16 lin_mfma(lin_s8 a, lin_s8 b, f32x16 c, LinBf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(lin_bf8, a), __builtin_bit_cast(lin_bf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 lin_mfma(lin_s8 a, lin_s8 b, f32x16 c, LinF16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(lin_h8, a), __builtin_bit_cast(lin_h8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lin_mfma16(lin_s8 a, lin_s8 b, f32x4 c, LinBf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lin_bf8, a), __builtin_bit_cast(lin_bf8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 lin_mfma16(lin_s8 a, lin_s8 b, f32x4 c, LinF16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(lin_h8, a), __builtin_bit_cast(lin_h8, b), c, 0, 0, 0);
}
// Transposing LDS read: within each group of 16 lanes, lane q's address names 4 elements of row q >> 2 (columns 4 (q & 3) ..), and lane q
// receives column q of the four rows.
__device__ __forceinline__ lin_s4 lin_lds_tr4(const unsigned short* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) lin_s4*)p);
}
// two fp32 -> two 16-bit values, round to nearest even (low half: a)
__device__ __forceinline__ unsigned lin_pack2(float a, float b, LinBf16) {
  typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, bf2));
}
__device__ __forceinline__ unsigned lin_pack2(float a, float b, LinF16) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, (h2){(_Float16)a, (_Float16)b});
}
__device__ __forceinline__ float lin_f16_up(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ void lin_wave_sync() { __builtin_amdgcn_wave_barrier(); }
// A store of 16 bytes reads its registers over several clocks: they stay unwritten for two wait states (see tnv3_buf_store_f4).
__device__ __forceinline__ void lin_store_hold(lin_u4 q) { asm volatile("s_nop 1" : : "v"(q)); }
// four fp32 at base + voffset + soffset, each checked against the descriptor's range (beyond it: 0)
__device__ __forceinline__ f32x4 lin_buf_load4(tnv3_rsrc_t r, unsigned voffset, unsigned soffset) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(voffset + soffset), 0, 0));
}
#else
__device__ __forceinline__ f32x16 lin_mfma(lin_s8 a, lin_s8 b, f32x16 c, LinBf16) { return emu_mfma_32x32x16(a, b, c, emu_bf16_up); }
__device__ __forceinline__ f32x16 lin_mfma(lin_s8 a, lin_s8 b, f32x16 c, LinF16) { return emu_mfma_32x32x16(a, b, c, emu_f16_up); }
__device__ __forceinline__ f32x4 lin_mfma16(lin_s8 a, lin_s8 b, f32x4 c, LinBf16) { return emu_mfma_16x16x32(a, b, c, emu_bf16_up); }
__device__ __forceinline__ f32x4 lin_mfma16(lin_s8 a, lin_s8 b, f32x4 c, LinF16) { return emu_mfma_16x16x32(a, b, c, emu_f16_up); }
__device__ __forceinline__ lin_s4 lin_lds_tr4(const unsigned short* p) { return emu_lds_tr4(p); }
__device__ __forceinline__ unsigned lin_pack2(float a, float b, LinBf16) { return (unsigned)emu_bf16_dn(a) | (unsigned)emu_bf16_dn(b) << 16; }
__device__ __forceinline__ unsigned lin_pack2(float a, float b, LinF16) { return (unsigned)emu_f16_dn(a) | (unsigned)emu_f16_dn(b) << 16; }
__device__ __forceinline__ float lin_f16_up(unsigned short h) { return emu_f16_up(h); }
__device__ __forceinline__ void lin_wave_sync() { emu::wave_barrier(); }
__device__ __forceinline__ void lin_store_hold(lin_u4) {}
__device__ __forceinline__ f32x4 lin_buf_load4(tnv3_rsrc_t r, unsigned voffset, unsigned soffset) {
  f32x4 v;
  for (int e = 0; e < 4; ++e) {
    const unsigned long long o = (unsigned long long)voffset + soffset + 4 * e;
    float f = 0.0f;
    if (o + 4 <= r.num_records) memcpy(&f, r.base + o, 4);
    v[e] = f;
  }
  return v;
}
#endif

__device__ __forceinline__ float lin_bits(unsigned u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ float lin_up(LinBf16 h) { return lin_bits((unsigned)h.v << 16); }
__device__ __forceinline__ float lin_up(LinF16 h) { return lin_f16_up(h.v); }
__device__ __forceinline__ float lin_up(float f) { return f; }
__device__ __forceinline__ void lin_down(float f, LinBf16& o) { o.v = (unsigned short)lin_pack2(f, f, LinBf16{}); }
__device__ __forceinline__ void lin_down(float f, LinF16& o) { o.v = (unsigned short)lin_pack2(f, f, LinF16{}); }
__device__ __forceinline__ void lin_down(float f, float& o) { o = f; }

// A pre-activation as a backward pass takes it: rounded to T, but no positive value to 0 -- in fp16 those below 2^-25 would be, and ReLU's derivative at 0
// is another one.
template <class T> __device__ __forceinline__ float lin_keep_positive(float z) { return z; }
template <> __device__ __forceinline__ float lin_keep_positive<LinF16>(float z) {
  return __builtin_bit_cast(unsigned, z) - 1u < 0x337fffffu ? 0x1p-24f : z;          // 0 < z < 2^-24, in one comparison of the bits
}

// ---- eight consecutive elements <-> fp32.  vec: all eight exist; else the first `n` one by one (the rest 0).
__device__ __forceinline__ void lin_unpack8(lin_u4 q, float (&v)[8], LinBf16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = lin_bits(q[i] << 16); v[2 * i + 1] = lin_bits(q[i] & 0xffff0000u); }
}
__device__ __forceinline__ void lin_unpack8(lin_u4 q, float (&v)[8], LinF16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = lin_f16_up((unsigned short)(q[i] & 0xffffu)); v[2 * i + 1] = lin_f16_up((unsigned short)(q[i] >> 16)); }
}
// from the registers of a 16-byte load (fp32: two)
template <class T> __device__ __forceinline__ void lin_unpack8(const lin_u4 (&q)[1], float (&v)[8], T) { lin_unpack8(q[0], v, T{}); }
__device__ __forceinline__ void lin_unpack8(const lin_u4 (&q)[2], float (&v)[8], float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = lin_bits(q[0][i]); v[4 + i] = lin_bits(q[1][i]); }
}
template <class T> __device__ __forceinline__ void lin_load8(const T* p, float (&v)[8], bool vec, int n) {
  if (vec) { lin_unpack8(*reinterpret_cast<const lin_u4_any*>(p), v, T{}); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? lin_up(p[i]) : 0.0f;
}
template <> __device__ __forceinline__ void lin_load8<float>(const float* p, float (&v)[8], bool vec, int n) {
  if (vec) {
    const f32x4 a = reinterpret_cast<const lin_f4_any*>(p)[0], b = reinterpret_cast<const lin_f4_any*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
}
template <class T> __device__ __forceinline__ void lin_store8(T* p, const float (&v)[8], bool vec, int n) {
  if (vec) {
    lin_u4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = lin_pack2(v[2 * i], v[2 * i + 1], T{});
    *reinterpret_cast<lin_u4_any*>(p) = q;
    lin_store_hold(q);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) lin_down(v[i], p[i]);
}
template <> __device__ __forceinline__ void lin_store8<float>(float* p, const float (&v)[8], bool vec, int n) {
  if (vec) {
    const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    reinterpret_cast<lin_f4_any*>(p)[0] = a;
    reinterpret_cast<lin_f4_any*>(p)[1] = b;
    lin_store_hold(__builtin_bit_cast(lin_u4, a));
    lin_store_hold(__builtin_bit_cast(lin_u4, b));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = v[i];
}

template <class T> __device__ __forceinline__ void lin_store_pre8(T* p, const float (&v)[8], bool vec, int n) {
  float z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = lin_keep_positive<T>(v[i]);
  lin_store8<T>(p, z, vec, n);
}

// ---- activations.  FAST (16-bit outputs): hardware exp2 and reciprocal, each within about 2^-23; the exponential's argument x carries |x| 2^-24 besides,
// and Phi's fitted factor 2^-17.  Relative errors are at most 2^-16 down to e^-87 -- a thirtieth of fp16's half step; where the exponential overflows the result is 0.
// fp32 outputs take the library's expf / erfcf.
template <bool FAST> __device__ __forceinline__ float lin_exp(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST> __device__ __forceinline__ float lin_rcp(float x) {
#ifndef TNV3_EMU
  if (FAST) return __builtin_amdgcn_rcpf(x);
#endif
  return 1.0f / x;
}
template <bool FAST> __device__ __forceinline__ float lin_sigmoid(float z) { return lin_rcp<FAST>(1.0f + lin_exp<FAST>(-z)); }
// Phi(z) = erfc(-z / sqrt 2) / 2, the normal distribution.  FAST: Phi(-y) = e^(-y^2 / 2) t P(t), t = 1 / (1 + 0.308 y), y = |z|, with P of degree 5 fitted to
// the least largest RELATIVE error over 0 <= y <= 14 (iteratively reweighted least squares against e^(y^2 / 2) Phi(-y) in 64 bits): 3.9e-6, 1e-5 with the
// exponential in fp32.  GELU's negative side is z Phi(z), so an absolute bound on erf would not do (a form
// of erf within 1.5e-7 gave 0.16 % at z = -5 and 2 % at -10: whole bf16 steps).
template <bool FAST> __device__ __forceinline__ float lin_phi(float z) {
  if (!FAST) return 0.5f * erfcf(-0.70710678118654752f * z);
  const float y = fabsf(z), t = lin_rcp<FAST>(1.0f + 0.308f * y);
  const float p = t * (0.123122714f + t * (0.118881114f + t * (0.13653404f + t * (0.0072720367f + t * (0.18961884f + t * -0.07543029f)))));
  const float tail = p * lin_exp<FAST>(-0.5f * y * y);          // Phi(-|z|)
  return z < 0.0f ? tail : 1.0f - tail;
}
constexpr float kGeluC = 0.79788456080286536f, kGeluA = 0.044715f;

template <bool FAST> __device__ __forceinline__ float lin_act1(float z, int act) {
  switch (act) {
    case kActLeaky: return z > 0.0f ? z : 0.01f * z;
    case kActSigmoid: return lin_sigmoid<FAST>(z);
    case kActRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);
    case kActSilu: return z * lin_sigmoid<FAST>(z);
    case kActGelu: return z * lin_phi<FAST>(z);
    case kActGeluTanh: return z * lin_sigmoid<FAST>(2.0f * kGeluC * (z + kGeluA * z * z * z));       // (1 + tanh a) / 2 = sigmoid(2 a)
    default: return z;
  }
}
// (act(z), act'(z)), act(z) the forward pass's own value.  Inside the exponentials and the derivative, arguments are clamped to +-128 (NaN kept): there
// sigmoid and Phi are exactly 0 or 1 in fp32 (e^-128 is below its least subnormal 2^-149 = e^-103.3), so nothing changes beyond, and products like
// z * (1 - sigmoid(z)) never are inf * 0.  (A clamp inside that range would show: z sigmoid(-64) is -160 at z = -1e30.)
template <bool FAST> __device__ __forceinline__ void lin_act_grad1(float z, int act, float& a, float& d) {
  const float zc = z < -128.0f ? -128.0f : (z > 128.0f ? 128.0f : z);
  switch (act) {
    case kActLeaky: a = z > 0.0f ? z : 0.01f * z; d = z > 0.0f ? 1.0f : 0.01f; return;
    case kActSigmoid: { const float s = lin_sigmoid<FAST>(zc); a = s; d = s * lin_sigmoid<FAST>(-zc); return; }      // (1 - s: 0 from z = 17 on)
    case kActRelu: a = z > 0.0f ? z : (z != z ? z : 0.0f); d = z <= 0.0f ? 0.0f : 1.0f; return;
    case kActSilu: { const float s = lin_sigmoid<FAST>(zc); a = z * s; d = s * (1.0f + zc * (1.0f - s)); return; }
    case kActGelu: { const float p = lin_phi<FAST>(zc); a = z * p; d = p + 0.39894228040143268f * zc * lin_exp<FAST>(-0.5f * zc * zc); return; }
    case kActGeluTanh: {
      const float s = lin_sigmoid<FAST>(2.0f * kGeluC * (zc + kGeluA * zc * zc * zc));
      a = z * s;
      d = s + 2.0f * zc * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluA * zc * zc);
      return;
    }
    default: a = z; d = 1.0f; return;
  }
}
template <bool FAST> __device__ __forceinline__ void lin_act8(float (&v)[8], int act) {
  // the switch is wave-uniform and outside the eight elements' loop
#define TNV3_LIN_ACT_CASE(A) case A: _Pragma("unroll") for (int i = 0; i < 8; ++i) v[i] = lin_act1<FAST>(v[i], A); break;
  switch (act) {
    TNV3_LIN_ACT_CASE(kActLeaky) TNV3_LIN_ACT_CASE(kActSigmoid) TNV3_LIN_ACT_CASE(kActRelu) TNV3_LIN_ACT_CASE(kActSilu)
    TNV3_LIN_ACT_CASE(kActGelu) TNV3_LIN_ACT_CASE(kActGeluTanh)
    default: break;
  }
#undef TNV3_LIN_ACT_CASE
}

// A raw buffer descriptor's range for `left` bytes up to the operand's end (negative: none): at most 2^31 - 1, in 32-bit scalar operations
__device__ __forceinline__ unsigned lin_range(long left) {
  const int hi = (int)(left >> 32);
  const unsigned lo = (unsigned)left;
  return hi < 0 ? 0u : (hi > 0 || lo > 0x7fffffffu ? 0x7fffffffu : lo);
}

// ---- LDS tiles
// Position (in 16-bit elements) of 8-element chunk c of row r in an LDS tile.  LDS has 64 banks of 4 bytes: a 16-byte fragment read serves 16 lanes
// (16 rows of one chunk) per clock if they name 16 different 16-byte slots of 256 bytes, the transposing read 32 lanes (4 rows of k, two 32-byte
// pieces each).  So the chunk index is exchanged with those row bits that rows of this length leave out of the bank number.  (With 32 banks' worth of row
// bits half of all LDS cycles were conflicts.)
template <int BK> __device__ __forceinline__ int lin_pos_kc(int r, int c) { return r * BK + ((c ^ (BK == 64 ? (r >> 1) & 7 : (r >> 2) & 3)) << 3); }
__device__ __forceinline__ int lin_pos_ks(int k, int c, int ld) { return k * ld + ((c ^ (ld == 64 ? (k & 2) << 1 : (k & 3) << 2)) << 3); }
// the same for fragments of 16 rows and 32 of k, whose transposing read takes rows k and k + 8 of one 32-byte piece at a time (rows of 128 elements and more)
__device__ __forceinline__ int lin_pos_ks16(int k, int c, int ld) { return k * ld + ((c ^ (((k & 3) << 2) | ((k & 8) >> 2))) << 3); }

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

// Fragments of one operand, 16x16x32: rows base + 16 t + (l & 15), k = 32 s + 8 (l >> 4) + 0..7, from a stage of 64 of k (base a multiple of 64).
// The lane's part of the address is computed once: k-contiguous rows differ by constants only, k-strided ones by one exclusive-or per 16 rows.
template <bool KS, int ROWS>
struct LinFrag16 {
  int off[KS ? 1 : 2];      // bytes
  __device__ __forceinline__ void init(int base, int lane) {
    const int q = lane & 15, g = lane >> 4;
    if (KS) {
      off[0] = 2 * (lin_pos_ks16(8 * g + (q >> 2), (base >> 3) + ((q & 3) >> 1), ROWS) + (q & 1) * 4);
    } else {
#pragma unroll
      for (int s = 0; s < (KS ? 1 : 2); ++s) off[s] = 2 * (base * 64 + lin_pos_kc<64>(q, 4 * s + g));
    }
  }
  __device__ __forceinline__ lin_s8 get(const unsigned short* tile, int t, int s) const {
    const char* p = reinterpret_cast<const char*>(tile);
    if (!KS) return *reinterpret_cast<const lin_s8*>(p + off[KS ? 0 : s] + t * 16 * 64 * 2);
    const unsigned short* r = reinterpret_cast<const unsigned short*>(p + (off[0] ^ (t << 5)) + s * 32 * ROWS * 2);
    const lin_s4 lo = lin_lds_tr4(r), hi = lin_lds_tr4(r + 4 * ROWS);      // row k + 4 has row k's order
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// ---- one product's arguments
struct LinGemmArgs {
  const void* a;          // element (i, k) at a[i * lda + k], or a[k * lda + i] where the kernel's operand is strided in k
  const void* b;          // element (j, k) likewise
  long rows_i, rows_j;    // valid i, j (gated: rows_j = the 2 F rows of the weight)
  long kk;                // contraction length
  long lda, ldb;
  const void* bias;       // [rows_j] or null
  const void* res;        // [rows_i][columns of out] or null
  void* out;              // [rows_i][rows_j], gated: [rows_i][F]
  void* pre;              // [rows_i][rows_j]: the pre-activation, for a backward pass, or null; gated: fp32 whatever the type
  float* part;            // splits > 1: [splits][rows_i][rows_j] partial sums instead of all of the above
  int act;
  int f;                  // gated: F
  int tiles_i, tiles_j, splits;
  long k_per_split;       // a multiple of the kernel's k step
};

// block -> (tile_i, tile_j, split); false: beyond the last.  Workgroups go to the 8 XCDs in turn, and each XCD has its own L2: XCD x gets the x-th contiguous
// eighth of the tile list, and the list walks 8 tiles of i within a panel before the next j, so that the ~32 tiles an XCD works on at a time
// share 8 panels of A and 4 of B.
__device__ __forceinline__ bool lin_tile(const LinGemmArgs& p, int b, int& ti, int& tj, int& sp) {
  const int tiles = p.tiles_i * p.tiles_j, total = tiles * p.splits;
  if (b >= total) return false;
  const int per = total >> 3, rem = total & 7, x = b & 7;
  int t = x * per + (x < rem ? x : rem) + (b >> 3);
  sp = t / tiles;
  t -= sp * tiles;
  const int group = 8 * p.tiles_j, g = t / group, in = t - g * group;
  const int left = p.tiles_i - 8 * g, gh = left < 8 ? left : 8;
  tj = in / gh;
  ti = 8 * g + (in - tj * gh);
  return true;
}

// ---- write-out of eight consecutive columns of one row; v: fp32 sums (gated: v gate, u the other factor).  PLAIN: no pre-activation is
// kept (a backward pass; known at compile time, its fp16 kernel of 256 x 256 spilled otherwise).
template <class T, bool PLAIN = false>
__device__ __forceinline__ void lin_finish8(const LinGemmArgs& p, long i, long j, float (&v)[8], const float (&bias)[8]) {
  if (i >= p.rows_i || j >= p.rows_j) return;
  const int n = p.rows_j - j < 8 ? (int)(p.rows_j - j) : 8;
  const bool vec = n == 8;
  const long o = i * p.rows_j + j;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += bias[e];
  if (!PLAIN && p.pre) lin_store_pre8<T>(static_cast<T*>(p.pre) + o, v, vec, n);
  lin_act8<sizeof(T) == 2>(v, p.act);
  if (p.res) {
    float r[8];
    lin_load8<T>(static_cast<const T*>(p.res) + o, r, vec, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  }
  lin_store8<T>(static_cast<T*>(p.out) + o, v, vec, n);
}
template <class T>
__device__ __forceinline__ void lin_finish_gated8(const LinGemmArgs& p, long i, long j, float (&g)[8], float (&u)[8], const float (&bg)[8],
                                                  const float (&bu)[8]) {
  if (i >= p.rows_i || j >= p.f) return;
  const int n = p.f - j < 8 ? (int)(p.f - j) : 8;
  const bool vec = n == 8;
#pragma unroll
  for (int e = 0; e < 8; ++e) { g[e] += bg[e]; u[e] += bu[e]; }
  if (p.pre) {
    float* pre = static_cast<float*>(p.pre) + i * p.rows_j + j;
    lin_store8<float>(pre, g, vec, n);
    lin_store8<float>(pre + p.f, u, vec, n);
  }
  lin_act8<sizeof(T) == 2>(g, p.act);
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] *= u[e];
  lin_store8<T>(static_cast<T*>(p.out) + i * p.f + j, g, vec, n);
}
template <class T>
__device__ __forceinline__ void lin_bias8(const LinGemmArgs& p, long j, float (&b)[8]) {
  const long left = p.rows_j - j;
  const int n = left < 8 ? (left < 0 ? 0 : (int)left) : 8;
  if (p.bias) lin_load8<T>(static_cast<const T*>(p.bias) + (n > 0 ? j : 0), b, n == 8, n);
  else
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = 0.0f;
}

// The write-out goes through LDS, 32 rows x 64 columns per wave at a time (a slab of its own: no workgroup barrier), because the accumulator
// layout gives a lane one column: read back by rows a lane holds eight consecutive columns, so bias, residual and outputs move in 16-byte pieces.
// A slab's residual is loaded before the exchange.  Where a row ends inside a lane's eight columns, that lane goes element by element.
// GATED: a wave's first TN/2 column tiles are the gate's, the last TN/2 the other factor's of the same outputs.
constexpr int kLinSlabLd = 68, kLinSlabFloats = 32 * kLinSlabLd;
__device__ __forceinline__ void lin_slab8(const float* s, float (&v)[8]) {
  const f32x4 a = reinterpret_cast<const f32x4*>(s)[0], b = reinterpret_cast<const f32x4*>(s)[1];
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
// put(slab, tm, left, right): the accumulators of rows 32 tm .. and column tiles (of 32) left, right into the slab.  PLAIN: the sums alone (a backward pass: no bias, activation, residual, pre-activation).
template <class T, int TM, int TN, bool GATED, bool PLAIN, class Put>
__device__ __forceinline__ void lin_write_out(const LinGemmArgs& p, Put put, float* slab, int lane, long i0, long j0, int sp) {
  static_assert(TN % 2 == 0, "a slab is two column tiles wide");
  constexpr int LPR = GATED ? 4 : 8, RPP = 64 / LPR, NP = 32 / RPP, NG = 2;        // lanes per row, rows per pass, passes, at a time
  constexpr bool FAST = sizeof(T) == 2;
  const long cols = GATED ? p.f : p.rows_j;
  float* part = p.part + (long)sp * p.rows_i * p.rows_j;
#pragma unroll
  for (int c = 0; c < TN / 2; ++c) {
    // linear: columns j0 + 64 c ..; gated: outputs j0 + 32 c .. (gate tile c, other factor's tile c + TN / 2)
    const long jc = j0 + (GATED ? 32 * c : 64 * c);
    const int left = GATED ? c : 2 * c, right = GATED ? c + TN / 2 : 2 * c + 1;
    const int lr = lane / LPR;
    const long j = jc + (lane % LPR) * 8;
    const bool in = j + 8 <= cols, rest = !in && j < cols;     // the lane's eight columns exist; some of them do
    float b0[8], b1[8];
    if (p.splits == 1) {                                     // (PLAIN: there is none, zeros)
      lin_bias8<T>(p, j < cols ? j : p.rows_j, b0);
      if (GATED) lin_bias8<T>(p, j < cols ? p.f + j : p.rows_j, b1);
    }
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) {
      const long ir = i0 + 32 * tm + lr;                     // pass q: row ir + q RPP
      lin_u4 r[GATED ? 1 : NP][sizeof(T) / 2];
      if (!GATED && !PLAIN && p.res && p.splits == 1) {
#pragma unroll
        for (int q = 0; q < (GATED ? 1 : NP); ++q)
          if (in && ir + q * RPP < p.rows_i) {
#pragma unroll
            for (int h = 0; h < (int)sizeof(T) / 2; ++h)
              r[q][h] = reinterpret_cast<const lin_u4_any*>(static_cast<const T*>(p.res) + (ir + q * RPP) * p.rows_j + j)[h];
          }
      }
      lin_wave_sync();
      put(slab, tm, left, right);
      lin_wave_sync();
      if (rest) {
#pragma unroll 1
        for (int q = 0; q < NP; ++q) {
          const float* s = slab + (q * RPP + lr) * kLinSlabLd + (lane % LPR) * 8;
          const long i = ir + q * RPP;
          float v[8], u[8];
          lin_slab8(s, v);
          if (GATED) lin_slab8(s + 32, u);
          if (p.splits > 1) {
            const int n = (int)(cols - j);
            if (i < p.rows_i) {
              lin_store8<float>(part + i * p.rows_j + j, v, false, n);
              if (GATED) lin_store8<float>(part + i * p.rows_j + p.f + j, u, false, n);
            }
          } else if (GATED) {
            lin_finish_gated8<T>(p, i, j, v, u, b0, b1);
          } else {
            lin_finish8<T, PLAIN>(p, i, j, v, b0);
          }
        }
      }
#pragma unroll
      for (int q0 = 0; q0 < NP; q0 += NG) {
        float v[NG][8], u[GATED ? NG : 1][8];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const float* s = slab + ((q0 + q) * RPP + lr) * kLinSlabLd + (lane % LPR) * 8;
          lin_slab8(s, v[q]);
          if (GATED) lin_slab8(s + 32, u[GATED ? q : 0]);
        }
        if (p.splits > 1) {
#pragma unroll
          for (int q = 0; q < NG; ++q)
            if (in && ir + (q0 + q) * RPP < p.rows_i) {
              float* o = part + (ir + (q0 + q) * RPP) * p.rows_j + j;
              lin_store8<float>(o, v[q], true, 8);
              if (GATED) lin_store8<float>(o + p.f, u[GATED ? q : 0], true, 8);
            }
          continue;
        }
#pragma unroll
        for (int q = 0; q < (PLAIN ? 0 : NG); ++q)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[q][e] += b0[e];
            if (GATED) u[GATED ? q : 0][e] += b1[e];
          }
        if (!PLAIN && p.pre) {
#pragma unroll
          for (int q = 0; q < NG; ++q)
            if (in && ir + (q0 + q) * RPP < p.rows_i) {
              const long o = (ir + (q0 + q) * RPP) * p.rows_j + j;
              if (GATED) {
                lin_store8<float>(static_cast<float*>(p.pre) + o, v[q], true, 8);
                lin_store8<float>(static_cast<float*>(p.pre) + o + p.f, u[GATED ? q : 0], true, 8);
              } else {
                lin_store_pre8<T>(static_cast<T*>(p.pre) + o, v[q], true, 8);
              }
            }
        }
        // the switch is wave-uniform and outside the elements' loops
#define TNV3_LIN_ACT_CASE(A)                                                                        \
    case A:                                                                                           \
      _Pragma("unroll") for (int q = 0; q < NG; ++q)                                                  \
        _Pragma("unroll") for (int e = 0; e < 8; ++e) v[q][e] = lin_act1<FAST>(v[q][e], A);           \
      break;
        switch (PLAIN ? kActNone : p.act) {
          TNV3_LIN_ACT_CASE(kActLeaky) TNV3_LIN_ACT_CASE(kActSigmoid) TNV3_LIN_ACT_CASE(kActRelu) TNV3_LIN_ACT_CASE(kActSilu)
          TNV3_LIN_ACT_CASE(kActGelu) TNV3_LIN_ACT_CASE(kActGeluTanh)
          default: break;
        }
#undef TNV3_LIN_ACT_CASE
#pragma unroll
        for (int q = 0; q < NG; ++q)
          if (in && ir + (q0 + q) * RPP < p.rows_i) {
            if (GATED) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[q][e] *= u[GATED ? q : 0][e];
              lin_store8<T>(static_cast<T*>(p.out) + (ir + (q0 + q) * RPP) * p.f + j, v[q], true, 8);
            } else {
              if (!PLAIN && p.res) {
                float a[8];
                lin_unpack8(r[GATED ? 0 : q0 + q], a, T{});
#pragma unroll
                for (int e = 0; e < 8; ++e) v[q][e] += a[e];
              }
              lin_store8<T>(static_cast<T*>(p.out) + (ir + (q0 + q) * RPP) * p.rows_j + j, v[q], true, 8);
            }
          }
      }
    }
  }
}

template <int TM, int TN>
__device__ __forceinline__ void lin_put32(const f32x16 (&acc)[TM][TN], float* slab, int tm, int left, int right, int lane) {
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float* d = slab + ((r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * kLinSlabLd + (lane & 31);
    d[0] = acc[tm][left][r];
    d[32] = acc[tm][right][r];
  }
}
template <int XM, int YN>
__device__ __forceinline__ void lin_put16(const f32x4 (&acc)[XM][YN], float* slab, int tm, int left, int right, int lane) {
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        slab[(16 * x + 4 * (lane >> 4) + r) * kLinSlabLd + 16 * y + (lane & 15)] = acc[2 * tm + x][2 * (y < 2 ? left : right) + (y & 1)][r];
}

// ---- joins the partial sums of a split contraction in a fixed order and finishes them: one work-item per 8 columns of a row
template <class T, bool GATED>
__device__ __forceinline__ void lin_join(const LinGemmArgs& p, long block) {
  const long cols = GATED ? p.f : p.rows_j, pieces = (cols + 7) / 8;
  const long t = block * 256 + threadIdx.x;
  const long i = t / pieces, j = (t - i * pieces) * 8;
  if (i >= p.rows_i) return;
  const int n = cols - j < 8 ? (int)(cols - j) : 8;
  const bool vec = n == 8;
  float v[8], u[8], q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = u[e] = 0.0f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* part = p.part + ((long)s * p.rows_i + i) * p.rows_j + j;
    lin_load8<float>(part, q, vec, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += q[e];
    if (GATED) {
      lin_load8<float>(part + p.f, q, vec, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] += q[e];
    }
  }
  float b0[8], b1[8];
  lin_bias8<T>(p, j, b0);
  if (GATED) {
    lin_bias8<T>(p, p.f + j, b1);
    lin_finish_gated8<T>(p, i, j, v, u, b0, b1);
  } else {
    lin_finish8<T>(p, i, j, v, b0);
  }
}

template <class T, bool GATED>
__global__ void __launch_bounds__(256) lin_join_kernel(const LinGemmArgs p) { lin_join<T, GATED>(p, blockIdx.x); }

// ---- a backward pass's products in one launch: blocks [0, blocks_dx) the gradient of x, then blocks_dw the gradient of W, then the bias gradient's
// column sums from their row blocks' partial sums; a count of 0 leaves one out.  The first two counts are multiples of 8 (XCDs).
struct LinPairArgs {
  LinGemmArgs dx, dw;
  const float* sums;      // [sum_rows][sum_cols]
  void* db;
  int blocks_dx, blocks_dw, sum_rows, sum_cols;
};
// 128 columns per workgroup, NT / 128 work-items per column, joined in order
template <class T, int NT>
__device__ __forceinline__ void lin_colsum(const float* __restrict__ part, T* __restrict__ out, int rows, int cols, int block, float* red) {
  constexpr int Y = NT / 128;
  const int c = threadIdx.x & 127, y = threadIdx.x >> 7, j = block * 128 + c;
  float s = 0.0f;
  if (j < cols) {
#pragma unroll 8
    for (int r = y; r < rows; r += Y) s += part[(long)r * cols + j];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (y || j >= cols) return;
#pragma unroll
  for (int q = 1; q < Y; ++q) s += red[q * 128 + c];
  lin_down(s, out[j]);
}
template <class T>
__global__ void __launch_bounds__(256) lin_join_pair_kernel(const LinPairArgs p) {
  // blocks_dx / blocks_dw: of this launch
  if ((int)blockIdx.x < p.blocks_dx) lin_join<T, false>(p.dx, blockIdx.x);
  else lin_join<T, false>(p.dw, (long)blockIdx.x - p.blocks_dx);
}

// ---- 16-bit operands whose rows are no whole 16-byte pieces: copied once into rows that are, the added columns 0.  Bound by memory (each element
// read and written once); the products then take the direct loads at full speed.
struct LinPadArgs {
  const unsigned short* src[2];
  unsigned short* dst[2];
  long rows[2];
  int width[2];
  long blocks0;           // workgroups of the first of the two
};
inline __host__ __device__ int lin_pad_width(int w) { return (w + 7) / 8 * 8; }
inline __global__ void __launch_bounds__(256) lin_pad_kernel(const LinPadArgs p) {
  const int o = (long)blockIdx.x >= p.blocks0;
  const long t = ((long)blockIdx.x - (o ? p.blocks0 : 0)) * 256 + threadIdx.x;
  const int w = p.width[o], pieces = (w + 7) / 8;
  const long r = t / pieces;
  const int c = (int)(t - r * pieces) * 8;
  if (r >= p.rows[o]) return;
  const unsigned short* s = p.src[o] + r * w + c;
  lin_u4 q = {0u, 0u, 0u, 0u};
  if (c + 8 <= w) {
    q = *reinterpret_cast<const lin_u4_any*>(s);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < w) q[e >> 1] |= (unsigned)s[e] << (16 * (e & 1));
  }
  *reinterpret_cast<lin_u4*>(p.dst[o] + (r * pieces) * 8 + c) = q;
}

}  // namespace tnv3

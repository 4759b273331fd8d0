// tnv3_linear_impl.h -- argument checks, workspaces and dispatch of the position-wise layers (tnv3_linear_*, tnv3_gated_linear_*).
#pragma once
#include "kernels/linear_common.h"
#include "kernels/linear_dma.h"
#include "kernels/linear_grad.h"
#include "kernels/linear_rows.h"
#include "kernels/linear_split.h"
#include "kernels/linear_staged.h"
#include "tnv3_impl.h"

namespace tnv3 {

using LinS128 = LinStagedCfg<2, 2, 2, 2>;       // 128 x 128, four waves of 64 x 64
using LinD256 = LinDmaCfg<2, 4, 4, 2>;          // 256 x 256, eight waves of 64 x 128: one workgroup per CU
using LinD128 = LinDmaCfg<2, 2, 2, 2>;          // 128 x 128, four waves of 64 x 64: two workgroups per CU
using LinF256 = LinSplitCfg<2, 2, 4, 2>;        // fp32: 256 x 128, eight waves of 64 x 64, one workgroup per CU (144 KB of LDS)
using LinF128 = LinSplitCfg<1, 2, 4, 1>;        // fp32: 128 x 64, four waves of 32 x 64, two workgroups per CU

constexpr long kLinMaxWidth = 1l << 20;         // columns: a tile's rows stay within 2^31 bytes of its first
constexpr long kLinMaxRows = 1l << 30;

inline size_t lin_pad(size_t b) { return (b + 255) & ~(size_t)255; }
inline int lin_size(int dtype) { return dtype == kLinF32 ? 4 : 2; }
inline bool lin_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// One product's tiling.  Sizes and type decide, never the pointers, so that the workspace queries and the launches agree; the kernel that runs it may
// still depend on alignment.
struct LinPlan {
  int bi, bj, splits;
  long k_per_split;
  size_t part_bytes;
};
inline LinPlan lin_plan(int dtype, long rows_i, long rows_j, long kk, bool gated) {
  LinPlan pl;
  pl.bi = pl.bj = 128;
  if (dtype == kLinF32) {
    const long big = ((rows_i + 255) / 256) * (gated ? (rows_j / 2 + 63) / 64 : (rows_j + 127) / 128);
    if (big >= num_cus()) pl.bi = 256;
    else pl.bj = 64;
  }
  // 16-bit products with at least a 256 x 256 tile for every CU take those: half the LDS and L2 traffic per product
  if (dtype != kLinF32) {
    const long big = ((rows_i + 255) / 256) * (gated ? (rows_j / 2 + 127) / 128 : (rows_j + 255) / 256);
    if (big >= num_cus()) pl.bi = pl.bj = 256;
  }
  const long ti = (rows_i + pl.bi - 1) / pl.bi, tj = gated ? (rows_j / 2 + pl.bj / 2 - 1) / (pl.bj / 2) : (rows_j + pl.bj - 1) / pl.bj;
  const long tiles = ti * tj, cus = num_cus(), step = 64, steps = (kk + step - 1) / step;
  // fewer tiles than CUs: the contraction is split so that all take part, as long as a part keeps 4 steps of 64
  long s = 1;
  if (tiles < cus) {
    s = cus / tiles;
    if (s > steps / 4) s = steps / 4;
    if (s > 32) s = 32;
    if (s < 1) s = 1;
  }
  const long per = (steps + s - 1) / s;
  pl.splits = (int)((steps + per - 1) / per);
  if (pl.splits < 1) pl.splits = 1;
  pl.k_per_split = per * step;
  pl.part_bytes = pl.splits > 1 ? lin_pad((size_t)pl.splits * rows_i * rows_j * 4) : 0;
  return pl;
}

template <class T, bool KSA, bool KSB, bool GATED, class Launcher>
int lin_launch(Launcher& L, LinGemmArgs& p, const LinPlan& pl) {
  p.splits = pl.splits;
  p.k_per_split = pl.k_per_split;
  const bool direct = sizeof(T) == 2 && (p.vec & kLinVecA) && (p.vec & kLinVecB);
  const int bi = direct || sizeof(T) == 4 ? pl.bi : 128, bj = direct || sizeof(T) == 4 ? pl.bj : 128;
  p.tiles_i = (int)((p.rows_i + bi - 1) / bi);
  p.tiles_j = GATED ? (p.f + bj / 2 - 1) / (bj / 2) : (int)((p.rows_j + bj - 1) / bj);
  const long grid = (long)p.tiles_i * p.tiles_j * p.splits;
  if (grid >= (1l << 31)) TNV3_FAIL(-1, "linear: %ld tiles are more than one launch takes", grid);
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (direct && bi == 256) rc = L.launch(lin_dma_kernel<LinD256, T, KSA, KSB, GATED>, (int)grid, LinD256::NT, p);
    else if (direct) rc = L.launch(lin_dma_kernel<LinD128, T, KSA, KSB, GATED>, (int)grid, LinD128::NT, p);
    else rc = L.launch(lin_staged_kernel<LinS128, T, KSA, KSB, GATED>, (int)grid, LinS128::NT, p);
  } else {
    if (bi == 256) rc = L.launch(lin_split_kernel<LinF256, KSA, KSB, GATED>, (int)grid, LinF256::NT, p);
    else rc = L.launch(lin_split_kernel<LinF128, KSA, KSB, GATED>, (int)grid, LinF128::NT, p);
  }
  if (rc || p.splits == 1) return rc;
  const long pieces = p.rows_i * (((GATED ? p.f : p.rows_j) + 7) / 8), blocks = (pieces + 255) / 256;
  if (blocks >= (1l << 31)) TNV3_FAIL(-1, "linear: %ld workgroups are more than one launch takes", blocks);
  return L.launch(lin_join_kernel<T, GATED>, (int)blocks, 256, p);
}

// Forward products of up to kLinFewRows rows.
constexpr long kLinFewRows = 64;
template <class T, bool GATED, class Launcher>
int lin_rows_launch(Launcher& L, LinGemmArgs& p) {
  p.splits = 1;
  const int grid = (int)(((GATED ? (long)p.f : p.rows_j) + 15) / 16);
  if (p.rows_i <= 16) return L.launch(lin_rows_kernel<T, 1, 16, GATED>, grid, 1024, p);
  if (p.rows_i <= 32) return L.launch(lin_rows_kernel<T, 2, 8, GATED>, grid, 512, p);
  return L.launch(lin_rows_kernel<T, 4, 8, GATED>, grid, 512, p);
}

// ---- the three products of a layer (n2: rows of the weight)
template <class T, bool GATED, class Launcher>
int lin_forward_t(Launcher& L, int dtype, const void* x, const void* w, const void* bias, const void* res, void* out, void* pre, void* ws, long rows,
                  int k, int n, int act) {
  LinGemmArgs p = {};
  const int n2 = GATED ? 2 * n : n;
  const int e16 = 16 / lin_size(dtype);
  p.a = x; p.b = w; p.rows_i = rows; p.rows_j = n2; p.kk = k; p.lda = p.ldb = k;
  p.bias = bias; p.res = res; p.out = out; p.pre = pre; p.part = static_cast<float*>(ws); p.act = act; p.f = GATED ? n : 0;
  const bool kvec = k % e16 == 0;
  p.vec = (kvec && lin_aligned(x) ? kLinVecA : 0) | (kvec && lin_aligned(w) ? kLinVecB : 0) |
          (n % 8 == 0 && lin_aligned(bias) && lin_aligned(res) && lin_aligned(out) && lin_aligned(pre) ? kLinVecOut : 0);
  if (rows <= kLinFewRows) return lin_rows_launch<T, GATED>(L, p);
  return lin_launch<T, false, false, GATED>(L, p, lin_plan(dtype, rows, n2, k, GATED));
}
template <class T, class Launcher>
int lin_dx_t(Launcher& L, int dtype, const void* dz, const void* w, void* dx, void* ws, long rows, int k, int n2) {
  LinGemmArgs p = {};
  const int e16 = 16 / lin_size(dtype);
  p.a = dz; p.b = w; p.rows_i = rows; p.rows_j = k; p.kk = n2; p.lda = n2; p.ldb = k; p.out = dx; p.part = static_cast<float*>(ws);
  p.vec = (n2 % e16 == 0 && lin_aligned(dz) ? kLinVecA : 0) | (k % e16 == 0 && lin_aligned(w) ? kLinVecB : 0) | (k % 8 == 0 && lin_aligned(dx) ? kLinVecOut : 0);
  return lin_launch<T, false, true, false>(L, p, lin_plan(dtype, rows, k, n2, false));
}
template <class T, class Launcher>
int lin_dw_t(Launcher& L, int dtype, const void* dz, const void* x, void* dw, void* ws, long rows, int k, int n2) {
  LinGemmArgs p = {};
  const int e16 = 16 / lin_size(dtype);
  p.a = dz; p.b = x; p.rows_i = n2; p.rows_j = k; p.kk = rows; p.lda = n2; p.ldb = k; p.out = dw; p.part = static_cast<float*>(ws);
  p.vec = (n2 % e16 == 0 && lin_aligned(dz) ? kLinVecA : 0) | (k % e16 == 0 && lin_aligned(x) ? kLinVecB : 0) | (k % 8 == 0 && lin_aligned(dw) ? kLinVecOut : 0);
  return lin_launch<T, true, true, false>(L, p, lin_plan(dtype, n2, k, rows, false));
}

// rows per workgroup of the element-wise pass: about four workgroups per CU, at least 8 rows (one per work-item) each
inline long lin_dz_rows(long rows, int n) {
  const long jt = (n + 255) / 256, want = 4l * num_cus() / jt, blocks = want < 1 ? 1 : (want > 256 ? 256 : want);
  const long per = ((rows + blocks - 1) / blocks + 7) / 8 * 8;
  return per < 8 ? 8 : per;
}
template <class T, bool GATED, class Launcher>
int lin_dz_t(Launcher& L, const void* dy, const void* pre, void* dz, float* part, void* db, long rows, int n, int act) {
  LinDzArgs a = {};
  a.dy = dy; a.pre = pre; a.dz = dz; a.part = part; a.rows = rows; a.n = n; a.act = act;
  a.rows_per_block = (int)lin_dz_rows(rows, n);
  a.vec = n % 8 == 0 && lin_aligned(dy) && lin_aligned(pre) && lin_aligned(dz);
  const long jt = (n + 255) / 256, blocks = (rows + a.rows_per_block - 1) / a.rows_per_block;
  int rc = L.launch(lin_dz_kernel<T, GATED>, (int)(jt * blocks), 256, a);
  if (rc || !db) return rc;
  const int n2 = GATED ? 2 * n : n;
  return L.launch(lin_colsum_kernel<T>, (n2 + 255) / 256, 256, part, static_cast<T*>(db), n2, (int)blocks);
}

inline int lin_check(const char* what, long rows, int k, int n, int act, int dtype, bool gated) {
  if (dtype < 0 || dtype > 2) TNV3_FAIL(-1, "%s: dtype %d is none of 0 (fp32), 1 (bf16), 2 (fp16)", what, dtype);
  if (act < 0 || act >= kActCount) TNV3_FAIL(-1, "%s: unknown activation %d", what, act);
  if (rows < 1 || k < 1 || n < 1) TNV3_FAIL(-1, "%s: sizes must be positive (rows %ld, k %d, n %d)", what, rows, k, n);
  if (rows > kLinMaxRows || k > kLinMaxWidth || (gated ? 2l * n : (long)n) > kLinMaxWidth)
    TNV3_FAIL(-1, "%s: rows %ld / widths %d, %d beyond 2^30 / 2^20", what, rows, k, n);
  return 0;
}

inline size_t lin_forward_workspace_bytes(long rows, int k, int n, int dtype, bool gated) {
  if (lin_check("workspace", rows, k, n, 0, dtype, gated)) return 0;
  return rows <= kLinFewRows ? 0 : lin_plan(dtype, rows, gated ? 2l * n : n, k, gated).part_bytes;
}
struct LinBackwardLayout { size_t dz, sums, part, total; };
inline LinBackwardLayout lin_backward_layout(long rows, int k, int n, int act, int dtype, bool gated) {
  const long n2 = gated ? 2l * n : n;
  LinBackwardLayout l;
  l.dz = 0;
  l.sums = l.dz + (gated || act != kActNone ? lin_pad((size_t)rows * n2 * lin_size(dtype)) : 0);
  const long per = lin_dz_rows(rows, n);
  l.part = l.sums + lin_pad((size_t)((rows + per - 1) / per) * n2 * 4);
  const size_t a = lin_plan(dtype, rows, k, n2, false).part_bytes, b = lin_plan(dtype, n2, k, rows, false).part_bytes;
  l.total = l.part + (a > b ? a : b);
  return l;
}
inline size_t lin_backward_workspace_bytes(long rows, int k, int n, int act, int dtype, bool gated) {
  if (lin_check("workspace", rows, k, n, act, dtype, gated)) return 0;
  return lin_backward_layout(rows, k, n, act, dtype, gated).total;
}

template <bool GATED, class Launcher>
int lin_forward_impl(Launcher& L, const void* x, const void* w, const void* bias, const void* res, void* out, void* pre, void* ws, size_t ws_bytes,
                     long rows, int k, int n, int act, int dtype) {
  const char* what = GATED ? "gated_linear_forward" : "linear_forward";
  if (int rc = lin_check(what, rows, k, n, act, dtype, GATED)) return rc;
  if (!x || !w || !out) TNV3_FAIL(-1, "%s: null tensor", what);
  const size_t need = lin_forward_workspace_bytes(rows, k, n, dtype, GATED);
  if (need && (!ws || ws_bytes < need || !lin_aligned(ws))) TNV3_FAIL(-1, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, ws_bytes, need);
  switch (dtype) {
    case kLinF32: return lin_forward_t<float, GATED>(L, dtype, x, w, bias, res, out, pre, ws, rows, k, n, act);
    case kLinBf16: return lin_forward_t<LinBf16, GATED>(L, dtype, x, w, bias, res, out, pre, ws, rows, k, n, act);
    default: return lin_forward_t<LinF16, GATED>(L, dtype, x, w, bias, res, out, pre, ws, rows, k, n, act);
  }
}

template <class T, bool GATED, class Launcher>
int lin_backward_t(Launcher& L, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw, void* db, char* ws,
                   const LinBackwardLayout& l, long rows, int k, int n, int act, int dtype) {
  const int n2 = GATED ? 2 * n : n;
  const bool act_pass = GATED || act != kActNone;
  const void* dz = act_pass ? ws + l.dz : dy;
  if (act_pass || db) {
    const int rc = lin_dz_t<T, GATED>(L, dy, act_pass ? pre : nullptr, act_pass ? ws + l.dz : nullptr, db ? reinterpret_cast<float*>(ws + l.sums) : nullptr, db,
                                      rows, n, act);
    if (rc) return rc;
  }
  if (dx)
    if (int rc = lin_dx_t<T>(L, dtype, dz, w, dx, ws + l.part, rows, k, n2)) return rc;
  if (dw)
    if (int rc = lin_dw_t<T>(L, dtype, dz, x, dw, ws + l.part, rows, k, n2)) return rc;
  return 0;
}
template <bool GATED, class Launcher>
int lin_backward_impl(Launcher& L, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                      long rows, int k, int n, int act, int dtype) {
  const char* what = GATED ? "gated_linear_backward" : "linear_backward";
  if (int rc = lin_check(what, rows, k, n, act, dtype, GATED)) return rc;
  if (!dy || (dx && !w) || (dw && !x)) TNV3_FAIL(-1, "%s: null tensor", what);
  if ((GATED || act != kActNone) && !pre) TNV3_FAIL(-1, "%s: the forward's pre-activation is required", what);
  const LinBackwardLayout l = lin_backward_layout(rows, k, n, act, dtype, GATED);
  if (!ws || ws_bytes < l.total || !lin_aligned(ws)) TNV3_FAIL(-1, "%s: workspace of %zu bytes, %zu needed (16-byte aligned)", what, ws_bytes, l.total);
  char* wsc = static_cast<char*>(ws);
  switch (dtype) {
    case kLinF32: return lin_backward_t<float, GATED>(L, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act, dtype);
    case kLinBf16: return lin_backward_t<LinBf16, GATED>(L, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act, dtype);
    default: return lin_backward_t<LinF16, GATED>(L, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act, dtype);
  }
}

}  // namespace tnv3

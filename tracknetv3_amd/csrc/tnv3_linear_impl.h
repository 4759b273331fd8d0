// tnv3_linear_impl.h -- argument checks, workspaces and dispatch of the position-wise layers (tnv3_linear_*, tnv3_gated_linear_*).
#pragma once
#include "kernels/linear_common.h"
#include "kernels/linear_dma.h"
#include "kernels/linear_grad.h"
#include "kernels/linear_rows.h"
#include "kernels/linear_split.h"
#include "tnv3_impl.h"

namespace tnv3 {

using LinD256 = LinDmaCfg<2, 4, 4, 2>;          // 256 x 256, eight waves of 64 x 128: one workgroup per CU
using LinD128 = LinDmaCfg<2, 2, 2, 2>;          // 128 x 128, four waves of 64 x 64: two workgroups per CU
using LinF256 = LinSplitCfg<2, 2, 4, 2>;        // fp32: 256 x 128, eight waves of 64 x 64, one workgroup per CU (144 KB of LDS)
using LinF128 = LinSplitCfg<1, 2, 4, 1>;        // fp32: 128 x 64, four waves of 32 x 64, two workgroups per CU

constexpr long kLinMaxWidth = 1l << 20;         // columns: a tile's rows stay within 2^31 bytes of its first
constexpr long kLinMaxRows = 1l << 30;

inline size_t lin_pad(size_t b) { return (b + 255) & ~(size_t)255; }
inline int lin_size(int dtype) { return dtype == kLinF32 ? 4 : 2; }

// One product's tiling.  Sizes and type decide, never the pointers, so that the workspace queries and the launches agree.
struct LinPlan {
  bool wide;              // the 256-row tiles
  int bi, bj, splits;
  long k_per_split, tiles;
  size_t part_bytes;
};
inline long lin_tiles(long rows_i, long rows_j, bool gated, int bi, int bj) {
  return ((rows_i + bi - 1) / bi) * (gated ? (rows_j / 2 + bj / 2 - 1) / (bj / 2) : (rows_j + bj - 1) / bj);
}
inline void lin_tile_shape(LinPlan& pl, int dtype, bool wide) {
  pl.wide = wide;
  pl.bi = wide ? 256 : 128;
  pl.bj = dtype == kLinF32 ? (wide ? 128 : 64) : (wide ? 256 : 128);
}
inline long lin_wide_tiles(int dtype, long rows_i, long rows_j, bool gated) { return lin_tiles(rows_i, rows_j, gated, 256, dtype == kLinF32 ? 128 : 256); }
// others: tiles of a product in the same launch
inline void lin_split_plan(LinPlan& pl, long rows_i, long rows_j, long kk, bool gated, long others) {
  pl.tiles = lin_tiles(rows_i, rows_j, gated, pl.bi, pl.bj);
  // fewer tiles than CUs: the contraction is split so that all take part, as long as a part keeps 4 steps of 64
  const long tiles = pl.tiles + others, cus = num_cus(), step = 64, steps = (kk + step - 1) / step;
  long s = 1;
  if (tiles < cus) {
    s = cus / tiles;
    if (s > steps / 4) s = steps / 4;
    if (s > 32) s = 32;
    if (s < 1) s = 1;
  }
  const long per = (steps + s - 1) / s;
  pl.splits = (int)((steps + per - 1) / per);
  pl.k_per_split = per * step;
  pl.part_bytes = pl.splits > 1 ? lin_pad((size_t)pl.splits * rows_i * rows_j * 4) : 0;
}
inline LinPlan lin_plan(int dtype, long rows_i, long rows_j, long kk, bool gated) {
  LinPlan pl;
  // at least a 256-row tile for every CU: half the LDS and L2 traffic per product
  lin_tile_shape(pl, dtype, lin_wide_tiles(dtype, rows_i, rows_j, gated) >= num_cus());
  lin_split_plan(pl, rows_i, rows_j, kk, gated, 0);
  return pl;
}
inline void lin_apply(LinGemmArgs& p, const LinPlan& pl, float* part) {
  p.splits = pl.splits;
  p.k_per_split = pl.k_per_split;
  p.tiles_i = (int)((p.rows_i + pl.bi - 1) / pl.bi);
  p.tiles_j = (int)(pl.tiles / p.tiles_i);
  p.part = part;
}
inline long lin_join_blocks(const LinGemmArgs& p, bool gated) { return (p.rows_i * (((gated ? (long)p.f : p.rows_j) + 7) / 8) + 255) / 256; }
inline int lin_grid_check(long blocks) {
  if (blocks >= (1l << 31)) TNV3_FAIL(-1, "linear: %ld workgroups are more than one launch takes", blocks);
  return 0;
}
// 16-bit rows that are no whole 16-byte pieces are copied into the workspace
inline bool lin_pads(int dtype, int width) { return dtype != kLinF32 && width % 8 != 0; }
inline int lin_ld(int dtype, int width) { return lin_pads(dtype, width) ? lin_pad_width(width) : width; }
inline size_t lin_pad_bytes(int dtype, long rows, int width) { return lin_pads(dtype, width) ? lin_pad((size_t)rows * lin_pad_width(width) * 2) : 0; }
struct LinPadder {
  LinPadArgs a = {};
  int count = 0;
  long blocks = 0;
  const void* add(int dtype, const void* src, long rows, int width, char* dst) {
    if (!lin_pads(dtype, width)) return src;
    a.src[count] = static_cast<const unsigned short*>(src);
    a.dst[count] = reinterpret_cast<unsigned short*>(dst);
    a.rows[count] = rows;
    a.width[count] = width;
    blocks += (rows * (lin_pad_width(width) / 8) + 255) / 256;
    if (count++ == 0) a.blocks0 = blocks;
    return dst;
  }
  template <class Launcher> int launch(Launcher& L) {
    if (!count) return 0;
    if (int rc = lin_grid_check(blocks)) return rc;
    return L.launch(lin_pad_kernel, (int)blocks, 256, a);
  }
};

// ---- forward
constexpr long kLinFewRows = 64;       // up to here the weight's bytes are the bound: lin_rows_kernel
struct LinForwardLayout { LinPlan plan; size_t x, w, part, total; };
inline LinForwardLayout lin_forward_layout(long rows, int k, int n2, int dtype, bool gated) {
  LinForwardLayout l = {};
  if (rows <= kLinFewRows) return l;
  l.plan = lin_plan(dtype, rows, n2, k, gated);
  l.x = 0;
  l.w = l.x + lin_pad_bytes(dtype, rows, k);
  l.part = l.w + lin_pad_bytes(dtype, n2, k);
  l.total = l.part + l.plan.part_bytes;
  return l;
}
template <class T, bool GATED, class Launcher>
int lin_forward_t(Launcher& L, int dtype, const void* x, const void* w, const void* bias, const void* res, void* out, void* pre, char* ws,
                  const LinForwardLayout& l, long rows, int k, int n, int act) {
  LinGemmArgs p = {};
  const int n2 = GATED ? 2 * n : n;
  p.a = x; p.b = w; p.rows_i = rows; p.rows_j = n2; p.kk = k; p.lda = p.ldb = k; p.splits = 1;
  p.bias = bias; p.res = res; p.out = out; p.pre = pre; p.act = act; p.f = GATED ? n : 0;
  p.vec = n % 8 == 0;
  if (rows <= kLinFewRows) {
    const int grid = (n + 15) / 16;
    if (rows <= 16) return L.launch(lin_rows_kernel<T, 1, 16, GATED>, grid, 1024, p);
    if (rows <= 32) return L.launch(lin_rows_kernel<T, 2, 8, GATED>, grid, 512, p);
    return L.launch(lin_rows_kernel<T, 4, 8, GATED>, grid, 512, p);
  }
  LinPadder pad;
  p.a = pad.add(dtype, x, rows, k, ws + l.x);
  p.b = pad.add(dtype, w, n2, k, ws + l.w);
  p.lda = p.ldb = lin_ld(dtype, k);
  lin_apply(p, l.plan, reinterpret_cast<float*>(ws + l.part));
  const long grid = l.plan.tiles * p.splits, join = lin_join_blocks(p, GATED);
  if (int rc = lin_grid_check(grid > join ? grid : join)) return rc;
  if (int rc = pad.launch(L)) return rc;
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (l.plan.wide) rc = L.launch(lin_dma_kernel<LinD256, T, GATED>, (int)grid, LinD256::NT, p);
    else rc = L.launch(lin_dma_kernel<LinD128, T, GATED>, (int)grid, LinD128::NT, p);
  } else {
    if (l.plan.wide) rc = L.launch(lin_split_kernel<LinF256, GATED>, (int)grid, LinF256::NT, p);
    else rc = L.launch(lin_split_kernel<LinF128, GATED>, (int)grid, LinF128::NT, p);
  }
  if (rc || p.splits == 1) return rc;
  return L.launch(lin_join_kernel<T, GATED>, (int)join, 256, p);
}

// ---- backward: dz (with the bias gradient's partial sums), then both products in one launch
// row blocks of the element-wise pass: about four workgroups per CU, at least 8 rows (one per work-item) each, and no more blocks than the final column
// sums can add quickly
inline long lin_dz_rows(long rows, int n) {
  const long jt = (n + 255) / 256, cap = rows / 128 < 64 ? 64 : (rows / 128 > 512 ? 512 : rows / 128);
  long blocks = 4l * num_cus() / jt;
  blocks = blocks < 1 ? 1 : (blocks > cap ? cap : blocks);
  const long per = ((rows + blocks - 1) / blocks + 7) / 8 * 8;
  return per < 8 ? 8 : per;
}
struct LinBackwardLayout { LinPlan dx, dw; size_t dz, sums, w, x, part_dx, part_dw, total; };
inline LinBackwardLayout lin_backward_layout(long rows, int k, int n, int act, int dtype, bool gated) {
  const int n2 = gated ? 2 * n : n;
  LinBackwardLayout l;
  const bool wide = lin_wide_tiles(dtype, rows, k, false) + lin_wide_tiles(dtype, n2, k, false) >= num_cus();
  lin_tile_shape(l.dx, dtype, wide);
  lin_tile_shape(l.dw, dtype, wide);
  lin_split_plan(l.dx, rows, k, n2, false, lin_tiles(n2, k, false, l.dw.bi, l.dw.bj));
  lin_split_plan(l.dw, n2, k, rows, false, lin_tiles(rows, k, false, l.dx.bi, l.dx.bj));
  const long per = lin_dz_rows(rows, n);
  l.dz = 0;
  l.sums = l.dz + (gated || act != kActNone ? lin_pad((size_t)rows * lin_ld(dtype, n2) * lin_size(dtype)) : lin_pad_bytes(dtype, rows, n2));
  l.w = l.sums + lin_pad((size_t)((rows + per - 1) / per) * n2 * 4);
  l.x = l.w + lin_pad_bytes(dtype, n2, k);
  l.part_dx = l.x + lin_pad_bytes(dtype, rows, k);
  l.part_dw = l.part_dx + l.dx.part_bytes;
  l.total = l.part_dw + l.dw.part_bytes;
  return l;
}
template <class T, bool GATED, class Launcher>
int lin_backward_t(Launcher& L, int dtype, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw, void* db, char* ws,
                   const LinBackwardLayout& l, long rows, int k, int n, int act) {
  const int n2 = GATED ? 2 * n : n, ldz = lin_ld(dtype, n2), ldk = lin_ld(dtype, k);
  const bool act_pass = GATED || act != kActNone;
  LinPairArgs q = {};
  const long per = lin_dz_rows(rows, n), row_blocks = (rows + per - 1) / per;
  if (act_pass || db) {
    LinDzArgs a = {};
    a.dy = dy; a.pre = act_pass ? pre : nullptr; a.dz = act_pass ? ws + l.dz : nullptr; a.ld_dz = ldz;
    a.part = db ? reinterpret_cast<float*>(ws + l.sums) : nullptr;
    a.rows = rows; a.n = n; a.act = act; a.rows_per_block = (int)per; a.vec = n % 8 == 0;
    const long blocks = (long)((n + 255) / 256) * row_blocks;
    if (int rc = lin_grid_check(blocks)) return rc;
    if (int rc = L.launch(lin_dz_kernel<T, GATED>, (int)blocks, 256, a)) return rc;
  }
  LinPadder pad, pad_dy;
  const void* dz = act_pass ? ws + l.dz : (dx || dw ? pad_dy.add(dtype, dy, rows, n2, ws + l.dz) : dy);
  const void* wp = dx ? pad.add(dtype, w, n2, k, ws + l.w) : nullptr;
  const void* xp = dw ? pad.add(dtype, x, rows, k, ws + l.x) : nullptr;
  if (int rc = pad_dy.launch(L)) return rc;
  if (int rc = pad.launch(L)) return rc;

  long joins_dx = 0, joins_dw = 0;
  if (dx) {
    LinGemmArgs& p = q.dx;
    p.a = dz; p.b = wp; p.rows_i = rows; p.rows_j = k; p.kk = n2; p.lda = ldz; p.ldb = ldk; p.out = dx; p.vec = k % 8 == 0;
    lin_apply(p, l.dx, reinterpret_cast<float*>(ws + l.part_dx));
    const long b = (l.dx.tiles * p.splits + 7) / 8 * 8;
    if (int rc = lin_grid_check(b)) return rc;
    q.blocks_dx = (int)b;
    if (p.splits > 1) joins_dx = lin_join_blocks(p, false);
  }
  if (dw) {
    LinGemmArgs& p = q.dw;
    p.a = dz; p.b = xp; p.rows_i = n2; p.rows_j = k; p.kk = rows; p.lda = ldz; p.ldb = ldk; p.out = dw; p.vec = k % 8 == 0;
    lin_apply(p, l.dw, reinterpret_cast<float*>(ws + l.part_dw));
    const long b = (l.dw.tiles * p.splits + 7) / 8 * 8;
    if (int rc = lin_grid_check(b)) return rc;
    q.blocks_dw = (int)b;
    if (p.splits > 1) joins_dw = lin_join_blocks(p, false);
  }
  q.sums = reinterpret_cast<const float*>(ws + l.sums); q.db = db; q.sum_rows = (int)row_blocks; q.sum_cols = n2;
  const long grid = (long)q.blocks_dx + q.blocks_dw + (db ? (n2 + 127) / 128 : 0);
  if (grid == 0) return 0;
  if (int rc = lin_grid_check(grid > joins_dx + joins_dw ? grid : joins_dx + joins_dw)) return rc;
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (l.dx.wide) rc = L.launch(lin_dma_pair_kernel<LinD256, T>, (int)grid, LinD256::NT, q);
    else rc = L.launch(lin_dma_pair_kernel<LinD128, T>, (int)grid, LinD128::NT, q);
  } else {
    if (l.dx.wide) rc = L.launch(lin_split_pair_kernel<LinF256>, (int)grid, LinF256::NT, q);
    else rc = L.launch(lin_split_pair_kernel<LinF128>, (int)grid, LinF128::NT, q);
  }
  if (rc || joins_dx + joins_dw == 0) return rc;
  q.blocks_dx = (int)joins_dx;
  q.blocks_dw = (int)joins_dw;
  return L.launch(lin_join_pair_kernel<T>, (int)(joins_dx + joins_dw), 256, q);
}

inline int lin_check(const char* what, long rows, int k, int n, int act, int dtype, bool gated) {
  if (dtype < 0 || dtype > 2) TNV3_FAIL(-1, "%s: dtype %d is none of 0 (fp32), 1 (bf16), 2 (fp16)", what, dtype);
  if (act < 0 || act >= kActCount) TNV3_FAIL(-1, "%s: unknown activation %d", what, act);
  if (rows < 1 || k < 1 || n < 1) TNV3_FAIL(-1, "%s: sizes must be positive (rows %ld, k %d, n %d)", what, rows, k, n);
  if (rows > kLinMaxRows || k > kLinMaxWidth || (gated ? 2l * n : (long)n) > kLinMaxWidth)
    TNV3_FAIL(-1, "%s: rows %ld / widths %d, %d beyond 2^30 / 2^20", what, rows, k, n);
  return 0;
}

// every tensor on a 16-byte boundary (nulls are)
template <class... P> inline bool lin_all_aligned(P... p) { return ((((uintptr_t)p & 15) == 0) && ...); }

inline size_t lin_forward_workspace_bytes(long rows, int k, int n, int dtype, bool gated) {
  if (lin_check("workspace", rows, k, n, 0, dtype, gated)) return 0;
  return lin_forward_layout(rows, k, gated ? 2 * n : n, dtype, gated).total;
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
  if (!lin_all_aligned(x, w, bias, res, out, pre, ws)) TNV3_FAIL(-1, "%s: tensors must be 16-byte aligned", what);
  const LinForwardLayout l = lin_forward_layout(rows, k, GATED ? 2 * n : n, dtype, GATED);
  if (l.total && (!ws || ws_bytes < l.total)) TNV3_FAIL(-1, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, l.total);
  char* wsc = static_cast<char*>(ws);
  switch (dtype) {
    case kLinF32: return lin_forward_t<float, GATED>(L, dtype, x, w, bias, res, out, pre, wsc, l, rows, k, n, act);
    case kLinBf16: return lin_forward_t<LinBf16, GATED>(L, dtype, x, w, bias, res, out, pre, wsc, l, rows, k, n, act);
    default: return lin_forward_t<LinF16, GATED>(L, dtype, x, w, bias, res, out, pre, wsc, l, rows, k, n, act);
  }
}
template <bool GATED, class Launcher>
int lin_backward_impl(Launcher& L, const void* dy, const void* x, const void* w, const void* pre, void* dx, void* dw, void* db, void* ws, size_t ws_bytes,
                      long rows, int k, int n, int act, int dtype) {
  const char* what = GATED ? "gated_linear_backward" : "linear_backward";
  if (int rc = lin_check(what, rows, k, n, act, dtype, GATED)) return rc;
  if (!dy || (dx && !w) || (dw && !x)) TNV3_FAIL(-1, "%s: null tensor", what);
  if ((GATED || act != kActNone) && !pre) TNV3_FAIL(-1, "%s: the forward's pre-activation is required", what);
  if (!lin_all_aligned(dy, x, w, pre, dx, dw, db, ws)) TNV3_FAIL(-1, "%s: tensors must be 16-byte aligned", what);
  const LinBackwardLayout l = lin_backward_layout(rows, k, n, act, dtype, GATED);
  if (!ws || ws_bytes < l.total) TNV3_FAIL(-1, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, l.total);
  char* wsc = static_cast<char*>(ws);
  switch (dtype) {
    case kLinF32: return lin_backward_t<float, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
    case kLinBf16: return lin_backward_t<LinBf16, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
    default: return lin_backward_t<LinF16, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
  }
}

}  // namespace tnv3

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
// products of few tiles, whose operands come from memory rather than a cache: four LDS stages, so that three steps' loads are in flight (two stages:
// 200 x 4096 -> 8192 in bf16 51 us instead of 29, 200 x 4096 -> 4096 32 instead of 21, the gradient of 1024 x 4096 alone 55 instead of 42)
using LinD128x4 = LinDmaCfg<2, 2, 2, 2, 4>;     // 128 x 128, one workgroup per CU
using LinD64 = LinDmaCfg<1, 2, 2, 1, 4>;        // 64 x 64, two waves of 32 x 64, two workgroups per CU (forward)
using LinF256 = LinSplitCfg<2, 2, 4, 2>;        // fp32: 256 x 128, eight waves of 64 x 64, one workgroup per CU (144 KB of LDS)
using LinF128 = LinSplitCfg<1, 2, 4, 1>;        // fp32: 128 x 64, four waves of 32 x 64, two workgroups per CU

constexpr long kLinMaxWidth = 1l << 20;         // columns: a tile's rows stay within 2^31 bytes of its first
constexpr long kLinMaxRows = 1l << 30;

inline size_t lin_pad(size_t b) { return (b + 255) & ~(size_t)255; }
inline int lin_size(int dtype) { return dtype == kLinF32 ? 4 : 2; }

// One product's tiling.  Sizes and type decide, never the pointers, so that the workspace queries and the launches agree.
enum { kTileSmall = 0, kTileDeep = 1, kTileNormal = 2, kTileWide = 3 };
struct LinPlan {
  int tile, bi, bj, splits;
  long k_per_split, tiles;
  size_t part_bytes;
  double time;              // expected, us
};
inline long lin_tiles(long rows_i, long rows_j, bool gated, int bi, int bj) {
  return ((rows_i + bi - 1) / bi) * (gated ? (rows_j / 2 + bj / 2 - 1) / (bj / 2) : (rows_j + bj - 1) / bj);
}
// What a launch takes, in microseconds, from timings of 16 to 4096 tiles at contractions of 256 to 2048 on 256 CUs: a workgroup's 64 of the contraction
// take `lat` alone on its CU and `thr` of the CU's time among others, `occ` of them share a CU, a launch costs `fix`, a further round of
// workgroups `again`.  16-bit, per 64: 64 x 64 tiles 0.27 alone, 0.42 with two a CU; 128 x 128 with four stages 0.47-0.52; with two stages 0.40-0.8
// alone with operands in a cache, 0.87 from memory, 3.1 with 8 a CU; 256 x 256 1.1-1.8, 6.1 with 4 a CU.  fp32: 128 x 64 1.7-2.2, 12.6 with 8 a CU;
// 256 x 128 3.4-4.4, 18.8 with 4 a CU.  Adding the parts of a split contraction: a launch of 2 and its bytes at 4.5 TB/s.
struct LinCost { int bi, bj, occ; double thr, lat, fix, again; };
inline const LinCost& lin_cost(int dtype, int tile) {
  static const LinCost t[2][4] = {{{64, 64, 2, 0.21, 0.27, 4.0, 1.0}, {128, 128, 1, 0.49, 0.49, 6.0, 4.0}, {128, 128, 2, 0.45, 0.8, 5.0, 2.0},
                                   {256, 256, 1, 1.55, 1.55, 8.0, 4.0}},
                                  {{0, 0, 0, 0, 0, 0, 0}, {0, 0, 0, 0, 0, 0, 0}, {128, 64, 2, 1.6, 1.9, 4.0, 1.5}, {256, 128, 1, 4.5, 4.5, 9.0, 4.0}}};
  return t[dtype == kLinF32 ? 1 : 0][tile];
}
inline double lin_steps_time(const LinCost& c, long groups, long steps) {
  const long per = (groups + num_cus() - 1) / num_cus(), full = per / c.occ, rem = per % c.occ;
  const double whole = c.occ * c.thr > c.lat ? c.occ * c.thr : c.lat, part = rem * c.thr > c.lat ? rem * c.thr : c.lat;
  return c.fix + steps * (full * whole + (rem ? part : 0.0)) + c.again * (full + (rem ? 1 : 0) - 1);
}
constexpr int kLinSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
inline double lin_join_bytes(long rows_i, long rows_j, long s) { return s > 1 ? 8.0 * s * rows_i * rows_j : 0.0; }
inline double lin_join_time(double bytes) { return bytes > 0 ? 2.0 + bytes / 4.5e6 : 0.0; }
inline void lin_set_plan(LinPlan& pl, int dtype, int tile, long rows_i, long rows_j, long kk, bool gated, long s) {
  const LinCost& c = lin_cost(dtype, tile);
  pl.tile = tile;
  pl.bi = c.bi;
  pl.bj = c.bj;
  pl.tiles = lin_tiles(rows_i, rows_j, gated, c.bi, c.bj);
  const long steps = (kk + 63) / 64, per = (steps + s - 1) / s;
  pl.splits = (int)((steps + per - 1) / per);
  pl.k_per_split = per * 64;
  pl.part_bytes = pl.splits > 1 ? lin_pad((size_t)pl.splits * rows_i * rows_j * 4) : 0;
}
// one product: the tile (smallest_tile or larger) and the number of parts of the contraction with the least expected time
inline LinPlan lin_plan(int dtype, long rows_i, long rows_j, long kk, bool gated, int smallest_tile) {
  LinPlan pl;
  double best = 0;
  int tile = kTileNormal;
  long split = 0;
  const long steps = (kk + 63) / 64;
  for (int t = smallest_tile; t <= kTileWide; ++t) {
    const LinCost& c = lin_cost(dtype, t);
    const long tiles = lin_tiles(rows_i, rows_j, gated, c.bi, c.bj);
    for (long s : kLinSplits) {
      if (s > 1 && (s > steps || tiles * s > 4 * num_cus())) break;
      const double e = lin_steps_time(c, tiles * s, (steps + s - 1) / s) + lin_join_time(lin_join_bytes(rows_i, rows_j, s));
      if (split == 0 || e < best) { best = e; tile = t; split = s; }
    }
  }
  lin_set_plan(pl, dtype, tile, rows_i, rows_j, kk, gated, split);
  pl.time = best;
  return pl;
}
// the smallest tile of a backward pass
inline int lin_backward_tile(int dtype) { return dtype == kLinF32 ? kTileNormal : kTileDeep; }
// The two products of a backward pass in one launch: the longest workgroup and the work per CU bound the time; the product with the longest
// workgroups is split further as long as that helps.
inline void lin_pair_plan(LinPlan& dx, LinPlan& dw, int dtype, long rows, int k, int n2) {
  const long ri[2] = {rows, n2}, steps[2] = {((long)n2 + 63) / 64, (rows + 63) / 64};
  double best = -1;
  int tile = kTileNormal;
  int choice[2] = {0, 0};
  for (int t = lin_backward_tile(dtype); t <= kTileWide; ++t) {
    const LinCost& c = lin_cost(dtype, t);
    const long tiles[2] = {lin_tiles(ri[0], k, false, c.bi, c.bj), lin_tiles(ri[1], k, false, c.bi, c.bj)};
    int at[2] = {0, 0};
    for (;;) {
      const long s[2] = {kLinSplits[at[0]], kLinSplits[at[1]]}, n[2] = {(steps[0] + s[0] - 1) / s[0], (steps[1] + s[1] - 1) / s[1]};
      const long groups = tiles[0] * s[0] + tiles[1] * s[1], per = (groups + num_cus() - 1) / num_cus();
      const double share = (per < c.occ ? per : c.occ) * c.thr, each = share > c.lat ? share : c.lat;
      const int longer = n[0] >= n[1] ? 0 : 1;
      const double longest = n[longer] * each;
      const double work = (tiles[0] * s[0] * (n[0] * c.thr + c.again / c.occ) + tiles[1] * s[1] * (n[1] * c.thr + c.again / c.occ)) / num_cus();
      // one round of workgroups: the longest; several: the work, and on average a part of the longest in which CUs run dry
      double e = groups <= (long)num_cus() * c.occ || work + 0.4 * longest < longest ? longest : work + 0.4 * longest;
      e += c.fix + lin_join_time(lin_join_bytes(ri[0], k, s[0]) + lin_join_bytes(ri[1], k, s[1]));
      if (best < 0 || e < best) { best = e; tile = t; choice[0] = at[0]; choice[1] = at[1]; }
      if (at[longer] + 1 >= (int)(sizeof(kLinSplits) / sizeof(int)) || kLinSplits[at[longer] + 1] > steps[longer] || groups > 8 * num_cus()) break;
      ++at[longer];
    }
  }
  lin_set_plan(dx, dtype, tile, rows, k, n2, false, kLinSplits[choice[0]]);
  lin_set_plan(dw, dtype, tile, n2, k, rows, false, kLinSplits[choice[1]]);
}
inline void lin_apply(LinGemmArgs& p, const LinPlan& pl, float* part) {
  p.splits = pl.splits;
  p.k_per_split = pl.k_per_split;
  p.tiles_i = (int)((p.rows_i + pl.bi - 1) / pl.bi);
  p.tiles_j = (int)(pl.tiles / p.tiles_i);
  p.part = part;
}
inline long lin_join_blocks(const LinGemmArgs& p, bool gated) { return (p.rows_i * (((gated ? (long)p.f : p.rows_j) + 7) / 8) + 255) / 256; }
// a launch counts its work-items in 32 bits
inline int lin_grid_check(long blocks, int threads) {
  if (blocks >= (1l << 32) / threads) TNV3_FAIL(-1, "linear: %ld workgroups of %d are more than one launch takes", blocks, threads);
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
    if (int rc = lin_grid_check(blocks, 256)) return rc;
    return L.launch(lin_pad_kernel, (int)blocks, 256, a);
  }
};

// ---- forward
constexpr long kLinFewRows = 64;       // the largest number that lin_rows_kernel takes
// Few rows: up to 16 the weight's bytes are the bound and lin_rows_kernel it is.  Beyond, its workgroups of 16 weight rows read all of x each, 55 KB per us
// and CU (64 x 8192 -> 1024 in bf16 21.6 us, 64 x 4096 -> 8192 27.5), which tiles of 64 rows do not (12.7, 20.6); but those pay for joining their parts and
// for copies of odd widths (64 x 2048 -> 2048 9.2 against 9.7, 64 x 1003 -> 1337 7.6 against 12.7).
inline double lin_rows_time(long rows, int k, int n2, int dtype, bool gated) {
  const long of = 128 / lin_size(dtype), blocks = (k + of - 1) / of, groups = (n2 / (gated ? 2 : 1) + 15) / 16;
  const long staged = 8 * ((gated ? 32 : 16) + (rows <= 32 ? 32 : 64)) * 128;                // bytes of a round of a workgroup's 8 waves
  return 3.5 + (double)((blocks + 7) / 8) * ((groups + num_cus() - 1) / num_cus()) * staged / 55e3;
}
struct LinForwardLayout { LinPlan plan; size_t x, w, part, total; bool few; };
inline LinForwardLayout lin_forward_layout(long rows, int k, int n2, int dtype, bool gated) {
  LinForwardLayout l = {};
  l.few = rows <= 16;
  if (l.few) return l;
  l.plan = lin_plan(dtype, rows, n2, k, gated, dtype == kLinF32 ? kTileNormal : kTileSmall);
  l.x = 0;
  l.w = l.x + lin_pad_bytes(dtype, rows, k);
  l.part = l.w + lin_pad_bytes(dtype, n2, k);
  l.total = l.part + l.plan.part_bytes;
  if (rows <= kLinFewRows) {
    const double weight = 2.0 + (double)n2 * k * lin_size(dtype) / 4.7e6, join = lin_join_time(lin_join_bytes(rows, n2, l.plan.splits));
    const double tiles = (l.plan.time - join > weight ? l.plan.time - join : weight) + join + (l.part ? 3.0 + 2.0 * l.part / 4.5e6 : 0.0);
    if (tiles > 0.9 * lin_rows_time(rows, k, n2, dtype, gated)) {
      l = {};
      l.few = true;
    }
  }
  return l;
}
template <class T, bool GATED, class Launcher>
int lin_forward_t(Launcher& L, int dtype, const void* x, const void* w, const void* bias, const void* res, void* out, void* pre, char* ws,
                  const LinForwardLayout& l, long rows, int k, int n, int act) {
  LinGemmArgs p = {};
  const int n2 = GATED ? 2 * n : n;
  p.a = x; p.b = w; p.rows_i = rows; p.rows_j = n2; p.kk = k; p.lda = p.ldb = k; p.splits = 1;
  p.bias = bias; p.res = res; p.out = out; p.pre = pre; p.act = act; p.f = GATED ? n : 0;
  if (l.few) {
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
  const long grid = l.plan.tiles * p.splits, join = p.splits > 1 ? lin_join_blocks(p, GATED) : 0;
  if (int rc = lin_grid_check(grid, 512)) return rc;
  if (int rc = lin_grid_check(join, 256)) return rc;
  if (int rc = pad.launch(L)) return rc;
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (l.plan.tile == kTileWide) rc = L.launch(lin_dma_kernel<LinD256, T, GATED>, (int)grid, LinD256::NT, p);
    else if (l.plan.tile == kTileSmall) rc = L.launch(lin_dma_kernel<LinD64, T, GATED>, (int)grid, LinD64::NT, p);
    else if (l.plan.tile == kTileDeep) rc = L.launch(lin_dma_kernel<LinD128x4, T, GATED>, (int)grid, LinD128x4::NT, p);
    else rc = L.launch(lin_dma_kernel<LinD128, T, GATED>, (int)grid, LinD128::NT, p);
  } else {
    if (l.plan.tile == kTileWide) rc = L.launch(lin_split_kernel<LinF256, GATED>, (int)grid, LinF256::NT, p);
    else rc = L.launch(lin_split_kernel<LinF128, GATED>, (int)grid, LinF128::NT, p);
  }
  if (rc || p.splits == 1) return rc;
  return L.launch(lin_join_kernel<T, GATED>, (int)join, 256, p);
}

// ---- backward: dz (with the bias gradient's partial sums), then both products in one launch
// row blocks of the element-wise pass: about four workgroups per CU, at least 8 rows (one per work-item) each, and no more blocks than the final column
// sums can add quickly
inline long lin_dz_rows(long rows, int n) {
  const long jt = (n + 255) / 256, cap = rows / 128 < 256 ? 256 : (rows / 128 > 512 ? 512 : rows / 128);
  long blocks = 4l * num_cus() / jt;
  blocks = blocks < 1 ? 1 : (blocks > cap ? cap : blocks);
  const long per = ((rows + blocks - 1) / blocks + 7) / 8 * 8;
  return per < 8 ? 8 : per;
}
struct LinBackwardLayout { LinPlan dx, dw; size_t dz, sums, w, x, part_dx, part_dw, total; };
// for the products that are wanted (the unwanted one's plan is empty)
inline LinBackwardLayout lin_backward_layout(long rows, int k, int n, int act, int dtype, bool gated, bool dx, bool dw) {
  const int n2 = gated ? 2 * n : n;
  LinBackwardLayout l = {};
  if (dx && dw) lin_pair_plan(l.dx, l.dw, dtype, rows, k, n2);
  else if (dx) l.dx = lin_plan(dtype, rows, k, n2, false, lin_backward_tile(dtype));
  else if (dw) l.dw = lin_plan(dtype, n2, k, rows, false, lin_backward_tile(dtype));
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
    a.rows = rows; a.n = n; a.act = act; a.rows_per_block = (int)per;
    const long blocks = (long)((n + 255) / 256) * row_blocks;
    if (int rc = lin_grid_check(blocks, 256)) return rc;
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
    p.a = dz; p.b = wp; p.rows_i = rows; p.rows_j = k; p.kk = n2; p.lda = ldz; p.ldb = ldk; p.out = dx;
    lin_apply(p, l.dx, reinterpret_cast<float*>(ws + l.part_dx));
    const long b = (l.dx.tiles * p.splits + 7) / 8 * 8;
    if (int rc = lin_grid_check(b, 512)) return rc;
    q.blocks_dx = (int)b;
    if (p.splits > 1) joins_dx = lin_join_blocks(p, false);
  }
  if (dw) {
    LinGemmArgs& p = q.dw;
    p.a = dz; p.b = xp; p.rows_i = n2; p.rows_j = k; p.kk = rows; p.lda = ldz; p.ldb = ldk; p.out = dw;
    lin_apply(p, l.dw, reinterpret_cast<float*>(ws + l.part_dw));
    const long b = (l.dw.tiles * p.splits + 7) / 8 * 8;
    if (int rc = lin_grid_check(b, 512)) return rc;
    q.blocks_dw = (int)b;
    if (p.splits > 1) joins_dw = lin_join_blocks(p, false);
  }
  q.sums = reinterpret_cast<const float*>(ws + l.sums); q.db = db; q.sum_rows = (int)row_blocks; q.sum_cols = n2;
  const long grid = (long)q.blocks_dx + q.blocks_dw + (db ? (n2 + 127) / 128 : 0);
  if (grid == 0) return 0;
  const int tile = dx ? l.dx.tile : (dw ? l.dw.tile : kTileNormal);
  if (int rc = lin_grid_check(grid, 512)) return rc;
  if (int rc = lin_grid_check(joins_dx + joins_dw, 256)) return rc;
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (tile == kTileWide) rc = L.launch(lin_dma_pair_kernel<LinD256, T>, (int)grid, LinD256::NT, q);
    else if (tile == kTileDeep) rc = L.launch(lin_dma_pair_kernel<LinD128x4, T>, (int)grid, LinD128x4::NT, q);
    else rc = L.launch(lin_dma_pair_kernel<LinD128, T>, (int)grid, LinD128::NT, q);
  } else {
    if (tile == kTileWide) rc = L.launch(lin_split_pair_kernel<LinF256>, (int)grid, LinF256::NT, q);
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
  size_t most = 0;
  for (int want = 1; want < 4; ++want) {
    const size_t t = lin_backward_layout(rows, k, n, act, dtype, gated, want & 1, want & 2).total;
    most = t > most ? t : most;
  }
  return most;
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
  const LinBackwardLayout l = lin_backward_layout(rows, k, n, act, dtype, GATED, dx != nullptr, dw != nullptr);
  if (!ws || ws_bytes < l.total) TNV3_FAIL(-1, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, l.total);
  char* wsc = static_cast<char*>(ws);
  switch (dtype) {
    case kLinF32: return lin_backward_t<float, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
    case kLinBf16: return lin_backward_t<LinBf16, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
    default: return lin_backward_t<LinF16, GATED>(L, dtype, dy, x, w, pre, dx, dw, db, wsc, l, rows, k, n, act);
  }
}

}  // namespace tnv3

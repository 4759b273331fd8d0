// linear_dma.h -- the wide products of 16-bit operands: tiles move from memory to LDS by direct loads, nothing passes through registers on the way.
//
// A workgroup of WM x WN waves computes (TM 32 WM) x (TN 32 WN) outputs, 64 of the contraction per step, two LDS stages (NS in general: NS - 1
// steps of loads are in flight, counted waits).  A wave owns 2 TM x 2 TN MFMA tiles (16x16x32).
// One barrier per step, placed before the LAST quarter of a step's products: at that point every wave has the step's last fragments in
// registers and its share of the next stage has landed, so behind the barrier the stage just read can be refilled (a whole step for the loads to
// arrive) and the next step's first fragments are read under the last quarter's products.  No product waits for a read that was not issued a
// quarter step (16, 8 or 4 MFMAs of 16 cycles per wave; two waves per SIMD with two stages, one with four) earlier.
#pragma once
#include "linear_common.h"

namespace tnv3 {

template <int TM_, int TN_, int WM_, int WN_, int NS_ = 2>
struct LinDmaCfg {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr int NS = NS_;                                                // LDS stages: NS - 1 steps of loads are in flight
  static constexpr int NW = WM * WN, NT = NW * 64, BI = TM * 32 * WM, BJ = TN * 32 * WN, BK = 64;
  static constexpr int STAGE = (BI + BJ) * BK;                                  // 16-bit elements
  static constexpr int SLABS = NW * kLinSlabFloats * 2;
  static constexpr int LDS = NS * STAGE > SLABS ? NS * STAGE : SLABS;
};

// One operand's direct loads: a wave moves ROWS / 8 / NW pieces of 1 KB per step (64 lanes x 16 bytes, consecutive in LDS; the lane picks the chunk
// that belongs there).  k-contiguous: 8 rows of 64; k-strided: 512 / ROWS rows of k.
template <bool KS, int ROWS, int NW>
struct LinDma {
  static constexpr int N = ROWS / 8 / NW;
  static_assert(N * 8 * NW == ROWS, "whole pieces per wave");
  unsigned off[N];          // bytes from the operand's first element of the step
  int kchunk;               // k-contiguous: first k of the lane's chunk in its even pieces
  const char* base;
  long left;                // bytes from base to the operand's end
  long step;                // bytes per step
  // base_el: the tile's first element; end_el: the operand's element count; row_off: rows to add to this wave's pieces
  __device__ __forceinline__ void init(const void* src, long base_el, long end_el, long ld, int wave, int lane) {
    base = static_cast<const char*>(src) + 2 * base_el;
    left = 2 * (end_el - base_el);
    step = KS ? 128 * ld : 128;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int piece = wave * N + i;
      if (KS) {
        constexpr int LPR = ROWS / 8;
        static_assert(!KS || ROWS >= 128, "lin_pos_ks16's order");
        const int k = piece * (64 / LPR) + lane / LPR, c = (lane % LPR) ^ (((k & 3) << 2) | ((k & 8) >> 2));
        off[i] = (unsigned)(k * (int)(2 * ld) + c * 16);
      } else {
        static_assert(N % 2 == 0, "piece i of a wave is odd where i is");
        const int r = lane >> 3, c = (lane & 7) ^ (r >> 1) ^ ((i & 1) << 2);            // lin_pos_kc's order
        off[i] = (unsigned)((piece * 8 + r) * (int)(2 * ld) + c * 16);
        if (i == 0) kchunk = c * 8;
      }
    }
  }
  // the step's descriptor; then the next step's base
  __device__ __forceinline__ tnv3_rsrc_t begin() {
    const tnv3_rsrc_t r = tnv3_make_rsrc(base, lin_range(left));
    base += step;
    left -= step;
    return r;
  }
  // piece i; kleft: elements of the contraction left in this split from the step's first on (none: zeros arrive)
  __device__ __forceinline__ void piece(tnv3_rsrc_t r, unsigned short* tile, int i, int kleft, int wave) {
    tnv3_buf_dma16(r, reinterpret_cast<float*>(tile + (wave * N + i) * 512), (KS ? 0 : kchunk ^ ((i & 1) << 5)) >= kleft ? kDmaOob : off[i]);
  }
};

// this wave's loads but for the newest LEAVE have landed, its fragments are in registers
template <int LEAVE> __device__ __forceinline__ void lin_dma_sync() {
  static_assert(LEAVE < 64, "vmcnt's range");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070 | (LEAVE & 15) | (LEAVE >> 4) << 14);              // vmcnt(LEAVE) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

template <class Cfg, class T, bool KSA, bool KSB, bool GATED>
__device__ __forceinline__ void lin_dma_product(const LinGemmArgs& p, int block, unsigned short* lds) {
  constexpr int TM = Cfg::TM, TN = Cfg::TN, BI = Cfg::BI, BJ = Cfg::BJ, BK = Cfg::BK, STAGE = Cfg::STAGE, NS = Cfg::NS, Q = BK / 16;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / Cfg::WN, wj = wave % Cfg::WN;
  int ti, tj, sp;
  if (!lin_tile(p, block, ti, tj, sp)) return;
  const long i0 = (long)ti * BI, j0 = (long)tj * (GATED ? BJ / 2 : BJ);
  const long kbeg = (long)sp * p.k_per_split, kend = kbeg + p.k_per_split < p.kk ? kbeg + p.k_per_split : p.kk;
  const int steps = kend > kbeg ? (int)((kend - kbeg + BK - 1) / BK) : 0;

  LinDma<KSA, BI, Cfg::NW> da;
  LinDma<KSB, BJ, Cfg::NW> db;
  da.init(p.a, KSA ? kbeg * p.lda + i0 : i0 * p.lda + kbeg, KSA ? p.kk * p.lda : p.rows_i * p.lda, p.lda, wave, lane);
  if (GATED) {
    // tile row r holds weight row (r / H odd ? f : 0) + j0 + (r / 2H) H + r % H, H = TN 16: a wave's pieces lie in one run of H rows, so the jump is
    // in its base
    constexpr int H = TN * 16, N8 = LinDma<KSB, BJ, Cfg::NW>::N * 8;
    static_assert(!GATED || H % N8 == 0, "a wave's pieces stay within one half");
    const int r0 = wave * N8, run = r0 / H;
    const long row = j0 + (long)(run >> 1) * H + (run & 1 ? p.f : 0) - (long)run * H;        // so that base + r0 rows is the wave's first row
    db.init(p.b, row * p.ldb + kbeg, p.rows_j * p.ldb, p.ldb, wave, lane);
  } else {
    db.init(p.b, KSB ? kbeg * p.ldb + j0 : j0 * p.ldb + kbeg, KSB ? p.kk * p.ldb : p.rows_j * p.ldb, p.ldb, wave, lane);
  }
  // the stage being filled: its descriptors, what is left of the contraction there
  int kleft = (int)(kend - kbeg);
  tnv3_rsrc_t ra, rb;
  int kl = 0;
  auto begin = [&]() {
    ra = da.begin();
    rb = db.begin();
    kl = kleft > 0 ? kleft : 0;
    kleft -= BK;
  };
  constexpr int NA = LinDma<KSA, BI, Cfg::NW>::N, NP = NA + LinDma<KSB, BJ, Cfg::NW>::N;
  auto piece = [&](unsigned short* into, int i) {
    if (i >= NP) return;
    if (i < NA) da.piece(ra, into, i, kl, wave);
    else db.piece(rb, into + BI * BK, i - NA, kl, wave);
  };

  // Quarter q of a step: 32 of the contraction (q / 2) for half of the wave's columns (q % 2).  16x16x32 products: the larger form writes and reads
  // twice the accumulator bytes per product, and at full tilt the card's power, not the issue of products, is the limit.
  constexpr int XM = 2 * TM, YN = 2 * TN;             // 16-row / 16-column tiles of the wave
  f32x4 acc[XM][YN];
#pragma unroll
  for (int x = 0; x < XM; ++x)
#pragma unroll
    for (int y = 0; y < YN; ++y) acc[x][y] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

  lin_s8 fa[2][XM], fb[2][TN];
  LinFrag16<KSA, BI> ga;
  LinFrag16<KSB, BJ> gb;
  ga.init(wi * TM * 32, lane);
  gb.init(wj * TN * 32, lane);
  auto read = [&](const unsigned short* t, int q) {
    // (opaque: an exclusive-or per fragment stays where it is instead of occupying a register per address across the loop)
    if (KSA) TNV3_OPAQUE_V(ga.off[0]);
    if (KSB) TNV3_OPAQUE_V(gb.off[0]);
    if (q % 2 == 0) {
#pragma unroll
      for (int x = 0; x < XM; ++x) fa[q / 2][x] = ga.get(t, x, q / 2);
    }
#pragma unroll
    for (int y = 0; y < TN; ++y) fb[q % 2][y] = gb.get(t + BI * BK, (q % 2) * TN + y, q / 2);
  };
  // the products of one quarter, PQ pieces of direct loads (first .. first + PQ - 1) between them: a wave's loads queue behind those of the CU's other
  // waves (16 clocks of the address path each), so they are spread over two quarters instead of standing in front of the products
  constexpr int PQ = 4, GAP = XM * TN / PQ;
  static_assert(Q == 4 && NP <= 2 * PQ && GAP > 0, "a stage's pieces: two quarters");
  auto products = [&](int q, unsigned short* into, int first) {
#pragma unroll
    for (int y = 0; y < TN; ++y)
#pragma unroll
      for (int x = 0; x < XM; ++x) {
        const int m = y * XM + x;
        f32x4& c = acc[x][(q % 2) * TN + y];
        c = lin_mfma16(fa[q / 2][x], fb[q % 2][y], c, T{});
        if (first >= 0 && m % GAP == GAP - 1 && m / GAP < PQ) {
          __builtin_amdgcn_sched_barrier(0);
          piece(into, first + m / GAP);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
  };
  // From one barrier to the next: the last quarter's products of the step before (its fragments are in registers), then three quarters of this one.
  // Every read is from `rd`, every direct load goes to `wr`, the stage that was read before.  (The qualifiers say so to the compiler, which otherwise lets each
  // transposing read wait for all loads in flight.  The fences keep the reads ahead of the products: left alone, the scheduler puts each read right
  // in front of its use.)
  auto step = [&](const unsigned short* __restrict__ rd, unsigned short* __restrict__ wr, auto first) {
    read(rd, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (decltype(first)::value) {
#pragma unroll
      for (int i = 0; i < PQ; ++i) piece(wr, i);
    } else {
      products(3, wr, 0);
    }
#pragma unroll
    for (int q = 0; q + 1 < Q; ++q) {
      __builtin_amdgcn_sched_barrier(0);
      read(rd, q + 1);
      __builtin_amdgcn_sched_barrier(0);
      products(q, wr, q == 0 ? PQ : -1);
      if (q == 1) begin();                      // the next step's descriptors (beyond the last step: zeros into a stage that is not read)
    }
    lin_dma_sync<(NS - 2) * NP>();
  };
  if (steps > 0) {
#pragma unroll
    for (int st = 0; st < NS - 1; ++st) {
      begin();
#pragma unroll
      for (int i = 0; i < NP; ++i) piece(lds + st * STAGE, i);
    }
    begin();
    lin_dma_sync<(NS - 2) * NP>();
    // (NS steps per turn: the stages' addresses are constants then, nothing is computed between the barrier and the first reads)
    step(lds, lds + (NS - 1) * STAGE, LinFlag<true>{});
    int s = 1;
    for (; s + NS - 1 < steps; s += NS) {
#pragma unroll
      for (int c = 0; c < NS; ++c) step(lds + (c + 1) % NS * STAGE, lds + c * STAGE, LinFlag<false>{});
    }
#pragma unroll
    for (int c = 0; c < NS - 1; ++c)
      if (s + c < steps) step(lds + (c + 1) % NS * STAGE, lds + c * STAGE, LinFlag<false>{});
    products(3, lds, -1);
    if (NS > 2) lin_dma_sync<0>();                // the stages become the write-out's slabs
  }
  auto put = [&](float* slab, int tm, int left, int right) { lin_put16(acc, slab, tm, left, right, lane); };
  lin_write_out<T, TM, TN, GATED, KSB>(p, put, reinterpret_cast<float*>(lds) + wave * kLinSlabFloats, lane, i0 + wi * TM * 32,
                                  j0 + (long)wj * TN * (GATED ? 16 : 32), sp);
}

template <class Cfg, class T, bool GATED>
__global__ void __launch_bounds__(Cfg::NT, 2) lin_dma_kernel(const LinGemmArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned short lds[Cfg::LDS];
  lin_dma_product<Cfg, T, false, false, GATED>(p, blockIdx.x, lds);
}
template <class Cfg, class T>
__global__ void __launch_bounds__(Cfg::NT, 2) lin_dma_pair_kernel(const LinPairArgs p) {
  __shared__ __attribute__((aligned(1024))) unsigned short lds[Cfg::LDS];
  const int b = blockIdx.x, c = b - p.blocks_dx, d = c - p.blocks_dw;
  if (c < 0) lin_dma_product<Cfg, T, false, true, false>(p.dx, b, lds);
  else if (d < 0) lin_dma_product<Cfg, T, true, true, false>(p.dw, c, lds);
  else lin_colsum<T, Cfg::NT>(p.sums, static_cast<T*>(p.db), p.sum_rows, p.sum_cols, d, reinterpret_cast<float*>(lds));
}

}  // namespace tnv3

// ssa_gemm.cuh — a persistent tcgen05 matrix product C[m, n] = sum_k A[m, k] B[n, k] whose epilogue
// is a template argument: the shared core of the linear cross entropy (ssa_linear_ce.cu) and the
// gated feed-forward (ssa_gated_ffn.cu).
//
// A tile is 128 CG rows by BN columns, made by a cluster of CG CTAs. Each CTA holds 128 rows of A and
// BN / CG = 128 rows of B per 64-wide K block in shared memory (32 KB a stage, 6 stages; 48 KB and 4 with NH = 2) and the
// fp32 accumulator of its 128 rows in BN TMEM columns, twice, so that the epilogue of one tile runs
// under the MMAs of the next. CG = 2, BN = 256 is the form for large products: the pair's MMA reads
// both halves of B, so a CTA fetches 32 KB per 4.2 MFLOP where a lone 128 x 256 tile fetches 48 KB.
// CG = 1, BN = 128 is for products with too few such tiles. NH = 2 gives the pair both accumulators
// for one 256 x 512 tile: 48 KB per 8.4 MFLOP, at the price of an epilogue that the next tile's MMAs
// mostly wait for; it is for the long contractions of the gradients.
//
// Roles (320 threads): warp 0 issues TMA loads, warp 1 of the leading CTA issues the MMAs, warps
// 2..9 run the epilogue: two warps per 32 accumulator rows, each with half of the columns. Results
// are exchanged through shared memory so that global accesses are whole 64- or 128-byte row pieces.
//
// Operands are 16-bit matrices in global memory, each either K-major (the contraction index is
// contiguous) or MN-major (the row index m or n is contiguous): a gradient product reads its
// operands in place, with no transposed copy. Both arrive as 64-element (128-byte) wide boxes in
// the 128-byte swizzle; a box past an edge of the matrix reads zeros, so M, N and K are arbitrary.
// Only alignment is asked for: 16-byte base and row stride.
//
// A launch may hold two products (dx and dW of one backward): their tiles are dealt out together,
// the longer ones first, which fills the multiprocessors where each alone leaves a part-filled last
// round.
//
// Every wait is bounded. When one expires, or an earlier launch left the device status set, the
// epilogue runs on NaN accumulators for every tile this CTA still owes, so the failure shows.
#pragma once

#include <cudaTypedefs.h>

#include "ssa_internal.h"
#include "ssa_sm100.cuh"
#include "ssa_tmap.h"

namespace ssa {
namespace sm100 {

// Division of 0 <= n < 2^31 by a fixed d >= 1 as a multiplication (Granlund and Montgomery, "Division
// by invariant integers using multiplication", 1994): with 2^s >= d, n / d = (hi(n m) + n) >> s for
// m = floor(2^32 (2^s - d) / d) + 1.
struct FastDiv {
  uint32_t d, m, s;
};
inline FastDiv fast_div(int d) {
  FastDiv f{(uint32_t)d, 0, 0};
  while ((1ull << f.s) < f.d) ++f.s;
  f.m = (uint32_t)(((1ull << 32) * ((1ull << f.s) - f.d)) / f.d + 1);
  return f;
}
__device__ __forceinline__ int div_by(int n, const FastDiv& f) {
  return (int)((__umulhi((uint32_t)n, f.m) + (uint32_t)n) >> f.s);
}

// mma m16n8k16, fp32 accumulators: c[0], c[1] are row lane / 4, c[2], c[3] row lane / 4 + 8.
template <typename T>
__device__ __forceinline__ void mma_16x8(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                 "{%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One product of a launch (plain data, passed by value).
struct GemmShape {
  int tiles_m, tiles_n;  // tiles of 128 CG rows and BN columns
  int splits;            // contiguous K ranges per tile, each a unit of work
  int kblocks;           // 64-wide K blocks of a tile
  int kb_split;          // K blocks per split
  int band;              // row tiles walked before the column advances (operand reuse in L2)
  int b_kjump_at;        // MN-major B: K blocks from here on read rows b_kjump + 64 (kb - at)
  int b_kjump;
  int a_rows;            // rows of a K-major A's box: 128, or fewer where a lone row tile has fewer
  int b_pair;            // 0, or B is a pair of row blocks this far apart, BN / 2 rows of each
  FastDiv by_splits, by_band, by_rows, by_last;  // splits, tiles of a band, rows of a band, of the last

  void set_divisors() {
    const int last = tiles_m % band;
    by_splits = fast_div(splits);
    by_band = fast_div(band * tiles_n);
    by_rows = fast_div(band);
    by_last = fast_div(last ? last : band);
  }
};

struct GemmUnit {
  int mt, nt, sp, k0, k1;
};

__device__ __forceinline__ GemmUnit gemm_unit(const GemmShape& g, int u) {
  GemmUnit w;
  const int t = div_by(u, g.by_splits);
  w.sp = u - t * g.splits;
  const int bd = div_by(t, g.by_band), r = t - bd * (g.band * g.tiles_n);
  const bool last = (bd + 1) * g.band > g.tiles_m;
  const int rows = last ? (int)g.by_last.d : g.band;
  w.nt = div_by(r, last ? g.by_last : g.by_rows);
  w.mt = bd * g.band + (r - w.nt * rows);
  w.k0 = w.sp * g.kb_split;
  w.k1 = min(g.kblocks, w.k0 + g.kb_split);
  return w;
}

// The products of a launch and how their units are dealt to `workers` clusters: the product with the
// longer units (`lead`) round robin; where its last round is part-filled, each cluster left out
// takes `extra` units of the other first; the rest of the other round robin.
struct GemmWork {
  GemmShape g[2];
  int units0, units1;  // of the leading product, of the other
  int rem, whole;      // units0 over the clusters: part-filled last round, whole rounds
  int lead;
  int extra;
  int turn;            // the cluster at which the last round robin begins: the one with least to do
  unsigned int* status;
};

// The i-th unit of cluster c (below gemm_count): its product in `which`, its index returned.
__device__ __forceinline__ int gemm_deal(const GemmWork& w, int c, int workers, int i, int& which) {
  const int rem = w.rem, mine = w.whole + (c < rem ? 1 : 0);
  which = w.lead;
  if (i < mine) return c + i * workers;
  which = w.lead ^ 1;
  int j = i - mine;
  const int at = c >= w.turn ? c - w.turn : c - w.turn + workers;
  int first = 0;
  if (rem) {
    first = (workers - rem) * w.extra;
    if (c >= rem) {
      if (j < w.extra) return (c - rem) * w.extra + j;
      j -= w.extra;
    }
  }
  return first + at + j * workers;
}

// How many units cluster c has.
__device__ __forceinline__ int gemm_count(const GemmWork& w, int c, int workers) {
  const int rem = w.rem;
  int n = w.whole + (c < rem ? 1 : 0);
  int at = c >= w.turn ? c - w.turn : c - w.turn + workers;  // in the other product's round robin
  if (rem) {
    at += (workers - rem) * w.extra;
    if (c >= rem) n += max(0, min(w.extra, w.units1 - (c - rem) * w.extra));
  }
  return n + (at < w.units1 ? (w.units1 - at - 1) / workers + 1 : 0);
}

template <int CG>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int c0, int c1) {
  if constexpr (CG == 1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  } else {  // into this CTA's memory, counted by the leading CTA's barrier
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address in the cluster's shared window of `addr` (this CTA's window) as seen in CTA `rank`.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What the arrival guards is TMEM, which the tcgen05 fence before it orders: a release at cluster scope
// would also wait for the warp's global stores (a quarter of the stalls of an epilogue warp).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// The pair forms of the TMEM and MMA instructions (both CTAs of the cluster take part).
template <int CG>
__device__ __forceinline__ void tmem_alloc_cg(uint32_t smem_dst, uint32_t ncols) {
  if constexpr (CG == 1) {
    tmem_alloc(smem_dst, ncols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void tmem_dealloc_cg(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 1)
    tmem_dealloc(taddr, ncols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_cg(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                       uint32_t accumulate) {
  if constexpr (CG == 1) {
    mma_ss_lo(d_tmem, a_lo, b_lo, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSW128)
        : "memory");
  }
}
// Arrives on the barrier (in both CTAs of a pair) once the MMAs issued so far have completed.
template <int CG>
__device__ __forceinline__ void mma_commit_cg(uint32_t bar) {
  if constexpr (CG == 1) {
    mma_commit(bar);
  } else {
    const uint16_t both = 3;
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(bar),
        "h"(both)
        : "memory");
  }
}

template <int CG_, int BN_, int NH_>
struct GemmCfg {
  static constexpr int CG = CG_, BM = 128, BN = BN_, NH = NH_, BK = 64;
  static constexpr int HB = BN / CG;   // rows of B in one CTA for one accumulator of BN columns
  static constexpr int RB = NH * HB;
  static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = RB * BK * 2;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr int EPI_WARPS = 8;
  static constexpr uint32_t OFF_EXCH = STAGES * STAGE;  // 4 KB per epilogue warp
  static constexpr uint32_t OFF_BAR = OFF_EXCH + EPI_WARPS * 4096;
  static constexpr uint32_t SMEM_BYTES = OFF_BAR + 256 + 1024;  // + slack for 1 KB alignment
  static constexpr uint32_t TMEM_COLS = 2 * BN;  // two accumulators: of two tiles, or NH = 2 of one
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static_assert(SMEM_BYTES <= 232448, "shared memory of one CTA");
};

// What an epilogue warp works on: accumulator rows row0 .. row0 + 31 of the unit's tile (one per
// lane), half `half` of its columns.
struct EpiCtx {
  uint32_t taddr;   // TMEM address of the accumulator's column 0 in this warp's lanes
  bool failed;
  uint8_t* exch;    // this warp's 4 KB of shared memory
  int lane, quad, half, turn;
  int row0;         // global row of lane 0

  // Accumulator columns [col, col + 32) of this lane's row, in two steps with other work between them
  // (every lane of the warp calls both): start the read, then wait for all reads started.
  __device__ __forceinline__ void fetch(int col, uint32_t (&r)[32]) const {
    if (!failed) {
      tmem_ld32(taddr + (uint32_t)col, r);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = 0x7FC00000u;
    }
  }
  __device__ __forceinline__ void settle() const {
    if (!failed) tmem_ld_wait_only();
  }
  // The values of a read that settle() has waited for.
  __device__ __forceinline__ static void values(uint32_t (&r)[32], float (&v)[32]) {
    tmem_pin(r);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  }
};

// Exchange of a [32 rows x 32 columns] block of 16-bit values within a warp: a lane's row of 64
// bytes on one side, four lanes per row (8 columns each, rows 8 it + lane / 4) on the other. Row r
// keeps its 16-byte pieces in order c ^ (r / 2 % 4), which spreads both sides over all banks.
__device__ __forceinline__ uint4* exch16(uint8_t* buf, int row, int piece) {
  return reinterpret_cast<uint4*>(buf + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
// The same for fp32 (128 bytes a row, eight lanes per row, rows 4 it + lane / 8).
__device__ __forceinline__ float4* exch32(uint8_t* buf, int row, int piece) {
  return reinterpret_cast<float4*>(buf + row * 128 + ((piece ^ (row & 7)) << 4));
}

template <bool BF16>
__device__ __forceinline__ void put_row16(const EpiCtx& e, const float (&v)[32], uint32_t mask) {
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *exch16(e.exch, e.lane, p) = make_uint4(
        pack2<BF16>(v[8 * p], v[8 * p + 1]) & mask, pack2<BF16>(v[8 * p + 2], v[8 * p + 3]) & mask,
        pack2<BF16>(v[8 * p + 4], v[8 * p + 5]) & mask, pack2<BF16>(v[8 * p + 6], v[8 * p + 7]) & mask);
}

// Stores the warp's block of 16-bit values (one row of 32 per lane) to rows base + r * ld of
// columns [col, col + 32), rows and columns below the limits only. base: row 0, column 0.
// vec: base and ld are multiples of 16 bytes. mask: 0 makes this lane's row zeros, whatever its values.
template <bool BF16>
__device__ __forceinline__ void store_block16(const EpiCtx& e, const float (&v)[32], uint16_t* base,
                                              int64_t ld, int rows, int col, int cols, bool vec,
                                              uint32_t mask = 0xffffffffu) {
  put_row16<BF16>(e, v, mask);
  __syncwarp();
  if (vec && col + 32 <= cols) {
    const int p = e.lane & 3;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int r = it * 8 + (e.lane >> 2);
      if (r < rows)
        *reinterpret_cast<uint4*>(base + (int64_t)r * ld + col + 8 * p) = *exch16(e.exch, r, p);
    }
  } else if (col + e.lane < cols) {
    const int n = min(rows, 32);
#pragma unroll 8
    for (int r = 0; r < n; ++r)
      base[(int64_t)r * ld + col + e.lane] =
          reinterpret_cast<const uint16_t*>(exch16(e.exch, r, e.lane >> 3))[e.lane & 7];
  }
  __syncwarp();
}

// Epi: struct with `Args`, `Row`, `static Row row(const Args&, int row)`, which reads what a lane needs
// to know of its row, and `static void tile(const Args&, const GemmUnit&, const Row&, const EpiCtx&)`,
// run by every epilogue warp for each unit; the next unit's rows are read before this one's tile.
// A_MODE: 0 A is K-major, 1 MN-major, 2 K-major in product 0 and MN-major in product 1.
template <class Epi, int CG, int BN, int NH, int A_MODE, bool B_MN, bool BF16>
__global__ void __launch_bounds__(320, 1)
    gemm_sm100_kernel(const __grid_constant__ CUtensorMap tmA0,
                      const __grid_constant__ CUtensorMap tmB0,
                      const __grid_constant__ CUtensorMap tmA1,
                      const __grid_constant__ CUtensorMap tmB1,
                      const __grid_constant__ GemmWork work,
                      const __grid_constant__ typename Epi::Args ea0,
                      const __grid_constant__ typename Epi::Args ea1) {
  using C = GemmCfg<CG, BN, NH>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + C::OFF_BAR;
  auto full = [&](int s) -> uint32_t { return bar0 + 8u * (uint32_t)s; };
  auto empty = [&](int s) -> uint32_t { return bar0 + 8u * (uint32_t)(C::STAGES + s); };
  auto tfull = [&](int s) -> uint32_t { return bar0 + 8u * (uint32_t)(2 * C::STAGES + s); };
  auto tempty = [&](int s) -> uint32_t { return bar0 + 8u * (uint32_t)(2 * C::STAGES + 2 + s); };
  const uint32_t bar_end = bar0 + 8u * (2 * C::STAGES + 4);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::OFF_BAR + 8 * (2 * C::STAGES + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* status_slot = tmem_slot + 2;
  // K blocks of a unit (negative: A is MN-major), from the producer to the MMA issuer. The producer
  // is at most STAGES units ahead.
  volatile int* unit_slot = reinterpret_cast<volatile int*>(tmem_slot + 4);
  static_assert(8 * (2 * C::STAGES + 5) + 16 + 4 * 8 <= 256 && C::STAGES < 8, "barrier page");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const int worker = (int)blockIdx.x / CG, workers = (int)gridDim.x / CG;
  // Launched programmatically: the set-up of this CTA may run while the previous kernel still does;
  // nothing global is touched before that is done.
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull(s), 1);
      mbar_init(tempty(s), CG * C::EPI_WARPS);
    }
    mbar_init(bar_end, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmA0);
    prefetch_tmap(&tmB0);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc_cg<CG>(smem_u32(tmem_slot), C::TMEM_COLS);
  }
  griddep_wait();
  griddep_launch_dependents();
  if (threadIdx.x == 0) *status_slot = *reinterpret_cast<const volatile unsigned int*>(work.status);
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // both CTAs' barriers are initialised
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The CTAs of a pair decide alike: either's view of the status word counts.
  uint32_t status = *status_slot;
  if constexpr (CG == 2) {
    uint32_t other;
    asm volatile("ld.shared::cluster.u32 %0, [%1];"
                 : "=r"(other)
                 : "r"(map_rank(smem_u32(tmem_slot + 2), rank ^ 1u))
                 : "memory");
    status |= other;
  }
  const bool dead = status != 0;

  // Warps 0 and 1 share their schedulers with epilogue warps and get few issue slots beside them, so
  // their loops are kept to what each K block needs: running stage and phase, no division, the
  // abort flag looked at once per unit, the unit's decoding left to the producer (which runs
  // ahead). Loss forward of 8192 x 2048, vocabulary 65,536: 1647 us before, 1528 us so.
  const int count = gemm_count(work, worker, workers);
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0 && !dead) {
      int st = 0, round = 0;
      bool ok = true;
      for (int i = 0; ok && i < count; ++i) {
        int which;
        const int u = gemm_deal(work, worker, workers, i, which);
        const bool second = A_MODE == 2 && which == 1;
        const GemmShape& g = work.g[second ? 1 : 0];
        const CUtensorMap* ta = second ? &tmA1 : &tmA0;
        const CUtensorMap* tb = second ? &tmB1 : &tmB0;
        const bool a_mn = A_MODE == 1 || second;
        const GemmUnit w = gemm_unit(g, u);
        const int m0 = (w.mt * CG + (int)rank) * C::BM;
        const int n0 = g.b_pair ? w.nt * (BN / 2) + (CG == 2 && rank ? g.b_pair : 0)
                                : w.nt * BN * NH + (int)rank * C::HB;
        const int n1 = g.b_pair ? n0 + g.b_pair : n0 + BN / 2;  // CG = 1: second half of B
        int k = w.k0 * C::BK, kr = k;
        int to_jump = B_MN ? g.b_kjump_at - w.k0 : 0;
        if (B_MN && to_jump <= 0) kr = g.b_kjump - to_jump * C::BK;
        unit_slot[i & 7] = a_mn ? w.k0 - w.k1 : w.k1 - w.k0;
        if (*abort_flag) ok = false;
        for (int n = w.k1 - w.k0; ok && n > 0; --n) {
          if (round > 0 && !mbar_wait(empty(st), (round - 1) & 1, work.status)) {
            ok = false;
            break;
          }
          const uint32_t sa = sbase + st * C::STAGE, sb = sa + C::A_BYTES;
          uint32_t fb = full(st);
          if constexpr (CG == 2) {
            if (rank == 0) mbar_expect_tx(fb, CG * C::STAGE);
            fb = map_rank(fb, 0);
          } else {
            mbar_expect_tx(fb, a_mn ? C::STAGE : C::B_BYTES + (uint32_t)g.a_rows * 128u);
          }
          if (a_mn) {
            tma_load_2d<CG>(sa, ta, fb, m0, k);
            tma_load_2d<CG>(sa + 8192, ta, fb, m0 + 64, k);
          } else {
            tma_load_2d<CG>(sa, ta, fb, k, m0);
          }
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const uint32_t sh = sb + h * (C::HB * 128);
            if constexpr (B_MN) {
#pragma unroll
              for (int j = 0; j < C::HB / 64; ++j)
                tma_load_2d<CG>(sh + j * 8192, tb, fb, n0 + h * BN + j * 64, kr);
            } else {
              tma_load_2d<CG>(sh, tb, fb, k, n0 + h * BN);
              if constexpr (CG == 1) tma_load_2d<CG>(sh + C::B_BYTES / 2, tb, fb, k, n1);
            }
          }
          if constexpr (B_MN) kr = --to_jump == 0 ? g.b_kjump : kr + C::BK;
          k += C::BK;
          if (++st == C::STAGES) st = 0, ++round;
        }
      }
      if (!ok) {
        *abort_flag = 1;
        // loads in flight land before the shared memory is released: each stage's last use
        if (rank == 0)
          for (int j = 0; j < C::STAGES; ++j) {
            const int uses = round + (j < st ? 1 : 0);
            if (uses > 0) mbar_wait(full(j), (uses - 1) & 1, work.status);
          }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && rank == 0 && !dead) {
      constexpr uint32_t IDESC = idesc_f16(BF16, A_MODE == 1, B_MN, 128 * CG, BN);
      constexpr uint32_t KB = B_MN ? 2048 >> 4 : 2;  // 16 k's on (descriptor units)
      constexpr uint32_t LBO = 8192;                 // MN-major: next 64 rows of m or n
      const uint32_t a_first = sdesc_lo(sbase, 16), b_first = sdesc_lo(sbase + C::A_BYTES, B_MN ? LBO : 16);
      uint32_t st = 0, ph = 0;
      bool ok = true;
      // The MMAs of one K block in stage `at` into accumulator `acc`, with half h of B.
      auto mmas = [&](uint32_t acc, uint32_t at, int h, bool a_mn, uint32_t keep) {
        const uint32_t a_lo = a_first + at * (C::STAGE >> 4) + (a_mn ? ((LBO - 16) >> 4) << 16 : 0u);
        const uint32_t b_lo = b_first + at * (C::STAGE >> 4) + (uint32_t)h * (C::HB * 128 >> 4);
        const uint32_t idesc = A_MODE == 2 && a_mn ? IDESC | (1u << 15) : IDESC;
        const uint32_t ka = a_mn ? 2048 >> 4 : 2;
#pragma unroll
        for (int kk = 0; kk < C::BK / 16; ++kk)
          mma_cg<CG>(acc, a_lo + kk * ka, b_lo + kk * KB, idesc, kk ? 1u : keep);
      };
      auto release = [&]() {
        mma_commit_cg<CG>(empty((int)st));
        if (++st == C::STAGES) st = 0, ph ^= 1;
      };
      for (int i = 0; ok && i < count; ++i) {
        int left = 0;
        bool a_mn = false;
        if constexpr (NH == 1) {
          const uint32_t acc = tmem + (uint32_t)((i & 1) * BN);
          if (i >= 2) ok = mbar_wait(tempty(i & 1), ((i >> 1) - 1) & 1, work.status);
          if (ok) ok = mbar_wait(full((int)st), ph, work.status) && !*abort_flag;
          if (!ok) break;
          tc_fence_after();
          const int n = unit_slot[i & 7];
          a_mn = A_MODE == 1 || (A_MODE == 2 && n < 0);
          mmas(acc, st, 0, a_mn, 0u);
          release();
          for (left = abs(n) - 1; left > 0; --left) {
            if (!mbar_wait(full((int)st), ph, work.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            mmas(acc, st, 0, a_mn, 1u);
            release();
          }
        } else {
          // Both accumulators are one tile's. The epilogue frees the first half of the columns
          // before the second: the first K blocks go into the first half alone, up to one stage
          // short of the ring, and are kept for the second.
          if (i >= 1) ok = mbar_wait(tempty(0), (i - 1) & 1, work.status);
          if (ok) ok = mbar_wait(full((int)st), ph, work.status) && !*abort_flag;
          if (!ok) break;
          tc_fence_after();
          const int n = unit_slot[i & 7];
          a_mn = A_MODE == 1 || (A_MODE == 2 && n < 0);
          const int lead = min(abs(n), C::STAGES - 1);
          uint32_t at = st, pt = ph;
          for (int j = 0; j < lead; ++j) {
            if (j > 0) {
              ok = mbar_wait(full((int)at), pt, work.status);
              if (!ok) break;
              tc_fence_after();
            }
            mmas(tmem, at, 0, a_mn, j ? 1u : 0u);
            if (++at == C::STAGES) at = 0, pt ^= 1;
          }
          if (ok && i >= 1) ok = mbar_wait(tempty(1), (i - 1) & 1, work.status);
          if (!ok) break;
          tc_fence_after();
          for (int j = 0; j < lead; ++j) {
            mmas(tmem + BN, st, 1, a_mn, j ? 1u : 0u);
            release();
          }
          for (left = abs(n) - lead; left > 0; --left) {
            if (!mbar_wait(full((int)st), ph, work.status)) {
              ok = false;
              break;
            }
            tc_fence_after();
            mmas(tmem, st, 0, a_mn, 1u);
            mmas(tmem + BN, st, 1, a_mn, 1u);
            release();
          }
        }
        if (ok) mma_commit_cg<CG>(tfull(NH == 1 ? i & 1 : 0));
      }
      if (!ok) *abort_flag = 1;
      mma_commit_cg<CG>(bar_end);  // every MMA retires before TMEM and shared memory are released
      mbar_wait(bar_end, 0, work.status);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue
    EpiCtx e;
    e.failed = dead;
    e.lane = lane;
    e.quad = warp & 3;  // the 32 TMEM lanes this warp can read
    e.half = (warp - 2) >> 2;
    e.exch = smem + C::OFF_EXCH + (warp - 2) * 4096;
    const int row_in = (int)rank * C::BM + e.quad * 32;
    GemmUnit next;
    bool next_second = false;
    typename Epi::Row next_row{};
    auto look = [&](int i) {
      int which;
      const int u = gemm_deal(work, worker, workers, i, which);
      next_second = A_MODE == 2 && which == 1;
      next = gemm_unit(work.g[next_second ? 1 : 0], u);
      next_row = Epi::row(next_second ? ea1 : ea0, next.mt * CG * C::BM + row_in + lane);
    };
    look(0);
    for (int i = 0; i < count; ++i) {
      const GemmUnit w = next;
      const bool second = next_second;
      const typename Epi::Row row = next_row;
      if (i + 1 < count) look(i + 1);
      if (!e.failed) {
        const bool ok = NH == 1 ? mbar_wait(tfull(i & 1), (i >> 1) & 1, work.status)
                                : mbar_wait(tfull(0), i & 1, work.status);
        if (!__all_sync(0xffffffffu, ok && !*abort_flag)) {
          e.failed = true;
          *abort_flag = 1;
        }
        tc_fence_after();
      }
      e.turn = i;
      e.row0 = w.mt * CG * C::BM + row_in;
#pragma unroll 1
      for (int h = 0; h < NH; ++h) {
        const int buf = NH == 1 ? i & 1 : h;
        e.taddr = tmem + ((uint32_t)(e.quad * 32) << 16) + (uint32_t)(buf * BN);
        GemmUnit wh = w;
        wh.nt = w.nt * NH + h;
        Epi::tile(second ? ea1 : ea0, wh, row, e);
        tc_fence_before();
        __syncwarp();
        if (!e.failed && lane == 0) {
          if constexpr (CG == 2) mbar_arrive_cluster(map_rank(tempty(buf), 0));
          else mbar_arrive(tempty(buf));
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {
    // every arrival the leading CTA's MMAs send here has come, and the other CTA is done with this
    // one's memory
    if (threadIdx.x == 0 && rank == 1 && !dead) mbar_wait(bar_end, 0, work.status);
    __syncthreads();
    cluster_sync();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_cg<CG>(tmem, C::TMEM_COLS);
  }
}

// Tensor map of a 16-bit matrix [rows, cols] (unit column stride, row stride ld elements) with a
// box of 64 columns x box_rows rows in the 128-byte swizzle.
inline int make_tmap_2d(CUtensorMap* map, const void* ptr, int dtype, int64_t cols, int64_t rows,
                        int64_t ld, int box_rows, const char* name) {
  auto enc = tmap_encoder();
  if (!enc) return abi_error(SSA_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? ld * 2 : ((cols * 2 + 15) & ~(int64_t)15))};
  cuuint32_t box[2] = {64u, (cuuint32_t)box_rows};
  cuuint32_t es[2] = {1u, 1u};
  const CUtensorMapDataType dt =
      dtype == SSA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r =
      enc(map, dt, 2, const_cast<void*>(ptr), dims, strides, box, es,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return abi_error(SSA_ERR_BAD_STRIDE,
                     "%s: cuTensorMapEncodeTiled failed (CUresult %d) for %p [%lld x %lld], row "
                     "stride %lld", name, (int)r, ptr, (long long)rows, (long long)cols,
                     (long long)ld);
  return SSA_OK;
}

// A matrix operand: [mn, k] when K-major (rows of length k), [k, mn] when MN-major.
struct GemmOperand {
  const void* ptr;
  int64_t mn, k, ld;
  const char* name;
};

int device_sm_count();  // multiprocessors of the current device (cached)

// Multiprocessors that plans are made for, so that a workspace size needs no device.
constexpr int kPlanSms = 148;
// A tile's cost outside its K blocks (epilogue, pipeline fill), in K blocks.
constexpr int kTileCost = 8;

// One product, or two that are dealt out together.
template <class Epi>
struct GemmProduct {
  GemmOperand a, b;
  GemmShape g;
  typename Epi::Args ea;
};

template <class Epi, int CG, int BN, int NH, int A_MODE, bool B_MN, bool BF16>
int launch_gemm(const GemmProduct<Epi>& p0, const GemmProduct<Epi>* p1, cudaStream_t st) {
  using C = GemmCfg<CG, BN, NH>;
  constexpr int dtype = BF16 ? SSA_DTYPE_BF16 : SSA_DTYPE_F16;
  CUtensorMap t[4];
  const GemmProduct<Epi>& q1 = p1 ? *p1 : p0;
  const int64_t u0 = (int64_t)p0.g.tiles_m * p0.g.tiles_n * p0.g.splits;
  const int64_t u1 = p1 ? (int64_t)q1.g.tiles_m * q1.g.tiles_n * q1.g.splits : 0;
  if (u0 + u1 > INT32_MAX / 2) return abi_error(SSA_ERR_BAD_SHAPE, "too many tiles");
  GemmWork w{};
  w.g[0] = p0.g;
  w.g[1] = q1.g;
  // A row of the result depends on its own row of A alone: a lone row tile loads the rows it has
  // (whole 8-row groups of the swizzle) and leaves the rest of the stage as it is. Boxes that lie
  // mostly outside the matrix are slow: 9 rows of the loss's head 79 us, 64 rows 59 us before.
  for (GemmShape& g : w.g) g.set_divisors();
  for (GemmShape& g : w.g) g.a_rows = CG == 1 && g.tiles_m == 1 ? 0 : C::BM;
  if (!w.g[0].a_rows) w.g[0].a_rows = p0.a.mn < C::BM ? (int)(p0.a.mn + 7) / 8 * 8 : C::BM;
  if (!w.g[1].a_rows) w.g[1].a_rows = q1.a.mn < C::BM ? (int)(q1.a.mn + 7) / 8 * 8 : C::BM;
  for (int i = 0; i < (p1 ? 2 : 1); ++i) {
    const GemmProduct<Epi>& p = i ? q1 : p0;
    const bool a_mn = A_MODE == 1 || (A_MODE == 2 && i == 1);
    int rc = a_mn ? make_tmap_2d(&t[2 * i], p.a.ptr, dtype, p.a.mn, p.a.k, p.a.ld, 64, p.a.name)
                  : make_tmap_2d(&t[2 * i], p.a.ptr, dtype, p.a.k, p.a.mn, p.a.ld,
                                 w.g[i].a_rows, p.a.name);
    if (rc != SSA_OK) return rc;
    rc = B_MN ? make_tmap_2d(&t[2 * i + 1], p.b.ptr, dtype, p.b.mn, p.b.k, p.b.ld, 64, p.b.name)
              : make_tmap_2d(&t[2 * i + 1], p.b.ptr, dtype, p.b.k, p.b.mn, p.b.ld, BN / 2, p.b.name);
    if (rc != SSA_OK) return rc;
  }
  if (!p1) t[2] = t[0], t[3] = t[1];
  const int most = device_sm_count() / CG;
  const int workers = (int)(u0 + u1 < most ? u0 + u1 : most);
  w.lead = p1 && q1.g.kb_split > p0.g.kb_split ? 1 : 0;
  w.units0 = (int)(w.lead ? u1 : u0);
  w.units1 = (int)(w.lead ? u0 : u1);
  w.rem = w.units0 % workers;
  w.whole = w.units0 / workers;
  if (p1) {
    const int a = w.g[w.lead].kb_split + kTileCost, b = w.g[w.lead ^ 1].kb_split + kTileCost;
    w.extra = (a + b / 2) / b;
    w.turn = w.extra * b <= a ? w.rem : 0;
  }
  w.status = device_status_ptr();
  if (!w.status) return abi_error(SSA_ERR_CUDA, "cannot resolve the device status word");
  auto kern = gemm_sm100_kernel<Epi, CG, BN, NH, A_MODE, B_MN, BF16>;
  if (set_smem_limit_once(reinterpret_cast<const void*>(kern), (int)C::SMEM_BYTES) != SSA_OK)
    return abi_error(SSA_ERR_CUDA, "cannot raise the shared memory limit");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(workers * CG));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, t[0], t[1], t[2], t[3], w, p0.ea, q1.ea);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "%s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Tile form. A K block costs about 512 cycles in both: a 256 x 256 pair is bound by the MMAs, a 128 x
// 128 tile by its 32 KB from L2. So the pairs are taken where they need fewer rounds than single CTAs
// do, and where more than half of their rows are used. Feed-forward at 256 rows of 2048, ffn 5632:
// 176 single tiles (two rounds) 22 us, 44 pairs 17 us; at 300 rows of 512, ffn 1024: 48 single tiles
// 8 us, 16 pairs 10.5 us.
struct GemmForm {
  bool pair;
  int bm, bn, workers;
  bool wide;  // gradients: 256 x 512 tiles
};
inline GemmForm make_form(bool pair) {
  return pair ? GemmForm{true, 256, 256, kPlanSms / 2, false}
              : GemmForm{false, 128, 128, kPlanSms, false};
}

// Of a product [rows, cols] with a fused epilogue.
inline GemmForm gemm_form(int64_t rows, int64_t cols) {
  const int pairs = cdiv((int64_t)cdiv(rows, 256) * cdiv(cols, 256), kPlanSms / 2);
  const int singles = cdiv((int64_t)cdiv(rows, 128) * cdiv(cols, 128), kPlanSms);
  return make_form(rows > 128 && pairs < singles);
}

// Of dx [rows, hidden] (kx K blocks) and dW [cols, hidden] (kw K blocks): pairs once one of the two
// fills the clusters (few rows included: dW is then bound by its stores; at 64 rows of 2048,
// vocabulary 32,768 loss and gradients take 153 us with pairs, 176 us without; with fewer tiles, 300
// rows of 512, ffn 1024, 26 us without and 35 us with pairs); 256 x 512 tiles, which read a quarter
// less per operation, when these fill the clusters and the K loops are long against an epilogue that
// no longer runs under the next tile's MMAs.
inline GemmForm gradient_form(int64_t rows, int64_t cols, int hidden, int kx, int kw) {
  const int64_t dx = (int64_t)cdiv(rows, 256) * cdiv(hidden, 256);
  const int64_t dw = (int64_t)cdiv(cols, 256) * cdiv(hidden, 256);
  GemmForm f = make_form((dx > dw ? dx : dw) >= kPlanSms / 2);
  f.wide = f.pair && hidden > 256 && dx + dw >= 2 * f.workers && kx >= 64 && kw >= 64;
  if (f.wide) f.bn = 512;
  return f;
}

// Row tiles walked before the column advances: all of them while that operand's panel stays in L2
// beside the other's stream; else, when the column tiles are few, as many as keep one whole set of
// columns in flight (A is then read once, B from L2); else 16, a square-ish set of tiles.
inline GemmShape plain_shape(int tiles_m, int tiles_n, int kblocks, int64_t a_bytes) {
  GemmShape g{};
  g.tiles_m = tiles_m;
  g.tiles_n = tiles_n;
  g.splits = 1;
  g.kblocks = g.kb_split = kblocks;
  int band = tiles_n <= 18 ? kPlanSms / 2 / tiles_n : 16;
  if (band < 1) band = 1;
  g.band = a_bytes <= (int64_t)40 << 20 || tiles_m < band ? tiles_m : band;
  g.b_kjump_at = INT32_MAX;
  return g;
}

// Splits of the contraction of `tiles` tiles of `kblocks` K blocks beside `other` K blocks of the
// launch's other product, so that no unit is longer than a worker's share of everything; of at least
// four blocks each, and only where that shortens the longest unit by 32 blocks (9 us): the splits'
// sums take another launch. The same whether the other product is asked for or not: so are the bits.
inline int split_count(int64_t tiles, int kblocks, int64_t other, int workers) {
  const int64_t share = (tiles * kblocks + other) / workers;
  int64_t s = share > 0 ? (kblocks + share - 1) / share : kblocks;
  if (s > kblocks / 4) s = kblocks / 4;
  if (s <= 1 || kblocks - kblocks / s < 32) return 1;
  return cdiv(kblocks, cdiv(kblocks, s));
}

// ------------------------------------------------------------------------- plain store epilogue
// out = acc * scale in 16 bits, or with out == nullptr the fp32 sum: one [rows, cols] matrix per split,
// written, or added to (a later piece of the same contraction).
struct StoreArgs {
  void* out;             // 16-bit [.., ldo], or nullptr
  float* sum;            // fp32 [splits][rows][cols], or nullptr
  const float* scale;    // device scalar, or nullptr (1)
  const float* row_scale;  // one factor per row (out only), or nullptr
  int64_t ldo;
  int rows, cols;        // cols: a multiple of 8
  int add_prev;          // add to sum
  int jump_at, jump;     // rows >= jump_at are stored at jump + row - jump_at; rows in
  int jump_rows;         //   [jump_rows, jump_at) and past jump_at + jump_rows are dropped
};

struct StoreProduct {
  GemmOperand a, b;
  GemmShape g;
  StoreArgs ea;
};

// dx = d W (d K-major) and dW = d^T x (d MN-major), B MN-major in both: one launch for both, or either
// alone where the other is nullptr.
int launch_gradients(bool bf16, const GemmForm& form, const StoreProduct* dx, const StoreProduct* dw,
                     cudaStream_t st);

// out[row, col] = scale * row_scale[row] * (the splits' sums [splits][rows][cols], added in split
// order); either factor may be nullptr.
int launch_sum_splits(bool bf16, const float* sum, void* out, const float* scale,
                      const float* row_scale, int64_t rows, int cols, int64_t ldo, int splits,
                      cudaStream_t st);

}  // namespace sm100
}  // namespace ssa

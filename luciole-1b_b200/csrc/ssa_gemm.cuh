// ssa_gemm.cuh — a persistent tcgen05 matrix product C[m, n] = sum_k A[m, k] B[n, k] whose epilogue
// is a template argument: the shared core of the linear cross entropy (ssa_linear_ce.cu) and the
// gated feed-forward (ssa_gated_ffn.cu).
//
// Roles (192 threads): warp 0 issues TMA loads, warp 1 issues the MMAs, warps 2..5 run the
// epilogue, one thread per accumulator row. A tile's fp32 accumulator is BN TMEM columns and there
// are two of them, so the epilogue of one tile runs under the MMAs of the next.
//
// Operands are 16-bit matrices in global memory, each either K-major (the contraction index is
// contiguous) or MN-major (the row index m or n is contiguous): a gradient product reads its
// operands in place, with no transposed copy. Both arrive as 64-element (128-byte) wide boxes in
// the 128-byte swizzle; a box past an edge of the matrix reads zeros, so M, N and K are arbitrary.
// Only alignment is asked for: 16-byte base and row stride.
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

// How the tiles of one launch are laid out (plain data, passed by value).
struct GemmShape {
  int tiles_m, tiles_n;  // 128-row and BN-column tiles
  int splits;            // contiguous K ranges per tile, each a unit of work
  int kblocks;           // 64-wide K blocks of a tile
  int kb_split;          // K blocks per split
  int band;              // row tiles walked before the column advances (operand reuse in L2)
  int b_kjump_at;        // MN-major B: K blocks from here on read rows b_kjump + 64 (kb - at)
  int b_kjump;
  int b_pair;            // 0, or B is a pair of row blocks this far apart, BN / 2 rows of each
  unsigned int* status;
};

struct GemmUnit {
  int mt, nt, sp, k0, k1;
};

__device__ __forceinline__ GemmUnit gemm_unit(const GemmShape& g, int u) {
  GemmUnit w;
  const int t = u / g.splits;
  w.sp = u - t * g.splits;
  const int per_band = g.band * g.tiles_n;
  const int bd = t / per_band, r = t - bd * per_band;
  const int rows = min(g.band, g.tiles_m - bd * g.band);
  w.nt = r / rows;
  w.mt = bd * g.band + (r - w.nt * rows);
  w.k0 = w.sp * g.kb_split;
  w.k1 = min(g.kblocks, w.k0 + g.kb_split);
  return w;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}

template <int BN_>
struct GemmCfg {
  static constexpr int BM = 128, BN = BN_, BK = 64;
  static constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE > 8 ? 8 : 196608 / STAGE;
  static constexpr uint32_t OFF_BAR = STAGES * STAGE;
  static constexpr uint32_t SMEM_BYTES = OFF_BAR + 256 + 1024;  // + slack for 1 KB alignment
  static constexpr uint32_t TMEM_COLS = 2 * BN;
  static constexpr int THREADS = 192;
};

// Reads accumulator columns [32 c, 32 c + 32) of the calling thread's row (every lane of the warp
// calls it): the values in TMEM, or NaN when the launch failed.
struct AccReader {
  uint32_t taddr;
  bool failed;
  __device__ __forceinline__ void operator()(int col, float (&v)[32]) const {
    if (failed) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = nan_f32();
      return;
    }
    uint32_t r[32];
    tmem_ld32(taddr + (uint32_t)col, r);
    tmem_ld_wait(r);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  }
};

// Epi: struct with `Args` and `static void tile(const Args&, const GemmUnit&, int row, const
// AccReader&)`, run by every epilogue thread for its accumulator row (0..127) of each unit.
template <class Epi, int BN, bool A_MN, bool B_MN, bool BF16>
__global__ void __launch_bounds__(192, 1)
    gemm_sm100_kernel(const __grid_constant__ CUtensorMap tmA,
                      const __grid_constant__ CUtensorMap tmB, const GemmShape g,
                      const typename Epi::Args ea) {
  using C = GemmCfg<BN>;
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

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Launched programmatically: nothing global is touched before the previous kernel is done.
  griddep_wait();
  griddep_launch_dependents();
  const int units = g.tiles_m * g.tiles_n * g.splits;

  if (block_status_failed(g.status)) {  // block-uniform
    if (warp >= 2) {
      const AccReader nan_acc{0, true};
      for (int u = blockIdx.x; u < units; u += gridDim.x)
        Epi::tile(ea, gemm_unit(g, u), (warp & 3) * 32 + lane, nan_acc);
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(tfull(s), 1);
      mbar_init(tempty(s), 128);
    }
    mbar_init(bar_end, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(smem_u32(tmem_slot), C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      prefetch_tmap(&tmA);
      prefetch_tmap(&tmB);
      int it = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const GemmUnit w = gemm_unit(g, u);
        const int m0 = w.mt * C::BM;
        const int n0 = g.b_pair ? w.nt * (BN / 2) : w.nt * BN;
        for (int kb = w.k0; kb < w.k1; ++kb, ++it) {
          const int st = it % C::STAGES, use = it / C::STAGES;
          if (use > 0) ok = mbar_wait(empty(st), (use - 1) & 1, g.status);
          if (!ok || *abort_flag) {
            ok = false;
            break;
          }
          const uint32_t sa = sbase + st * C::STAGE, sb = sa + C::A_BYTES;
          mbar_expect_tx(full(st), C::STAGE);
          const int k = kb * C::BK;
          if constexpr (A_MN) {
#pragma unroll
            for (int i = 0; i < C::BM / 64; ++i)
              tma_load_2d(sa + i * 8192, &tmA, full(st), m0 + i * 64, k);
          } else {
            tma_load_2d(sa, &tmA, full(st), k, m0);
          }
          if constexpr (B_MN) {
            const int kr = kb < g.b_kjump_at ? k : g.b_kjump + (kb - g.b_kjump_at) * C::BK;
#pragma unroll
            for (int i = 0; i < BN / 64; ++i)
              tma_load_2d(sb + i * 8192, &tmB, full(st), n0 + i * 64, kr);
          } else {  // two boxes of BN / 2 rows: one after the other, or the two of a pair
            tma_load_2d(sb, &tmB, full(st), k, n0);
            tma_load_2d(sb + C::B_BYTES / 2, &tmB, full(st), k,
                        g.b_pair ? g.b_pair + n0 : n0 + BN / 2);
          }
        }
      }
      if (!ok) {
        *abort_flag = 1;
        // this CTA's own loads land before its shared memory is released
        for (int j = max(0, it - C::STAGES); j < it; ++j)
          mbar_wait(full(j % C::STAGES), (j / C::STAGES) & 1, g.status);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f16(BF16, A_MN, B_MN, C::BM, BN);
      constexpr uint32_t LBO = 8192;                  // MN-major: next 64 rows of m or n
      constexpr uint32_t KA = A_MN ? 2048 >> 4 : 2, KB = B_MN ? 2048 >> 4 : 2;  // 16 k's on
      int it = 0, i = 0;
      bool ok = true;
      for (int u = blockIdx.x; ok && u < units; u += gridDim.x, ++i) {
        const GemmUnit w = gemm_unit(g, u);
        const uint32_t acc = tmem + (uint32_t)((i & 1) * BN);
        if (i >= 2) ok = mbar_wait(tempty(i & 1), ((i >> 1) - 1) & 1, g.status);
        if (!ok || *abort_flag) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int kb = w.k0; kb < w.k1; ++kb, ++it) {
          const int st = it % C::STAGES;
          ok = mbar_wait(full(st), (it / C::STAGES) & 1, g.status);
          if (!ok || *abort_flag) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_lo = sdesc_lo(sbase + st * C::STAGE, A_MN ? LBO : 16);
          const uint32_t b_lo = sdesc_lo(sbase + st * C::STAGE + C::A_BYTES, B_MN ? LBO : 16);
#pragma unroll
          for (int kk = 0; kk < C::BK / 16; ++kk)
            mma_ss_lo(acc, a_lo + kk * KA, b_lo + kk * KB, idesc, (kb > w.k0 || kk > 0) ? 1u : 0u);
          mma_commit(empty(st));
        }
        if (ok) mma_commit(tfull(i & 1));
      }
      if (!ok) *abort_flag = 1;
      mma_commit(bar_end);  // every MMA of this CTA retires before TMEM is freed
      mbar_wait(bar_end, 0, g.status);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ epilogue rows
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    AccReader rd{tmem + ((uint32_t)(quad * 32) << 16), false};
    int i = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x, ++i) {
      const GemmUnit w = gemm_unit(g, u);
      if (!rd.failed) {
        const bool ok = mbar_wait(tfull(i & 1), (i >> 1) & 1, g.status);
        if (!__all_sync(0xffffffffu, ok && !*abort_flag)) {
          rd.failed = true;
          *abort_flag = 1;
        }
        tc_fence_after();
        rd.taddr = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)((i & 1) * BN);
      }
      Epi::tile(ea, w, row, rd);
      tc_fence_before();
      if (!rd.failed) mbar_arrive(tempty(i & 1));
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
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

template <class Epi, int BN, bool A_MN, bool B_MN, bool BF16>
int launch_gemm(const GemmOperand& a, const GemmOperand& b, GemmShape g,
                const typename Epi::Args& ea, cudaStream_t st) {
  using C = GemmCfg<BN>;
  constexpr int dtype = BF16 ? SSA_DTYPE_BF16 : SSA_DTYPE_F16;
  CUtensorMap ta, tb;
  int rc;
  rc = A_MN ? make_tmap_2d(&ta, a.ptr, dtype, a.mn, a.k, a.ld, 64, a.name)
            : make_tmap_2d(&ta, a.ptr, dtype, a.k, a.mn, a.ld, C::BM, a.name);
  if (rc != SSA_OK) return rc;
  rc = B_MN ? make_tmap_2d(&tb, b.ptr, dtype, b.mn, b.k, b.ld, 64, b.name)
            : make_tmap_2d(&tb, b.ptr, dtype, b.k, b.mn, b.ld, BN / 2, b.name);
  if (rc != SSA_OK) return rc;
  g.status = device_status_ptr();
  if (!g.status) return abi_error(SSA_ERR_CUDA, "cannot resolve the device status word");
  auto kern = gemm_sm100_kernel<Epi, BN, A_MN, B_MN, BF16>;
  if (set_smem_limit_once(reinterpret_cast<const void*>(kern), (int)C::SMEM_BYTES) != SSA_OK)
    return abi_error(SSA_ERR_CUDA, "cannot raise the shared memory limit");
  const int64_t units = (int64_t)g.tiles_m * g.tiles_n * g.splits;
  const int grid = (int)(units < device_sm_count() ? units : device_sm_count());
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)grid), dim3(C::THREADS), C::SMEM_BYTES, st,
                                   ta, tb, g, ea);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "%s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

inline int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
inline size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// Row tiles walked before the column advances: all of them while that operand's panel stays in L2
// beside the other's stream, else 16, a square-ish set of tiles in flight.
inline int gemm_band(int tiles_m, int64_t a_bytes) {
  return a_bytes <= (int64_t)40 << 20 ? tiles_m : (tiles_m < 16 ? tiles_m : 16);
}

inline GemmShape plain_shape(int tiles_m, int tiles_n, int kblocks, int64_t a_bytes) {
  GemmShape g{};
  g.tiles_m = tiles_m;
  g.tiles_n = tiles_n;
  g.splits = 1;
  g.kblocks = g.kb_split = kblocks;
  g.band = gemm_band(tiles_m, a_bytes);
  g.b_kjump_at = INT32_MAX;
  return g;
}

// Splits of each tile's contraction when there are fewer tiles than multiprocessors, of at least
// four K blocks each.
inline int split_count(int tiles, int kblocks) {
  int s = tiles < kPlanSms ? kPlanSms / tiles : 1;
  if (s > kblocks / 4) s = kblocks / 4;
  return s > 1 ? cdiv(kblocks, cdiv(kblocks, s)) : 1;
}

// ------------------------------------------------------------------------- plain store epilogue
// out = (acc + earlier partial sum) * scale in 16 bits, or the running fp32 sum itself. `sum` holds
// one [rows, cols] fp32 matrix per split; adding to it across launches is ordered by the stream.
struct StoreArgs {
  void* out;             // 16-bit [.., ldo], or nullptr: keep the sum in fp32
  float* sum;            // fp32 [splits][rows][cols], or nullptr
  const float* scale;    // device scalar, or nullptr (1)
  int64_t rows, ldo;
  int cols;              // a multiple of 8
  int add_prev;          // add the matching element of sum
  int jump_at, jump;     // rows >= jump_at are stored at jump + row - jump_at; rows in
  int jump_rows;         //   [jump_rows, jump_at) and past jump_at + jump_rows are dropped
};

template <int BN, bool BF16>
struct EpiStore {
  using Args = StoreArgs;
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, int r,
                                              const AccReader& rd) {
    const int64_t row = (int64_t)w.mt * 128 + r;
    const int col0 = w.nt * BN;
    int64_t orow = row;
    bool ok = row < a.rows;
    if (a.jump_at) {
      const int64_t in = row < a.jump_at ? row : row - a.jump_at;
      ok = ok && in < a.jump_rows;
      orow = row < a.jump_at ? row : a.jump + in;
    }
    const float sc = a.scale ? __ldg(a.scale) : 1.f;
    float* srow = a.sum ? a.sum + ((int64_t)w.sp * a.rows + row) * a.cols : nullptr;
    uint16_t* drow = a.out ? reinterpret_cast<uint16_t*>(a.out) + orow * a.ldo : nullptr;
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      if (col0 + c >= a.cols) break;
      float v[32];
      rd(c, v);
      if (!ok) continue;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const int col = col0 + c + i;
        if (col >= a.cols) break;
        if (a.add_prev) {
          const float4* p = reinterpret_cast<const float4*>(srow + col);
          const float4 x = p[0], y = p[1];
          v[i] += x.x, v[i + 1] += x.y, v[i + 2] += x.z, v[i + 3] += x.w;
          v[i + 4] += y.x, v[i + 5] += y.y, v[i + 6] += y.z, v[i + 7] += y.w;
        }
        if (drow) {
          *reinterpret_cast<uint4*>(drow + col) =
              make_uint4(pack2<BF16>(v[i] * sc, v[i + 1] * sc), pack2<BF16>(v[i + 2] * sc, v[i + 3] * sc),
                         pack2<BF16>(v[i + 4] * sc, v[i + 5] * sc), pack2<BF16>(v[i + 6] * sc, v[i + 7] * sc));
        } else {
          float4* p = reinterpret_cast<float4*>(srow + col);
          p[0] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
          p[1] = make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
        }
      }
    }
  }
};

// out[row, col] = scale * sum over splits, in split order (deterministic).
template <bool BF16>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* sum, void* out,
                                                         const float* scale, int64_t rows, int cols,
                                                         int64_t ldo, int splits) {
  griddep_wait();
  griddep_launch_dependents();
  const float sc = scale ? __ldg(scale) : 1.f;
  const int per_row = cols / 4;
  const int64_t total = rows * per_row, plane = rows * (int64_t)cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 4;
    const float* p = sum + row * cols + col;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(p + k * plane);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + row * ldo + col) =
        make_uint2(pack2<BF16>(s.x * sc, s.y * sc), pack2<BF16>(s.z * sc, s.w * sc));
  }
}

template <bool BF16>
int launch_sum_splits(const float* sum, void* out, const float* scale, int64_t rows, int cols,
                      int64_t ldo, int splits, cudaStream_t st) {
  const int64_t blocks = (rows * (cols / 4) + 255) / 256;
  const int64_t most = (int64_t)device_sm_count() * 8;
  const cudaError_t e =
      launch_pdl(sum_splits_kernel<BF16>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256),
                 0, st, sum, out, scale, rows, cols, ldo, splits);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "%s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

}  // namespace sm100
}  // namespace ssa

// ssa_gated_ffn.cu — the gated feed-forward's first half, h = silu(x Wg^T) * (x Wu^T), in one
// kernel, and its backward. Weights are one [2 ffn, hidden] matrix: the gate's rows, then the up
// projection's.
//
// Forward: a tile of the tensor-core product takes half its B rows from the gate and half from the
// up projection, so both fp32 pre-activations of an output sit in the same thread's TMEM lane and h
// leaves directly. Nothing but x and the weights is kept for the backward, which forms the
// pre-activations again (fp32: the derivative sees no rounding) and writes
//     dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = sigmoid(g)
// as one 16-bit matrix d = [dg | du]; then dx = d W and dW = d^T x are two plain products. d is
// rounded to 16 bits because it is their operand: with the rounding of the results both are 0.029% off
// in fp16 and 0.23% in bf16, where the results' rounding alone is 0.021% and 0.17%; an fp32 d would take
// two or three products for each. In fp16 d has that type's range too, as dh has: 6e-8 to 65,504. Bound:
// the tensor cores, 16 rows hidden ffn operations for forward and backward against the 12 that
// kept pre-activations would need (at 8 bytes of memory per row and ffn column, held over the whole
// forward). A forward of few rows has a kernel of its own, bound by memory.
#include "ssa_gemm.cuh"

namespace ssa {
namespace sm100 {

__device__ __forceinline__ float sigmoid_approx(float g) {
  return rcp_approx(1.f + ex2_approx(-g * kLog2e));  // g = -inf: 1 / inf = 0
}

struct FfnFwdArgs {
  void* h;
  int64_t ldh;
  int rows, ffn, vec;  // vec: h's rows take 16-byte stores
};

template <int BN, bool BF16>
struct EpiFfnFwd {
  using Args = FfnFwdArgs;
  struct Row {};
  __device__ static __forceinline__ Row row(const Args&, int) { return Row{}; }
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, const Row&,
                                              const EpiCtx& e) {
    const int off = e.half * (BN / 4);  // a warp's gate columns; the up projection's are BN / 2 on
    uint16_t* base = reinterpret_cast<uint16_t*>(a.h) + (int64_t)e.row0 * a.ldh;
    // Only columns that exist are fetched: every read of TMEM is waited for before the tile is handed
    // back to the MMAs.
    const int col0 = w.nt * (BN / 2) + off, n = min(BN / 4, a.ffn - col0);
    if (n <= 0) return;
    uint32_t xg[32], xu[32];
    e.fetch(off, xg);
    e.fetch(BN / 2 + off, xu);
#pragma unroll 1
    for (int c = 0; c < n; c += 32) {
      const int col = col0 + c;
      float g[32], u[32];
      e.settle();
      e.values(xg, g);
      e.values(xu, u);
      if (c + 32 < n) {
        e.fetch(off + c + 32, xg);
        e.fetch(BN / 2 + off + c + 32, xu);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) g[i] = g[i] * sigmoid_approx(g[i]) * u[i];
      store_block16<BF16>(e, g, base, a.ldh, a.rows - e.row0, col, a.ffn, a.vec);
    }
  }
};

struct FfnBwdArgs {
  const void* dh;
  int64_t lddh;
  void* d;       // 16-bit [rows][2 wide]: dg in columns [0, wide), du in [wide, 2 wide); 0 past ffn
  int wide;      // ffn rounded up to whole tiles: every column of d is written
  int rows, ffn, vec;
};

template <int BN, bool BF16>
struct EpiFfnBwd {
  using Args = FfnBwdArgs;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  struct Row {};
  __device__ static __forceinline__ Row row(const Args&, int) { return Row{}; }
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, const Row&,
                                              const EpiCtx& e) {
    const int off = e.half * (BN / 4);
    const int rows = a.rows - e.row0;
    const uint16_t* dhbase = reinterpret_cast<const uint16_t*>(a.dh) + (int64_t)e.row0 * a.lddh;
    uint16_t* base = reinterpret_cast<uint16_t*>(a.d) + (int64_t)e.row0 * (2 * a.wide);
    uint8_t* in = e.exch + 2048;  // dh's block; the first half of the buffer carries d's
    uint32_t xg[32], xu[32];
    e.fetch(off, xg);
    e.fetch(BN / 2 + off, xu);
#pragma unroll 1
    for (int c = 0; c < BN / 4; c += 32) {
      const int col = w.nt * (BN / 2) + off + c;
      if (a.vec && col + 32 <= a.ffn) {
        const int p = e.lane & 3;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + (e.lane >> 2);
          *exch16(in, r, p) = r < rows ? __ldg(reinterpret_cast<const uint4*>(
                                             dhbase + (int64_t)r * a.lddh + col + 8 * p))
                                       : make_uint4(0u, 0u, 0u, 0u);
        }
      } else {
        // All of a batch is read before any of it is written: 4096 x 1024, ffn 2815, forward and
        // backward 272 us element by element, 180 us so, 164 us with aligned rows (ffn 2816).
#pragma unroll 1
        for (int r0 = 0; r0 < 32; r0 += 8) {
          uint16_t y[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            y[r] = r0 + r < rows && col + e.lane < a.ffn
                       ? __ldg(reinterpret_cast<const unsigned short*>(dhbase) +
                               (int64_t)(r0 + r) * a.lddh + col + e.lane) : 0;
#pragma unroll
          for (int r = 0; r < 8; ++r)
            reinterpret_cast<uint16_t*>(exch16(in, r0 + r, e.lane >> 3))[e.lane & 7] = y[r];
        }
      }
      __syncwarp();
      float g[32], u[32];
      e.settle();
      e.values(xg, g);
      e.values(xu, u);
      if (c + 32 < BN / 4) {
        e.fetch(off + c + 32, xg);
        e.fetch(BN / 2 + off + c + 32, xu);
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint4 x = *exch16(in, e.lane, p);
        const T* t = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int i = 8 * p + j;
          const float dh = to_f32<T>(t[j]), z = g[i], s = sigmoid_approx(z);
          g[i] = dh * u[i] * (s * fmaf(z, 1.f - s, 1.f));
          u[i] = dh * (z * s);
          if (col + i >= a.ffn) g[i] = u[i] = 0.f;
        }
      }
      store_block16<BF16>(e, g, base, 2 * a.wide, rows, col, a.wide, true);
      store_block16<BF16>(e, u, base, 2 * a.wide, rows, a.wide + col, 2 * a.wide, true);
    }
  }
};

// Few rows: KW warps share the contraction of 8 output columns and 8 NT rows; a block has 8 / KW such
// groups. The 16 rows of a warp's matrix instruction are 8 gate and 8 up columns, its 8 columns are
// rows of x, so g and u of an output meet in one thread. A sum does not mind the order of its terms:
// lane (r, t) takes the 16 bytes k = 8 t .. 8 t + 7 of weight row r as they lie in memory and hands
// them to two instructions, x in the same order. The partial sums are joined in a fixed order. Bound:
// memory, every weight read once per 16 rows with 16 16-byte loads per lane under way; the tensor
// cores only save the conversions, which cost more than the reads from two rows on.
template <typename T, int NT, int KW>
__global__ void __launch_bounds__(256, 2)
    ffn_rows_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, T* h, int64_t ldh, int rows,
                    int hidden, int ffn) {
  constexpr int kCols = 64 / KW, kLd = 20;  // a joined row: 8 gate sums, 8 up sums, 4 to part banks
  __shared__ float part[8][8 * NT][kLd];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * (8 * NT), col0 = blockIdx.x * kCols;
  const int wcol = col0 + warp / KW * 8 + r;
  const bool live = wcol < ffn;
  rows -= row0;
  x += row0 * ldx;
  h += row0 * ldh;
  const T* wg = w + (int64_t)(live ? wcol : 0) * ldw + 8 * t;
  const T* wu = w + (int64_t)(live ? ffn + wcol : 0) * ldw + 8 * t;
  const T* xr = x + r * ldx + 8 * t;
  float c[NT][4] = {};
  constexpr int U = 4, kStep = KW * 64;  // U 64-wide pieces of the contraction under way per warp
  for (int k0 = warp % KW * 64; k0 < hidden; k0 += U * kStep) {
    uint4 g[U][2], u[U][2], b[U][2][NT];
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = k0 + i * kStep + j * 32;
        const bool in = k + 8 * t < hidden;
        const uint4 z = make_uint4(0u, 0u, 0u, 0u);
        g[i][j] = in && live ? __ldg(reinterpret_cast<const uint4*>(wg + k)) : z;
        u[i][j] = in && live ? __ldg(reinterpret_cast<const uint4*>(wu + k)) : z;
#pragma unroll
        for (int n = 0; n < NT; ++n)
          b[i][j][n] = in && 8 * n + r < rows
                           ? __ldg(reinterpret_cast<const uint4*>(xr + 8 * n * ldx + k)) : z;
      }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint4 v = b[i][j][n];
          mma_16x8<T>(c[n], g[i][j].x, u[i][j].x, g[i][j].y, u[i][j].y, v.x, v.y);
          mma_16x8<T>(c[n], g[i][j].z, u[i][j].z, g[i][j].w, u[i][j].w, v.z, v.w);
        }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[warp][8 * n + 2 * t + (j & 1)][r + 8 * (j >> 1)] = c[n][j];
  __syncthreads();
  for (int i = threadIdx.x; i < kCols * 8 * NT; i += 256) {
    const int row = i / kCols, col = i % kCols;
    if (row >= rows || col0 + col >= ffn) continue;
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      g += part[col / 8 * KW + s][row][col % 8];
      u += part[col / 8 * KW + s][row][8 + col % 8];
    }
    h[(int64_t)row * ldh + col0 + col] = from_f32<T>(g * sigmoid_approx(g) * u);
  }
}

}  // namespace sm100

namespace {

using namespace sm100;

template <typename T, int NT, int KW>
int ffn_rows(const ssa_gated_ffn_t* p, void* h, int64_t ldh, cudaStream_t st) {
  const dim3 grid((unsigned)cdiv(p->ffn, 64 / KW), (unsigned)cdiv(p->rows, 8 * NT));
  const cudaError_t e = launch_pdl(ffn_rows_kernel<T, NT, KW>, grid, dim3(256), 0, st,
                                   static_cast<const T*>(p->x), p->x_stride,
                                   static_cast<const T*>(p->w), p->w_stride, static_cast<T*>(h), ldh,
                                   p->rows, p->hidden, p->ffn);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "ffn_rows: %s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

// Warps per contraction: as few as take it with one batch of loads each.
int few_rows_warps(const ssa_gated_ffn_t* p) {
  return p->hidden <= 512 ? 2 : p->hidden <= 1024 ? 4 : 8;
}

// Up to 16 rows, and as long as all blocks of 16 rows take one round of the multiprocessors (two where
// the contraction is long): 128-row tiles wait for one tile's whole contraction, so that few tiles are
// slow however small the product. Hidden 2048, ffn 5632 (46 MB, from L2): 1 row 5.8 us, 8 rows 6.9,
// 16 rows 9.6 against 12.8 on tiles, 32 rows would take 15.7; 180 MB of weights from memory, 8 rows
// 28.9 us (6.2 TB/s) against 47.8. Hidden 2048, ffn 1024: 64 rows 7.2 us against 12.0.
bool few_rows(const ssa_gated_ffn_t* p) {
  const int64_t blocks = (int64_t)cdiv(p->ffn, 64 / few_rows_warps(p)) * cdiv(p->rows, 16);
  return p->rows <= 16 || blocks <= (p->hidden <= 512 ? 2 : 4) * kPlanSms;
}

template <typename T>
int ffn_few_rows(const ssa_gated_ffn_t* p, void* h, int64_t ldh, cudaStream_t st) {
  const int kw = few_rows_warps(p);
  if (p->rows <= 8)
    return kw == 2   ? ffn_rows<T, 1, 2>(p, h, ldh, st)
           : kw == 4 ? ffn_rows<T, 1, 4>(p, h, ldh, st)
                     : ffn_rows<T, 1, 8>(p, h, ldh, st);
  return kw == 2   ? ffn_rows<T, 2, 2>(p, h, ldh, st)
         : kw == 4 ? ffn_rows<T, 2, 4>(p, h, ldh, st)
                   : ffn_rows<T, 2, 8>(p, h, ldh, st);
}

struct FfnPlan {
  GemmForm pair, bwd;  // tiles of the pre-activations, and of dx and dw
  int wide;
  int dx_splits;
  size_t off_sum, bwd_bytes;
};

FfnPlan ffn_plan(const ssa_gated_ffn_t* p) {
  FfnPlan q{};
  q.pair = gemm_form(p->rows, 2 * (int64_t)p->ffn);
  q.wide = cdiv(p->ffn, q.pair.bn / 2) * (q.pair.bn / 2);
  q.bwd = gradient_form(p->rows, 2 * (int64_t)q.wide, p->hidden, 2 * q.wide / 64,
                        cdiv(p->rows, 64));
  const int64_t dx_tiles = (int64_t)cdiv(p->rows, q.bwd.bm) * cdiv(p->hidden, q.bwd.bn);
  const int64_t dw_tiles = (int64_t)cdiv(2 * q.wide, q.bwd.bm) * cdiv(p->hidden, q.bwd.bn);
  q.dx_splits = split_count(dx_tiles, 2 * q.wide / 64, dw_tiles * (cdiv(p->rows, 64) + kTileCost),
                            q.bwd.workers);
  q.off_sum = up256(4 * (size_t)p->rows * q.wide);
  q.bwd_bytes = q.off_sum;
  if (q.dx_splits > 1)
    q.bwd_bytes += up256(sizeof(float) * (size_t)q.dx_splits * p->rows * p->hidden);
  return q;
}

int ffn_check(const ssa_gated_ffn_t* p) {
  if (!p) return abi_error(SSA_ERR_NULL, "problem is NULL");
  if (p->dtype != SSA_DTYPE_F16 && p->dtype != SSA_DTYPE_BF16)
    return abi_error(SSA_ERR_UNSUPPORTED, "gated_ffn: dtype %d not supported (fp16, bf16)", p->dtype);
  if (p->rows <= 0 || p->hidden <= 0 || p->ffn <= 0)
    return abi_error(SSA_ERR_BAD_SHAPE, "gated_ffn: non-positive shape rows=%d hidden=%d ffn=%d",
                     p->rows, p->hidden, p->ffn);
  if (p->hidden % 8)
    return abi_error(SSA_ERR_BAD_SHAPE, "gated_ffn: hidden=%d must be a multiple of 8", p->hidden);
  if (p->rows > (1 << 24) || p->hidden > (1 << 24) || p->ffn > (1 << 24))
    return abi_error(SSA_ERR_BAD_SHAPE, "gated_ffn: rows, hidden and ffn must not exceed 2^24");
  if (!p->x || !p->w) return abi_error(SSA_ERR_NULL, "gated_ffn: x or w is NULL");
  if (((uintptr_t)p->x | (uintptr_t)p->w) % 16 || p->x_stride % 8 || p->w_stride % 8 ||
      p->x_stride < p->hidden || p->w_stride < p->hidden)
    return abi_error(SSA_ERR_BAD_STRIDE, "gated_ffn: x and w need 16-byte aligned rows of at least "
                     "hidden elements");
  return SSA_OK;
}

// The product of x with both projections, with a forward or backward epilogue.
template <template <int, bool> class Epi, bool BF16, class Args>
int ffn_pair_gemm(const ssa_gated_ffn_t* p, const FfnPlan& q, const Args& a, cudaStream_t st) {
  const GemmOperand A{p->x, p->rows, p->hidden, p->x_stride, "x"};
  const GemmOperand B{p->w, 2 * (int64_t)p->ffn, p->hidden, p->w_stride, "w"};
  GemmShape g = plain_shape(cdiv(p->rows, q.pair.bm), cdiv(p->ffn, q.pair.bn / 2),
                            cdiv(p->hidden, 64), 2 * (int64_t)p->rows * p->hidden);
  g.b_pair = p->ffn;
  return q.pair.pair
             ? launch_gemm<Epi<256, BF16>, 2, 256, 1, 0, false, BF16>({A, B, g, a}, nullptr, st)
             : launch_gemm<Epi<128, BF16>, 1, 128, 1, 0, false, BF16>({A, B, g, a}, nullptr, st);
}

template <bool BF16>
int ffn_bwd(const ssa_gated_ffn_t* p, const FfnPlan& q, const void* dh, int64_t lddh, void* dx,
            void* dw, uint8_t* ws, cudaStream_t st) {
  const FfnBwdArgs a{dh, lddh, ws, q.wide, p->rows, p->ffn,
                     (uintptr_t)dh % 16 == 0 && lddh % 8 == 0 ? 1 : 0};
  int rc = ffn_pair_gemm<EpiFfnBwd, BF16>(p, q, a, st);
  if (rc != SSA_OK) return rc;
  const int64_t k2 = 2 * (int64_t)q.wide;
  float* sum = reinterpret_cast<float*>(ws + q.off_sum);
  StoreArgs sx{}, sw{};
  sx.out = q.dx_splits == 1 ? dx : nullptr;
  sx.sum = sum;
  sx.rows = p->rows;
  sx.ldo = sx.cols = sw.ldo = sw.cols = p->hidden;
  const int kblocks = (int)(k2 / 64), tiles_h = cdiv(p->hidden, q.bwd.bn);
  GemmShape gx = plain_shape(cdiv(p->rows, q.bwd.bm), tiles_h, kblocks, 2 * (int64_t)p->rows * k2);
  gx.kb_split = cdiv(kblocks, q.dx_splits);
  gx.splits = q.dx_splits;
  gx.b_kjump_at = q.wide / 64;  // du's columns meet the up projection's rows
  gx.b_kjump = p->ffn;
  sw.out = dw;
  sw.rows = (int)k2;
  sw.jump_at = q.wide;
  sw.jump = sw.jump_rows = p->ffn;
  const GemmShape gw = plain_shape(cdiv(k2, q.bwd.bm), tiles_h, cdiv(p->rows, 64),
                                   2 * (int64_t)p->rows * k2);
  const GemmOperand dk{ws, p->rows, k2, k2, "d"}, dmn{ws, k2, p->rows, k2, "d"};
  const GemmOperand wb{p->w, p->hidden, 2 * (int64_t)p->ffn, p->w_stride, "w"};
  const GemmOperand xb{p->x, p->hidden, p->rows, p->x_stride, "x"};
  const StoreProduct px{dk, wb, gx, sx}, pw{dmn, xb, gw, sw};
  rc = launch_gradients(BF16, q.bwd, dx ? &px : nullptr, dw ? &pw : nullptr, st);
  if (rc != SSA_OK) return rc;
  if (dx && q.dx_splits > 1)
    return launch_sum_splits(BF16, sum, dx, nullptr, nullptr, p->rows, p->hidden, p->hidden, q.dx_splits, st);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" {

size_t ssa_gated_ffn_bwd_workspace_size(const ssa_gated_ffn_t* p) {
  abi_clear_error();
  return ffn_check(p) == SSA_OK ? ffn_plan(p).bwd_bytes : 0;
}

int ssa_gated_ffn_fwd(const ssa_gated_ffn_t* p, void* h, int64_t h_stride, void* stream) {
  abi_clear_error();
  int rc = ffn_check(p);
  if (rc != SSA_OK) return rc;
  if (!h) return abi_error(SSA_ERR_NULL, "gated_ffn: h is NULL");
  if (h_stride < p->ffn || (uintptr_t)h % 2)
    return abi_error(SSA_ERR_BAD_STRIDE, "gated_ffn: h's row stride is below ffn");
  if ((rc = abi_bind_device(p->x, "x")) != SSA_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_rows(p))
    return p->dtype == SSA_DTYPE_BF16 ? ffn_few_rows<__nv_bfloat16>(p, h, h_stride, st)
                                      : ffn_few_rows<__half>(p, h, h_stride, st);
  const FfnPlan q = ffn_plan(p);
  const FfnFwdArgs a{h, h_stride, p->rows, p->ffn,
                     (uintptr_t)h % 16 == 0 && h_stride % 8 == 0 ? 1 : 0};
  return p->dtype == SSA_DTYPE_BF16 ? ffn_pair_gemm<EpiFfnFwd, true>(p, q, a, st)
                                    : ffn_pair_gemm<EpiFfnFwd, false>(p, q, a, st);
}

int ssa_gated_ffn_bwd(const ssa_gated_ffn_t* p, const void* dh, int64_t dh_stride, void* dx,
                      void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  abi_clear_error();
  int rc = ffn_check(p);
  if (rc != SSA_OK) return rc;
  if (!dh) return abi_error(SSA_ERR_NULL, "gated_ffn: dh is NULL");
  if (dh_stride < p->ffn || (uintptr_t)dh % 2)
    return abi_error(SSA_ERR_BAD_STRIDE, "gated_ffn: dh's row stride is below ffn");
  if (((uintptr_t)dx | (uintptr_t)dw) % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "gated_ffn: dx and dw must be 16-byte aligned");
  if (!dx && !dw) return SSA_OK;
  if ((rc = abi_bind_device(p->x, "x")) != SSA_OK) return rc;
  const FfnPlan q = ffn_plan(p);
  if (!workspace || workspace_bytes < q.bwd_bytes || (uintptr_t)workspace % 256)
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu",
                     q.bwd_bytes, workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == SSA_DTYPE_BF16 ? ffn_bwd<true>(p, q, dh, dh_stride, dx, dw, ws, st)
                                    : ffn_bwd<false>(p, q, dh, dh_stride, dx, dw, ws, st);
}

}  // extern "C"

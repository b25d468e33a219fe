// ssa_gated_ffn.cu — the gated feed-forward's first half, h = silu(x Wg^T) * (x Wu^T), in one
// kernel, and its backward. Weights are one [2 ffn, hidden] matrix: the gate's rows, then the up
// projection's.
//
// Forward: a tile of the tensor-core product takes half its B rows from the gate and half from the
// up projection, so both fp32 pre-activations of an output sit in the same thread's TMEM lane and h
// leaves directly. Nothing but x and the weights is kept for the backward, which forms the
// pre-activations again (fp32: the derivative sees no rounding) and writes
//     dg = dh u s (1 + g (1 - s)),  du = dh g s,  s = sigmoid(g)
// as one 16-bit matrix d = [dg | du]; then dx = d W and dW = d^T x are two plain products. Bound:
// the tensor cores, 16 rows hidden ffn operations for forward and backward against the 12 that
// kept pre-activations would need (at 8 bytes of memory per row and ffn column, held over the whole
// forward).
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
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, int r,
                                              const AccReader& rd) {
    const int row = w.mt * 128 + r;
    const int col0 = w.nt * (BN / 2);
    T* hrow = reinterpret_cast<T*>(a.h) + (int64_t)row * a.ldh;
#pragma unroll 1
    for (int c = 0; c < BN / 2; c += 32) {
      if (col0 + c >= a.ffn) break;
      float g[32], u[32];
      rd(c, g);
      rd(BN / 2 + c, u);
      if (row >= a.rows) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) g[i] = g[i] * sigmoid_approx(g[i]) * u[i];
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const int col = col0 + c + i;
        if (a.vec && col + 8 <= a.ffn) {
          *reinterpret_cast<uint4*>(hrow + col) =
              make_uint4(pack2<BF16>(g[i], g[i + 1]), pack2<BF16>(g[i + 2], g[i + 3]),
                         pack2<BF16>(g[i + 4], g[i + 5]), pack2<BF16>(g[i + 6], g[i + 7]));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (col + j < a.ffn) hrow[col + j] = from_f32<T>(g[i + j]);
        }
      }
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
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, int r,
                                              const AccReader& rd) {
    const int row = w.mt * 128 + r;
    const int col0 = w.nt * (BN / 2);
    const T* dhrow = reinterpret_cast<const T*>(a.dh) + (int64_t)row * a.lddh;
    T* drow = reinterpret_cast<T*>(a.d) + (int64_t)row * (2 * a.wide);
#pragma unroll 1
    for (int c = 0; c < BN / 2; c += 32) {
      float g[32], u[32];
      rd(c, g);
      rd(BN / 2 + c, u);
      if (row >= a.rows) continue;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const int col = col0 + c + i;
        float dh[8];
        if (a.vec && col + 8 <= a.ffn) {
          const uint4 x = __ldg(reinterpret_cast<const uint4*>(dhrow + col));
          const T* t = reinterpret_cast<const T*>(&x);
#pragma unroll
          for (int j = 0; j < 8; ++j) dh[j] = to_f32<T>(t[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) dh[j] = col + j < a.ffn ? to_f32<T>(dhrow[col + j]) : 0.f;
        }
        float dg[8], du[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = g[i + j], s = sigmoid_approx(x);
          dg[j] = dh[j] * u[i + j] * (s * fmaf(x, 1.f - s, 1.f));
          du[j] = dh[j] * (x * s);
          if (col + j >= a.ffn) dg[j] = du[j] = 0.f;
        }
        *reinterpret_cast<uint4*>(drow + col) =
            make_uint4(pack2<BF16>(dg[0], dg[1]), pack2<BF16>(dg[2], dg[3]),
                       pack2<BF16>(dg[4], dg[5]), pack2<BF16>(dg[6], dg[7]));
        *reinterpret_cast<uint4*>(drow + a.wide + col) =
            make_uint4(pack2<BF16>(du[0], du[1]), pack2<BF16>(du[2], du[3]),
                       pack2<BF16>(du[4], du[5]), pack2<BF16>(du[6], du[7]));
      }
    }
  }
};

}  // namespace sm100

namespace {

using namespace sm100;

struct FfnPlan {
  int bn;         // 128-row tiles of bn / 2 gate and bn / 2 up columns
  int wide;
  int dx_bn, dx_splits;
  size_t off_sum, bwd_bytes;
};

FfnPlan ffn_plan(const ssa_gated_ffn_t* p) {
  FfnPlan q{};
  const int tm = cdiv(p->rows, 128);
  // Fewer tiles than multiprocessors at the wide tile: the narrow one.
  q.bn = (int64_t)tm * cdiv(p->ffn, 128) >= kPlanSms ? 256 : 128;
  q.wide = cdiv(p->ffn, q.bn / 2) * (q.bn / 2);
  q.dx_bn = (int64_t)tm * cdiv(p->hidden, 256) >= kPlanSms ? 256 : 128;
  q.dx_splits = split_count(tm * cdiv(p->hidden, q.dx_bn), 2 * q.wide / 64);
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
  if (p->rows > (1 << 24) || p->ffn > (1 << 24))
    return abi_error(SSA_ERR_BAD_SHAPE, "gated_ffn: rows and ffn must not exceed 2^24");
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
  GemmShape g = plain_shape(cdiv(p->rows, 128), cdiv(p->ffn, q.bn / 2), cdiv(p->hidden, 64),
                            2 * (int64_t)p->rows * p->hidden);
  g.b_pair = p->ffn;
  return q.bn == 256 ? launch_gemm<Epi<256, BF16>, 256, false, false, BF16>(A, B, g, a, st)
                     : launch_gemm<Epi<128, BF16>, 128, false, false, BF16>(A, B, g, a, st);
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
  const int tm = cdiv(p->rows, 128);
  if (dx) {
    StoreArgs s{};
    s.out = q.dx_splits == 1 ? dx : nullptr;
    s.sum = sum;
    s.rows = p->rows;
    s.ldo = s.cols = p->hidden;
    const int kblocks = (int)(k2 / 64);
    GemmShape g = plain_shape(tm, cdiv(p->hidden, q.dx_bn), kblocks, 2 * (int64_t)p->rows * k2);
    g.kb_split = cdiv(kblocks, q.dx_splits);
    g.splits = q.dx_splits;
    g.b_kjump_at = q.wide / 64;  // du's columns meet the up projection's rows
    g.b_kjump = p->ffn;
    const GemmOperand A{ws, p->rows, k2, k2, "d"};
    const GemmOperand B{p->w, p->hidden, 2 * (int64_t)p->ffn, p->w_stride, "w"};
    rc = q.dx_bn == 256 ? launch_gemm<EpiStore<256, BF16>, 256, false, true, BF16>(A, B, g, s, st)
                        : launch_gemm<EpiStore<128, BF16>, 128, false, true, BF16>(A, B, g, s, st);
    if (rc != SSA_OK) return rc;
    if (q.dx_splits > 1) {
      rc = launch_sum_splits<BF16>(sum, dx, nullptr, p->rows, p->hidden, p->hidden, q.dx_splits, st);
      if (rc != SSA_OK) return rc;
    }
  }
  if (dw) {
    StoreArgs s{};
    s.out = dw;
    s.rows = k2;
    s.ldo = s.cols = p->hidden;
    s.jump_at = q.wide;
    s.jump = s.jump_rows = p->ffn;
    rc = launch_gemm<EpiStore<256, BF16>, 256, true, true, BF16>(
        GemmOperand{ws, k2, p->rows, k2, "d"},
        GemmOperand{p->x, p->hidden, p->rows, p->x_stride, "x"},
        plain_shape((int)(k2 / 128), cdiv(p->hidden, 256), cdiv(p->rows, 64),
                    2 * (int64_t)p->rows * k2), s, st);
    if (rc != SSA_OK) return rc;
  }
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
  const FfnPlan q = ffn_plan(p);
  const FfnFwdArgs a{h, h_stride, p->rows, p->ffn,
                     (uintptr_t)h % 16 == 0 && h_stride % 8 == 0 ? 1 : 0};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
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

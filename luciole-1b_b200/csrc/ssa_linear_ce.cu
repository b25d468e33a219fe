// ssa_linear_ce.cu — cross entropy of a linear head, without its logits:
//     l = x W^T,  lse_r = log sum_v exp(l_rv),  loss_r = lse_r - l_r,t(r)
//     d_rv = g_r (exp(l_rv - lse_r) - [v = t(r)]),  dx = d W,  dW = d^T x
// for x [rows, hidden], W [vocab, hidden] in bf16 or fp16, fp32 logits that never leave the chip.
//
// Forward: one tensor-core product whose epilogue reduces each row of a tile to a running maximum
// and sum of exponentials (and picks the target's logit); a second kernel joins the tiles' pairs.
// Backward: the vocabulary is walked in pieces that fit the workspace. Per piece the logits are
// formed again and leave as d in 16 bits (the products' operands; the rounding, with that of the
// result, puts both gradients 0.02% off in fp16 and 0.17% in bf16, as the inputs' type allows), then
// two products read that piece: dx is summed over the pieces in fp32, dW's rows of the piece are final. Bound: the tensor cores, 8 rows hidden vocab
// operations for forward and backward against the 6 that a kept logit matrix would need.
#include <cmath>

#include "ssa_gemm.cuh"

namespace ssa {
namespace sm100 {

constexpr float kLowest = -1.0e38f;  // start of a running maximum: finite, so that max - max is 0

struct CeFwdArgs {
  const int64_t* targets;
  float2* part;   // [tiles_n][rows]: (maximum, sum of exp(l - maximum)) of a tile's columns
  float* target_logit;
  int rows, vocab;
};

// A row's target column, -1 where there is none in the vocabulary.
__device__ __forceinline__ int ce_target(const int64_t* targets, int row, int rows, int vocab) {
  const int64_t t = row < rows ? __ldg(targets + row) : -1;
  return t >= 0 && t < vocab ? (int)t : -1;
}

template <int BN>
struct EpiCeFwd {
  using Args = CeFwdArgs;
  struct Row {
    int t;
  };
  __device__ static __forceinline__ Row row(const Args& a, int row) {
    return Row{ce_target(a.targets, row, a.rows, a.vocab)};
  }
  // A lane holds its half row, BN / 2 columns, in registers: one maximum, then the exponentials in
  // eight independent sums.
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, const Row& rw,
                                              const EpiCtx& e) {
    constexpr int NC = BN / 64;  // 32-column pieces of the half
    const int row = e.row0 + e.lane;
    const int off = e.half * (BN / 2), col0 = w.nt * BN + off;
    const bool ok = row < a.rows;
    float m = kLowest, s = 0.f;
    if (col0 < a.vocab) {  // warp-uniform
      uint32_t x[NC][32];
      float v[NC][32];
#pragma unroll
      for (int c = 0; c < NC; ++c) e.fetch(off + 32 * c, x[c]);
      e.settle();
#pragma unroll
      for (int c = 0; c < NC; ++c) e.values(x[c], v[c]);
      if (col0 + 32 * NC > a.vocab) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (col0 + 32 * c + i >= a.vocab) v[c][i] = -INFINITY;
      }
      float m8[8], s8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m8[i] = kLowest, s8[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) m8[i & 7] = fmaxf(m8[i & 7], v[c][i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, m8[i]);
      const float b = -m * kLog2e, lost = fmaf(-m, kLog2e, -b);  // b's rounding: 2^lost on every term
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < 32; ++i) s8[i & 7] += ex2_approx(fmaf(v[c][i], kLog2e, b));
#pragma unroll
      for (int i = 0; i < 8; ++i) s += s8[i];
      s = fmaf(s, lost * kLn2, s);
      const int at = rw.t - col0;
      if (at >= 0 && at < 32 * NC) {
        float y = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) y = at == 32 * c + i ? v[c][i] : y;
        a.target_logit[row] = y;
      }
    }
    // The row's other half is in the warp with the same lanes: its pair comes through shared
    // memory, in two places in turn, so that one barrier per tile is enough.
    float2* mine = reinterpret_cast<float2*>(e.exch + (e.turn & 1) * 256) + e.lane;
    if (e.half == 1) *mine = make_float2(m, s);
    named_bar_sync(1 + e.quad, 64);
    if (e.half == 0 && ok) {
      const float2 p = *reinterpret_cast<const float2*>(reinterpret_cast<uint8_t*>(mine) + 4 * 4096);
      const float mn = fmaxf(m, p.x);
      s = s * ex2_approx((m - mn) * kLog2e) + p.y * ex2_approx((p.x - mn) * kLog2e);
      a.part[(int64_t)w.nt * a.rows + row] = make_float2(mn, s);
    }
  }
};

__device__ __forceinline__ void join_pair(float& m, float& s, float2 p) {
  const float mn = fmaxf(m, p.x);
  s = s * ex2_approx((m - mn) * kLog2e) + p.y * ex2_approx((p.x - mn) * kLog2e);
  m = mn;
}

// Joins the tiles' pairs: 32 rows per block (one per lane), 32 warps that each walk every 32nd tile
// (four loads under way at a time), then a warp per row. lse in natural units; loss 0 where the
// target is ignored, NaN where it is out of range.
__global__ void __launch_bounds__(1024)
    ce_join_kernel(const float2* part, const float* target_logit, const int64_t* targets,
                   int64_t ignore_index, int rows, int vocab, int tiles, float* lse, float* loss) {
  __shared__ float2 sh[32][33];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  float m = kLowest, s = 0.f;
  if (row < rows)
    for (int i = y; i < tiles; i += 128) {
      float2 p[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        p[k] = i + 32 * k < tiles ? part[(int64_t)(i + 32 * k) * rows + row] : make_float2(kLowest, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) join_pair(m, s, p[k]);
    }
  sh[y][lane] = make_float2(m, s);
  __syncthreads();
  const float2 p = sh[lane][y];
  m = p.x, s = p.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 q = make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    join_pair(m, s, q);
  }
  const int r = blockIdx.x * 32 + y;
  if (lane == 0 && r < rows) {
    const float ls = logf(s);
    lse[r] = m + ls;
    const int64_t t = targets[r];
    // (m - l_t) + log s: no cancellation between a large lse and a large logit
    loss[r] = t == ignore_index ? 0.f
              : (t < 0 || t >= vocab) ? nan_f32()
                                      : (m - target_logit[r]) + ls;
  }
}

// Few rows: the forward without tiles. KW warps share the contraction of 16 vocabulary rows with
// 8 NT rows of x, 8 / KW such groups a block; blocks walk the vocabulary. The 16 x 8 matrix
// instruction takes W's rows as they lie in memory: lane (r, t) hands the 16 bytes k = 8 t .. 8 t + 7
// of rows r and r + 8 to two instructions, x in the same order, which changes only the order of the
// sum's terms. Every thread keeps the running pair of a row over its share of the columns. Bound:
// memory, W read once per 16 rows.
template <typename T, int NT, int KW>
__global__ void __launch_bounds__(256, 2)
    ce_rows_kernel(const T* x, int64_t ldx, const T* w, int64_t ldw, int hidden, const CeFwdArgs a) {
  constexpr int kCols = 128 / KW, kLd = 20;  // a joined row: 16 logits, 4 to part the banks
  constexpr int kOut = kCols * 8 * NT, kPer = (kOut + 255) / 256;  // logits of a step, and per thread
  static_assert(kCols == 16 || kCols == 32, "a row's columns are lanes of one warp");
  __shared__ float part[2][8][8 * NT][kLd];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.y * (8 * NT), rows = a.rows - row0;
  const T* xr = x + (row0 + r) * ldx + 8 * t;
  const int cc = threadIdx.x % kCols;
  float m[kPer], s[kPer];
  int target[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    m[q] = kLowest, s[q] = 0.f;
    target[q] = ce_target(a.targets, row0 + (threadIdx.x + 256 * q) / kCols, a.rows, a.vocab);
  }
  int turn = 0;
  for (int v0 = blockIdx.x * kCols; v0 < a.vocab; v0 += gridDim.x * kCols) {
    const int v = v0 + warp / KW * 16 + r;
    const bool live0 = v < a.vocab, live1 = v + 8 < a.vocab;
    const T* w0 = w + (int64_t)(live0 ? v : 0) * ldw + 8 * t;
    const T* w1 = w + (int64_t)(live1 ? v + 8 : 0) * ldw + 8 * t;
    float c[NT][4] = {};
    constexpr int U = 4, kStep = KW * 64;  // U 64-wide pieces of the contraction under way per warp
    for (int k0 = warp % KW * 64; k0 < hidden; k0 += U * kStep) {
      uint4 u0[U][2], u1[U][2], b[U][2][NT];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = k0 + i * kStep + j * 32;
          const bool in = k + 8 * t < hidden;
          const uint4 z = make_uint4(0u, 0u, 0u, 0u);
          u0[i][j] = in && live0 ? __ldg(reinterpret_cast<const uint4*>(w0 + k)) : z;
          u1[i][j] = in && live1 ? __ldg(reinterpret_cast<const uint4*>(w1 + k)) : z;
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
            const uint4 y = b[i][j][n];
            mma_16x8<T>(c[n], u0[i][j].x, u1[i][j].x, u0[i][j].y, u1[i][j].y, y.x, y.y);
            mma_16x8<T>(c[n], u0[i][j].z, u1[i][j].z, u0[i][j].w, u1[i][j].w, y.z, y.w);
          }
    }
    // The partial sums meet in two places in turn, so that one barrier per step is enough.
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        part[turn][warp][8 * n + 2 * t + (j & 1)][r + 8 * (j >> 1)] = c[n][j];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int i = threadIdx.x + 256 * q, row = i / kCols;
      if (i < kOut && row < rows && v0 + cc < a.vocab) {
        float l = 0.f;
#pragma unroll
        for (int k = 0; k < KW; ++k) l += part[turn][cc / 16 * KW + k][row][cc % 16];
        if (target[q] == v0 + cc) a.target_logit[row0 + row] = l;
        join_pair(m[q], s[q], make_float2(l, 1.f));
      }
    }
    turn ^= 1;
  }
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
#pragma unroll
    for (int o = kCols / 2; o > 0; o >>= 1) {
      const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, m[q], o),
                                   __shfl_xor_sync(0xffffffffu, s[q], o));
      join_pair(m[q], s[q], y);
    }
    const int i = threadIdx.x + 256 * q, row = i / kCols;
    if (i < kOut && row < rows && cc == 0)
      a.part[(int64_t)blockIdx.x * a.rows + row0 + row] = make_float2(m[q], s[q]);
  }
}

// Sum over a block of 1024 threads in a fixed order; the result in thread 0.
__device__ __forceinline__ double block_sum_1024(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < 32 ? red[threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  return v;
}

// Sum of the rows' losses in 64 bits (mean: over the rows that are not ignored), and that count.
__global__ void __launch_bounds__(1024)
    ce_total_kernel(const float* loss_rows, const int64_t* targets, int64_t ignore_index, int rows,
                    int mean, float* loss, float* count) {
  __shared__ double red[32];
  griddep_wait();
  griddep_launch_dependents();
  double s = 0.0;
  int n = 0;
  for (int i = threadIdx.x; i < rows; i += 4096) {
    float l[4];
    int64_t t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = i + 1024 * k;
      l[k] = at < rows ? loss_rows[at] : 0.f;
      t[k] = at < rows ? targets[at] : ignore_index;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) s += (double)l[k], n += t[k] != ignore_index;
  }
  s = block_sum_1024(s, red);
  const double c = block_sum_1024((double)n, red);
  if (threadIdx.x == 0) {
    *loss = (float)(mean ? s / c : s);
    *count = (float)c;
  }
}

// What the backward multiplies (p - [v = t]) by before it is rounded to 16 bits: a power of two, so that
// the target's p - 1, which weighs most, is rounded as a number just below a power of two and not
// times an arbitrary factor that would put one error, up to 2^-8 in bf16, on a whole row (0.4% of the
// gradients of 8192 rows before). The power is 2^14, which keeps the small probabilities of a large
// vocabulary normal numbers in fp16; ignored rows and gradients of 0 have 0. The gradients enter in fp32:
//   one for all rows (mean, sum): grad / count 2^-14 in both products' epilogues (inv);
//   one per row: dx_r = grad_r 2^-14 (d W)_r, in the epilogue, so that a row's gradient depends on its
//   own factor alone. dW sums over rows, so there d has to carry the factors: a second matrix, d times
//   grad_r / top (top: the largest), rounded once, with top 2^-14 in the epilogue. Equal gradients,
//   as of a sum or a mean taken outside, give the factor 1. (One matrix for both products, with the
//   powers of two of grad_r in d and the rest rounded into x: 3-5% faster at 4096 and 8192 rows, dW's
//   terms rounded twice, and in fp16 the small probabilities of a row lost once another row's
//   gradient was 10^5 times as large.)
//
// Blocks after the first copy x, with ignored rows as zeros, for the product that sums over rows: what
// an ignored row holds (padding, an infinity) must not reach dW as 0 times it.
__global__ void __launch_bounds__(1024)
    ce_row_weights_kernel(const float* grad, int per_row, const int64_t* targets,
                          int64_t ignore_index, int rows, int vocab, const float* count, int mean,
                          float* weight, float* scale_x, float* factor, float* inv, const uint16_t* x,
                          int64_t ldx, int hidden, uint16_t* x_kept) {
  __shared__ float red[32];
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x > 0) {
    const int chunks = hidden / 8;  // of 16 bytes, per row
    const int64_t total = (int64_t)rows * chunks, step = (int64_t)(gridDim.x - 1) * 1024;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < total; i += step) {
      const int row = (int)(i / chunks), c = (int)(i - (int64_t)row * chunks);
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + (int64_t)row * ldx) + c);
      reinterpret_cast<uint4*>(x_kept)[i] =
          __ldg(targets + row) == ignore_index ? make_uint4(0u, 0u, 0u, 0u) : v;
    }
    return;
  }
  constexpr float kUp = 16384.f, kDown = 1.f / 16384.f;
  float top = 0.f;
  if (per_row) {
    for (int i = threadIdx.x; i < rows; i += 1024)
      if (targets[i] != ignore_index) top = fmaxf(top, fabsf(grad[i]));
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
    top = red[threadIdx.x & 31];
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!(top > 0.f && top < INFINITY)) top = 1.f;
    if (threadIdx.x == 0) inv[0] = kDown, inv[1] = top * kDown;
  } else if (threadIdx.x == 0) {
    const float n = mean ? *count : 1.f;  // no row counts: nothing to divide, gradients of 0
    inv[0] = inv[1] = n > 0.f ? grad[0] / n * kDown : 0.f;
  }
  for (int i = threadIdx.x; i < rows; i += 4096) {
    int64_t t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = i + 1024 * k < rows ? targets[i + 1024 * k] : ignore_index;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = i + 1024 * k;
      if (at >= rows) break;
      const bool skip = t[k] == ignore_index;
      const float g = skip ? 0.f : per_row ? grad[at] : 1.f;
      weight[at] = !skip && (t[k] < 0 || t[k] >= vocab) ? nan_f32() : g == 0.f ? 0.f : kUp;
      if (per_row) scale_x[at] = g, factor[at] = g / top;
    }
  }
}

struct CeBwdArgs {
  const int64_t* targets;
  const float* lse;
  const float* weight;
  const float* factor;  // one gradient per row: what d2 has above d
  void* d;         // 16-bit [rows][ldd], this piece's columns; columns past the vocabulary are 0
  void* d2;        // one gradient per row: d for dW; either may be nullptr
  int64_t ldd;
  int rows, piece0, vocab;
};

template <int BN, bool BF16, bool PER_ROW>
struct EpiCeBwd {
  using Args = CeBwdArgs;
  struct Row {
    float g, b, f;
    int t;
  };
  __device__ static __forceinline__ Row row(const Args& a, int row) {
    const bool ok = row < a.rows;
    return Row{ok ? __ldg(a.weight + row) : 0.f, ok ? -__ldg(a.lse + row) * kLog2e : 0.f,
               PER_ROW && ok ? __ldg(a.factor + row) : 0.f, ce_target(a.targets, row, a.rows, a.vocab)};
  }
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, const Row& rw,
                                              const EpiCtx& e) {
    const int off = e.half * (BN / 2);
    const int64_t first = (int64_t)e.row0 * a.ldd + w.nt * BN + off;
    const float g = rw.g, b = rw.b;
    const uint32_t mask = g == 0.f ? 0u : 0xffffffffu;  // an ignored row adds nothing, whatever it holds
    uint32_t x[32];
    e.fetch(off, x);
#pragma unroll 1
    for (int c = 0; c < BN / 2; c += 32) {
      const int col = a.piece0 + w.nt * BN + off + c;
      float v[32];
      e.settle();
      e.values(x, v);
      if (c + 32 < BN / 2) e.fetch(off + c + 32, x);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = ex2_approx(fmaf(v[i], kLog2e, b)) * g;
      const int at = rw.t - col;
      if (at >= 0 && at < 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = at == i ? v[i] - g : v[i];
      }
      if (col + 32 > a.vocab) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (col + i >= a.vocab) v[i] = 0.f;
      }
      if (!PER_ROW || a.d)
        store_block16<BF16>(e, v, reinterpret_cast<uint16_t*>(a.d) + first, a.ldd, a.rows - e.row0, c,
                            BN / 2, true, mask);
      if (PER_ROW && a.d2) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= rw.f;
        store_block16<BF16>(e, v, reinterpret_cast<uint16_t*>(a.d2) + first, a.ldd, a.rows - e.row0, c,
                            BN / 2, true, mask);
      }
    }
  }
};

}  // namespace sm100

namespace {

using namespace sm100;

// d of one piece (each of two matrices with one gradient per row); the larger, the fewer passes over the fp32 sums of dx
constexpr int64_t kPieceBytes = (int64_t)256 << 20;

// Warps per contraction: as few as take it with one batch of loads each, but a row's columns must
// be lanes of one warp.
int few_rows_warps(const ssa_linear_ce_t* p) { return p->hidden <= 1024 ? 4 : 8; }

// Up to 8 rows, and as long as all steps of 16 rows take one round of the multiprocessors (two where
// the contraction is long); 128-row tiles otherwise, with their join. Hidden 2048, vocabulary 65,536
// (268 MB): 1 to 8 rows 45-46 us (6.2 TB/s without the join) against 56 on tiles, 16 rows would take
// 58. Hidden 2048, vocabulary 1024: 64 rows 7.4 us against 14.1.
bool few_rows(const ssa_linear_ce_t* p) {
  const int64_t steps = (int64_t)cdiv(p->vocab, 128 / few_rows_warps(p)) * cdiv(p->rows, 16);
  return p->rows <= 8 || steps <= (p->hidden <= 512 ? 2 : 4) * kPlanSms;
}

struct CePlan {
  GemmForm fwd, bwd;           // tiles of the logits, and of dx and dw
  bool few;                    // forward without tiles
  int fwd_tiles;               // column tiles of the forward, or blocks that share the columns
  int64_t ldd;                 // columns of a piece (a multiple of 256)
  int pieces;
  int dx_splits;
  size_t off_target, off_rows, fwd_bytes;
  size_t off_scale, off_factor, off_inv, off_x, off_d, off_d2, off_sum, bwd_bytes;
};

CePlan ce_plan(const ssa_linear_ce_t* p) {
  CePlan q{};
  const int64_t rows = p->rows;
  q.fwd = gemm_form(rows, p->vocab);
  q.few = few_rows(p);
  q.fwd_tiles = cdiv(p->vocab, q.few ? 128 / few_rows_warps(p) : q.fwd.bn);
  if (q.few && q.fwd_tiles > 2 * kPlanSms) q.fwd_tiles = 2 * kPlanSms;
  q.off_target = up256(sizeof(float2) * (size_t)q.fwd_tiles * rows);
  q.off_rows = q.off_target + up256(sizeof(float) * rows);
  q.fwd_bytes = q.off_rows + up256(sizeof(float) * rows);

  const int matrices = p->reduction ? 1 : 2;  // one gradient per row: d for dx and d for dW
  int64_t cols = kPieceBytes / (2 * rows) / 256 * 256;
  if (cols < 1024) cols = 1024;
  const int64_t all = (int64_t)cdiv(p->vocab, 256) * 256;
  if (cols > all) cols = all;
  q.pieces = cdiv(all, cols);
  q.ldd = (int64_t)cdiv(all / 256, q.pieces) * 256;  // pieces of about equal width
  q.pieces = cdiv(all, q.ldd);
  q.bwd = gradient_form(rows, q.ldd, p->hidden, (int)(q.ldd / 64), cdiv(rows, 64));
  const int64_t dx_tiles = (int64_t)cdiv(rows, q.bwd.bm) * cdiv(p->hidden, q.bwd.bn);
  const int64_t dw_tiles = (int64_t)cdiv(q.ldd, q.bwd.bm) * cdiv(p->hidden, q.bwd.bn);
  q.dx_splits = split_count(dx_tiles, (int)(q.ldd / 64), dw_tiles * (cdiv(rows, 64) + kTileCost),
                            q.bwd.workers);
  q.off_scale = up256(sizeof(float) * rows);
  q.off_factor = 2 * q.off_scale;
  q.off_inv = 3 * q.off_scale;
  q.off_x = q.off_inv + 256;
  q.off_d = q.off_x + up256(2 * (size_t)rows * p->hidden);
  q.off_d2 = q.off_d + up256(2 * (size_t)rows * q.ldd);
  q.off_sum = matrices == 1 ? q.off_d2 : 2 * q.off_d2 - q.off_d;
  q.bwd_bytes = q.off_sum;
  if (q.pieces > 1 || q.dx_splits > 1)
    q.bwd_bytes += up256(sizeof(float) * (size_t)q.dx_splits * rows * p->hidden);
  return q;
}

int ce_check(const ssa_linear_ce_t* p) {
  if (!p) return abi_error(SSA_ERR_NULL, "problem is NULL");
  if (p->dtype != SSA_DTYPE_F16 && p->dtype != SSA_DTYPE_BF16)
    return abi_error(SSA_ERR_UNSUPPORTED, "linear_ce: dtype %d not supported (fp16, bf16)", p->dtype);
  if (p->rows <= 0 || p->hidden <= 0 || p->vocab <= 0)
    return abi_error(SSA_ERR_BAD_SHAPE, "linear_ce: non-positive shape rows=%d hidden=%d vocab=%d",
                     p->rows, p->hidden, p->vocab);
  if (p->hidden % 8)
    return abi_error(SSA_ERR_BAD_SHAPE, "linear_ce: hidden=%d must be a multiple of 8", p->hidden);
  if (p->rows > (1 << 24) || p->hidden > (1 << 24) || p->vocab > (1 << 24))
    return abi_error(SSA_ERR_BAD_SHAPE, "linear_ce: rows, hidden and vocab must not exceed 2^24");
  if (p->reduction < 0 || p->reduction > 2)
    return abi_error(SSA_ERR_UNSUPPORTED, "linear_ce: reduction %d (0 none, 1 mean, 2 sum)",
                     p->reduction);
  if (!p->x || !p->w || !p->targets)
    return abi_error(SSA_ERR_NULL, "linear_ce: x, w or targets is NULL");
  if (((uintptr_t)p->x | (uintptr_t)p->w) % 16 || p->x_stride % 8 || p->w_stride % 8 ||
      p->x_stride < p->hidden || p->w_stride < p->hidden)
    return abi_error(SSA_ERR_BAD_STRIDE, "linear_ce: x and w need 16-byte aligned rows of at least "
                     "hidden elements");
  return SSA_OK;
}

// The product of x with (a piece of) W, with a forward or backward epilogue.
template <class Epi256, class Epi128, bool BF16, class Args>
int ce_logits(const ssa_linear_ce_t* p, const GemmForm& f, const void* w, int64_t cols, int tiles_n,
              const Args& a, cudaStream_t st) {
  const GemmOperand A{p->x, p->rows, p->hidden, p->x_stride, "x"};
  const GemmOperand B{w, cols, p->hidden, p->w_stride, "w"};
  const GemmShape g = plain_shape(cdiv(p->rows, f.bm), tiles_n, cdiv(p->hidden, 64),
                                  2 * (int64_t)p->rows * p->hidden);
  return f.pair ? launch_gemm<Epi256, 2, 256, 1, 0, false, BF16>({A, B, g, a}, nullptr, st)
                : launch_gemm<Epi128, 1, 128, 1, 0, false, BF16>({A, B, g, a}, nullptr, st);
}

template <typename T, int NT, int KW>
int ce_rows(const ssa_linear_ce_t* p, int blocks, const CeFwdArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)blocks, (unsigned)cdiv(p->rows, 8 * NT));
  const cudaError_t e = launch_pdl(ce_rows_kernel<T, NT, KW>, grid, dim3(256), 0, st,
                                   static_cast<const T*>(p->x), p->x_stride,
                                   static_cast<const T*>(p->w), p->w_stride, p->hidden, a);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "ce_rows: %s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

template <bool BF16>
int ce_few_rows(const ssa_linear_ce_t* p, int blocks, const CeFwdArgs& a, cudaStream_t st) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const bool four = few_rows_warps(p) == 4;
  if (p->rows <= 8) return four ? ce_rows<T, 1, 4>(p, blocks, a, st) : ce_rows<T, 1, 8>(p, blocks, a, st);
  return four ? ce_rows<T, 2, 4>(p, blocks, a, st) : ce_rows<T, 2, 8>(p, blocks, a, st);
}

template <bool BF16>
int ce_fwd(const ssa_linear_ce_t* p, const CePlan& q, float* loss, float* lse, float* count,
           uint8_t* ws, cudaStream_t st) {
  CeFwdArgs a{p->targets, reinterpret_cast<float2*>(ws),
              reinterpret_cast<float*>(ws + q.off_target), p->rows, p->vocab};
  const int rc = q.few
                     ? ce_few_rows<BF16>(p, q.fwd_tiles, a, st)
                     : ce_logits<EpiCeFwd<256>, EpiCeFwd<128>, BF16>(p, q.fwd, p->w, p->vocab,
                                                                     q.fwd_tiles, a, st);
  if (rc != SSA_OK) return rc;
  float* rows_loss = p->reduction ? reinterpret_cast<float*>(ws + q.off_rows) : loss;
  cudaError_t e = launch_pdl(ce_join_kernel, dim3((unsigned)cdiv(p->rows, 32)), dim3(1024), 0, st,
                             (const float2*)a.part, (const float*)a.target_logit, p->targets,
                             p->ignore_index, p->rows, p->vocab, q.fwd_tiles, lse, rows_loss);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "ce_join: %s", cudaGetErrorString(e));
  note_launches(1);
  if (p->reduction) {
    e = launch_pdl(ce_total_kernel, dim3(1), dim3(1024), 0, st, (const float*)rows_loss, p->targets,
                   p->ignore_index, p->rows, (int)(p->reduction == 1), loss, count);
    if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "ce_total: %s", cudaGetErrorString(e));
    note_launches(1);
  }
  return SSA_OK;
}

template <bool BF16>
int ce_bwd(const ssa_linear_ce_t* p, const CePlan& q, const float* lse, const float* count,
           const float* grad, void* dx, void* dw, uint8_t* ws, cudaStream_t st) {
  float* weight = reinterpret_cast<float*>(ws);
  float* scale_x = reinterpret_cast<float*>(ws + q.off_scale);
  float* factor = reinterpret_cast<float*>(ws + q.off_factor);
  float* inv = reinterpret_cast<float*>(ws + q.off_inv);
  const bool per_row = p->reduction == 0;
  uint8_t* d = ws + q.off_d;
  uint8_t* d_w = per_row ? ws + q.off_d2 : d;  // what dW reads
  float* sum = reinterpret_cast<float*>(ws + q.off_sum);
  uint16_t* x_kept = reinterpret_cast<uint16_t*>(ws + q.off_x);
  int copies = dw ? cdiv((int64_t)p->rows * (p->hidden / 8), 4 * 1024) : 0;
  if (copies > 2 * device_sm_count()) copies = 2 * device_sm_count();
  const cudaError_t e =
      launch_pdl(ce_row_weights_kernel, dim3((unsigned)(1 + copies)), dim3(1024), 0, st, grad,
                 (int)per_row, p->targets, p->ignore_index, p->rows, p->vocab, count,
                 (int)(p->reduction == 1), weight, scale_x, factor, inv,
                 static_cast<const uint16_t*>(p->x), p->x_stride, p->hidden, x_kept);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "ce_row_weights: %s", cudaGetErrorString(e));
  note_launches(1);
  for (int i = 0; i < q.pieces; ++i) {
    const int64_t v0 = (int64_t)i * q.ldd;
    const int64_t cols = p->vocab - v0 < q.ldd ? p->vocab - v0 : q.ldd;  // of the vocabulary
    const int64_t wide = (int64_t)cdiv(cols, 256) * 256;                 // written to d
    const uint8_t* w0 = static_cast<const uint8_t*>(p->w) + 2 * v0 * p->w_stride;
    const CeBwdArgs a{p->targets, lse, weight, factor, per_row && !dx ? nullptr : d,
                      per_row && dw ? d_w : nullptr, q.ldd, p->rows, (int)v0, p->vocab};
    const GemmForm form = gemm_form(p->rows, wide);
    const int tiles_n = (int)(wide / form.bn);
    int rc = per_row ? ce_logits<EpiCeBwd<256, BF16, true>, EpiCeBwd<128, BF16, true>, BF16>(
                           p, form, w0, cols, tiles_n, a, st)
                     : ce_logits<EpiCeBwd<256, BF16, false>, EpiCeBwd<128, BF16, false>, BF16>(
                           p, form, w0, cols, tiles_n, a, st);
    if (rc != SSA_OK) return rc;

    StoreArgs sx{}, sw{};
    sx.out = q.dx_splits == 1 && q.pieces == 1 ? dx : nullptr;
    sx.sum = sum;
    sx.scale = inv;
    sw.scale = inv + 1;
    sx.row_scale = per_row ? scale_x : nullptr;
    sx.rows = p->rows;
    sx.ldo = sx.cols = sw.ldo = sw.cols = p->hidden;
    sx.add_prev = i > 0;
    const int kblocks = (int)(wide / 64), tiles_h = cdiv(p->hidden, q.bwd.bn);
    GemmShape gx = plain_shape(cdiv(p->rows, q.bwd.bm), tiles_h, kblocks, 2 * (int64_t)p->rows * q.ldd);
    // every piece fills the same split planes: a narrower last piece takes thinner splits
    gx.kb_split = cdiv(kblocks, q.dx_splits);
    gx.splits = cdiv(kblocks, gx.kb_split);
    sw.out = static_cast<uint8_t*>(dw) + 2 * v0 * p->hidden;
    sw.rows = (int)cols;
    const GemmShape gw = plain_shape(cdiv(cols, q.bwd.bm), tiles_h, cdiv(p->rows, 64),
                                     2 * (int64_t)p->rows * q.ldd);
    const GemmOperand dk{d, p->rows, wide, q.ldd, "d"}, dmn{d_w, wide, p->rows, q.ldd, "d"};
    const GemmOperand wb{w0, p->hidden, cols, p->w_stride, "w"};
    const GemmOperand xb{x_kept, p->hidden, p->rows, p->hidden, "x"};
    const StoreProduct px{dk, wb, gx, sx}, pw{dmn, xb, gw, sw};
    rc = launch_gradients(BF16, q.bwd, dx ? &px : nullptr, dw ? &pw : nullptr, st);
    if (rc != SSA_OK) return rc;
  }
  if (dx && (q.dx_splits > 1 || q.pieces > 1))
    return launch_sum_splits(BF16, sum, dx, inv, per_row ? scale_x : nullptr, p->rows, p->hidden,
                             p->hidden, q.dx_splits, st);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" {

size_t ssa_linear_ce_fwd_workspace_size(const ssa_linear_ce_t* p) {
  abi_clear_error();
  if (ce_check(p) != SSA_OK) return 0;
  return ce_plan(p).fwd_bytes;
}

size_t ssa_linear_ce_bwd_workspace_size(const ssa_linear_ce_t* p) {
  abi_clear_error();
  if (ce_check(p) != SSA_OK) return 0;
  return ce_plan(p).bwd_bytes;
}

int ssa_linear_ce_fwd(const ssa_linear_ce_t* p, float* loss, float* lse, float* count,
                      void* workspace, size_t workspace_bytes, void* stream) {
  abi_clear_error();
  int rc = ce_check(p);
  if (rc != SSA_OK) return rc;
  if (!loss || !lse || (p->reduction && !count))
    return abi_error(SSA_ERR_NULL, "linear_ce: loss, lse or count is NULL");
  if ((rc = abi_bind_device(p->x, "x")) != SSA_OK) return rc;
  const CePlan q = ce_plan(p);
  if (!workspace || workspace_bytes < q.fwd_bytes || (uintptr_t)workspace % 256)
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu", q.fwd_bytes,
                     workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == SSA_DTYPE_BF16 ? ce_fwd<true>(p, q, loss, lse, count, ws, st)
                                    : ce_fwd<false>(p, q, loss, lse, count, ws, st);
}

int ssa_linear_ce_bwd(const ssa_linear_ce_t* p, const float* lse, const float* count,
                      const float* grad_loss, void* dx, void* dw, void* workspace,
                      size_t workspace_bytes, void* stream) {
  abi_clear_error();
  int rc = ce_check(p);
  if (rc != SSA_OK) return rc;
  if (!lse || !grad_loss || (p->reduction == 1 && !count))
    return abi_error(SSA_ERR_NULL, "linear_ce: lse, grad_loss or count is NULL");
  if (((uintptr_t)dx | (uintptr_t)dw) % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "linear_ce: dx and dw must be 16-byte aligned");
  if (!dx && !dw) return SSA_OK;
  if ((rc = abi_bind_device(p->x, "x")) != SSA_OK) return rc;
  const CePlan q = ce_plan(p);
  if (!workspace || workspace_bytes < q.bwd_bytes || (uintptr_t)workspace % 256)
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu", q.bwd_bytes,
                     workspace_bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return p->dtype == SSA_DTYPE_BF16
             ? ce_bwd<true>(p, q, lse, count, grad_loss, dx, dw, ws, st)
             : ce_bwd<false>(p, q, lse, count, grad_loss, dx, dw, ws, st);
}

}  // extern "C"

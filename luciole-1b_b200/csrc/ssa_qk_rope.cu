// ssa_qk_rope.cu — queries and keys out of the packed qkv projection: per-head RMS norm (optional)
// and position rotation in one pass, and the backward into the gradient of qkv.
//     n = x r w,  r = rsqrt(mean(x^2) + eps);   y = n cos + rot(n) sin,  rot([a, b]) = [-b, a]
//     dn = dy cos + rot^T(dy sin),  rot^T([a, b]) = [b, -a]
//     dw = sum dn x r,  dx = r (dn w - x r mean(dn w x r))
// Everything in fp32, one rounding at the end.
//
// Bound: memory. D / 8 lanes share a head; a lane holds 4 columns of the first half and the 4 they
// rotate with, so the rotation needs no exchange and the norm a few shuffles. A lane walks kHeads
// heads of one token with that token's cos and sin in registers (a table row is 4 to 8 times as wide
// as a 16-bit head), all heads' loads issued before the first is used: 8 heads forward (65,536
// tokens of 32 + 8 heads of 64, no norm: 4 heads 114 us, 8 heads 110 us; heads_per_lane has more),
// 4 backward, where more registers leave too few warps. Few tokens: one head each. What is read is
// not read again here (streaming loads); what is written is left in L2 for the attention, unless it
// is larger than that (streaming stores: 115 us without, 105 us with, 6.4 TB/s).
//
// A position outside the tables gives NaN; nothing is read out of range.
#include <type_traits>

#include "ssa_internal.h"
#include "ssa_sm100.cuh"

namespace ssa {
namespace {

constexpr int kThreads = 256;

struct RopeArgs {
  int B, S, Hq, Hkv;
  TensorRef qkv;
  const float* cos;
  const float* sin;
  int table_rows;
  const void* pos;     // nullptr: the row's index in its sequence
  int pos64;
  int64_t pos_sB;      // positions per sequence (0: shared by all)
  const void* qw;      // nullptr: no norm
  const void* kw;
  int w_f32;
  float eps;
  void* q;             // forward outputs, [B, S, H, D] contiguous
  void* k;
  TensorRef dq, dk, dv;
  void* dqkv;          // [B, S, (Hq + 2 Hkv) D] contiguous
  float* part;         // [blocks of q, then of k][D]
  int bq, bk, bv;      // backward blocks for queries, keys and values
  bool stream;         // what is written does not stay in L2
};

template <typename T>
using Words = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;  // four elements

template <typename T>
struct Row8 {  // a lane's elements of a head: 4 of each half
  Words<T> a, b;
};

template <typename T>
__device__ __forceinline__ Row8<T> load_row(const T* head, int lane, int D) {
  return Row8<T>{__ldcs(reinterpret_cast<const Words<T>*>(head + lane * 4)),
                 __ldcs(reinterpret_cast<const Words<T>*>(head + D / 2 + lane * 4))};
}
template <typename T>
__device__ __forceinline__ void unpack(const Row8<T>& r, float (&a)[4], float (&b)[4]) {
  const T* x = reinterpret_cast<const T*>(&r.a);
  const T* y = reinterpret_cast<const T*>(&r.b);
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = to_f32<T>(x[i]), b[i] = to_f32<T>(y[i]);
}
template <typename T>
__device__ __forceinline__ void store_row(T* head, int lane, int D, const float (&a)[4],
                                          const float (&b)[4], bool stream) {
  Row8<T> r;
  T* x = reinterpret_cast<T*>(&r.a);
  T* y = reinterpret_cast<T*>(&r.b);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = from_f32<T>(a[i]), y[i] = from_f32<T>(b[i]);
  if (stream) {
    __stcs(reinterpret_cast<Words<T>*>(head + lane * 4), r.a);
    __stcs(reinterpret_cast<Words<T>*>(head + D / 2 + lane * 4), r.b);
  } else {
    *reinterpret_cast<Words<T>*>(head + lane * 4) = r.a;
    *reinterpret_cast<Words<T>*>(head + D / 2 + lane * 4) = r.b;
  }
}

__device__ __forceinline__ void load4f(const float* p, float (&v)[4]) {
  const float4 x = __ldg(reinterpret_cast<const float4*>(p));
  v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
}

struct Angles {
  float ca[4], cb[4], sa[4], sb[4];
};

// cos and sin of row (b, s) for this lane's columns.
template <int D>
__device__ __forceinline__ void load_angles(const RopeArgs& a, int b, int s, int lane, Angles& t) {
  int64_t p = s;
  if (a.pos) {
    const int64_t at = (int64_t)b * a.pos_sB + s;
    p = a.pos64 ? __ldg(reinterpret_cast<const long long*>(a.pos) + at)
                : (int64_t)__ldg(reinterpret_cast<const int*>(a.pos) + at);
  }
  if (p < 0 || p >= a.table_rows) {
#pragma unroll
    for (int i = 0; i < 4; ++i) t.ca[i] = t.cb[i] = t.sa[i] = t.sb[i] = nan_f32();
    return;
  }
  const int64_t o = p * D + lane * 4;
  load4f(a.cos + o, t.ca);
  load4f(a.cos + o + D / 2, t.cb);
  load4f(a.sin + o, t.sa);
  load4f(a.sin + o + D / 2, t.sb);
}

template <typename T, int D>
__device__ __forceinline__ void load_weight(const void* w, int f32, int lane, float (&a)[4],
                                            float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = lane * 4 + i;
    a[i] = f32 ? __ldg(reinterpret_cast<const float*>(w) + c)
               : to_f32<T>(reinterpret_cast<const T*>(w)[c]);
    b[i] = f32 ? __ldg(reinterpret_cast<const float*>(w) + D / 2 + c)
               : to_f32<T>(reinterpret_cast<const T*>(w)[D / 2 + c]);
  }
}

// Sum over the D / 8 lanes of a head.
template <int D>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = D / 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A lane's heads are all queries or all keys, so with the norm the weights join that token's cos and sin
// once: y_a = r (x_a (w_a cos_a) - x_b (w_b sin_a)), y_b = r (x_b (w_b cos_b) + x_a (w_a sin_b)).
template <typename T, int D, int kHeads, bool NORM>
__global__ void __launch_bounds__(kThreads) rope_fwd_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = D / 8, G = kThreads / L;
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  const int lane = threadIdx.x % L;
  const int qslots = (a.Hq + kHeads - 1) / kHeads, slots = qslots + (a.Hkv + kHeads - 1) / kHeads;
  const int64_t items = (int64_t)a.B * a.S * slots;
  int64_t item = (int64_t)blockIdx.x * G + threadIdx.x / L;
  const bool live = item < items;  // lanes past the end repeat the last item and store nothing
  if (!live) item = items - 1;
  const int64_t tok = item / slots;
  const int slot = (int)(item - tok * slots);
  const bool is_k = slot >= qslots;
  const int H = is_k ? a.Hkv : a.Hq, h0 = (is_k ? slot - qslots : slot) * kHeads;
  const int b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
  const T* row = reinterpret_cast<const T*>(a.qkv.ptr) + (int64_t)b * a.qkv.sB + (int64_t)s * a.qkv.sN +
                 (is_k ? (int64_t)a.Hq * a.qkv.sH : 0);
  Row8<T> x[kHeads];
#pragma unroll
  for (int j = 0; j < kHeads; ++j)
    x[j] = load_row<T>(row + (int64_t)min(h0 + j, H - 1) * a.qkv.sH, lane, D);
  Angles t;
  load_angles<D>(a, b, s, lane, t);
  if constexpr (NORM) {
    float wa[4], wb[4];
    load_weight<T, D>(is_k ? a.kw : a.qw, a.w_f32, lane, wa, wb);
#pragma unroll
    for (int i = 0; i < 4; ++i) t.ca[i] *= wa[i], t.sa[i] *= wb[i], t.cb[i] *= wb[i], t.sb[i] *= wa[i];
  }
  T* out = reinterpret_cast<T*>(is_k ? a.k : a.q) + (tok * H + h0) * D;
#pragma unroll
  for (int j = 0; j < kHeads; ++j) {
    float u[4], v[4], ya[4], yb[4], r = 1.f;
    unpack<T>(x[j], u, v);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fmaf(u[i], u[i], fmaf(v[i], v[i], ss));
      r = rsqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ya[i] = fmaf(u[i], t.ca[i], -v[i] * t.sa[i]);
      yb[i] = fmaf(v[i], t.cb[i], u[i] * t.sb[i]);
      if (NORM) ya[i] *= r, yb[i] *= r;
    }
    if (live && h0 + j < H) store_row<T>(out + j * D, lane, D, ya, yb, a.stream);
  }
}

// Blocks [0, bq) take queries, the next bk keys, the next bv copy the values' gradient.
template <typename T, int D, int kHeads, bool NORM>
__global__ void __launch_bounds__(kThreads) rope_bwd_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int L = D / 8, G = kThreads / L;
  __shared__ float red[NORM ? kThreads * 8 : 1];
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  int blk = blockIdx.x;
  const int kind = blk < a.bq ? 0 : blk < a.bq + a.bk ? 1 : 2;
  blk -= kind == 0 ? 0 : kind == 1 ? a.bq : a.bq + a.bk;
  const int nblk = kind == 0 ? a.bq : kind == 1 ? a.bk : a.bv;
  const int H = kind == 0 ? a.Hq : a.Hkv;
  const int base = kind == 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hkv;  // first head within qkv
  const TensorRef& g = kind == 0 ? a.dq : kind == 1 ? a.dk : a.dv;
  const int slots = (H + kHeads - 1) / kHeads;
  const int64_t items = (int64_t)a.B * a.S * slots;
  const int64_t C = (int64_t)(a.Hq + 2 * a.Hkv) * D;
  float wa[4], wb[4], dwa[4], dwb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) wa[i] = wb[i] = dwa[i] = dwb[i] = 0.f;
  if (NORM && kind < 2) load_weight<T, D>(kind ? a.kw : a.qw, a.w_f32, lane, wa, wb);
  // An item's rows: its gradients and, for the norm, its projections. With the norm's arithmetic the next
  // item's are on their way while this one's are used (8192 tokens of 32 + 8 heads of 64: 48 -> 41
  // us; without the norm that only costs warps: 135 -> 159 us at 65,536 tokens). Every lane of the block makes the same number of turns: the
  // shuffles need whole warps.
  struct Item {
    int64_t tok;
    int b, s, h0;
    bool live;
  };
  auto find = [&](int64_t at) {
    Item it;
    int64_t item = at + group;
    it.live = item < items;
    if (!it.live) item = items - 1;
    it.tok = item / slots;
    it.h0 = (int)(item - it.tok * slots) * kHeads;
    it.b = (int)(it.tok / a.S);
    it.s = (int)(it.tok - (int64_t)it.b * a.S);
    return it;
  };
  Row8<T> gr[kHeads], xr[kHeads];
  auto load = [&](const Item& it) {
    const T* grow = reinterpret_cast<const T*>(g.ptr) + (int64_t)it.b * g.sB + (int64_t)it.s * g.sN;
    const T* xrow = reinterpret_cast<const T*>(a.qkv.ptr) + (int64_t)it.b * a.qkv.sB +
                    (int64_t)it.s * a.qkv.sN + (int64_t)base * a.qkv.sH;
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const int h = min(it.h0 + j, H - 1);
      gr[j] = load_row<T>(grow + (int64_t)h * g.sH, lane, D);
      if (NORM && kind < 2) xr[j] = load_row<T>(xrow + (int64_t)h * a.qkv.sH, lane, D);
    }
  };
  int64_t at = (int64_t)blk * G;
  Item it = find(at);
  if (NORM && at < items) load(it);
  for (; at < items;) {
    if (!NORM) load(it);
    T* orow = reinterpret_cast<T*>(a.dqkv) + it.tok * C + (int64_t)base * D;
    const int h0 = it.h0;
    const bool live = it.live;
    Angles t;
    if (kind < 2) load_angles<D>(a, it.b, it.s, lane, t);
    Row8<T> g0[kHeads], x0[kHeads];
#pragma unroll
    for (int j = 0; j < kHeads; ++j) g0[j] = gr[j], x0[j] = xr[j];
    at += (int64_t)nblk * G;
    if (at < items) {
      it = find(at);
      if (NORM) load(it);
    }
#pragma unroll
    for (int j = 0; j < kHeads; ++j) {
      const bool on = live && h0 + j < H;
      float ga[4], gb[4], na[4], nb[4];
      unpack<T>(g0[j], ga, gb);
      if (kind == 2) {
        if (on) store_row<T>(orow + (int64_t)(h0 + j) * D, lane, D, ga, gb, a.stream);
        continue;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        na[i] = fmaf(ga[i], t.ca[i], gb[i] * t.sb[i]);
        nb[i] = fmaf(gb[i], t.cb[i], -ga[i] * t.sa[i]);
      }
      if constexpr (NORM) {
        float xa[4], xb[4], ss = 0.f, c = 0.f;
        unpack<T>(x0[j], xa, xb);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
#pragma unroll
        for (int i = 0; i < 4; ++i)  // sum of dn w x; r enters after
          c = fmaf(na[i] * wa[i], xa[i], fmaf(nb[i] * wb[i], xb[i], c));
        const float r = rsqrtf(head_sum<D>(ss) * (1.f / D) + a.eps);
        c = head_sum<D>(c) * (1.f / D) * r * r;
        const float ro = on ? r : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dwa[i] = fmaf(na[i] * xa[i], ro, dwa[i]), dwb[i] = fmaf(nb[i] * xb[i], ro, dwb[i]);
          na[i] = r * fmaf(-xa[i], c, na[i] * wa[i]);
          nb[i] = r * fmaf(-xb[i], c, nb[i] * wb[i]);
        }
      }
      if (on) store_row<T>(orow + (int64_t)(h0 + j) * D, lane, D, na, nb, a.stream);
    }
  }
  if constexpr (NORM) {
    if (kind == 2) return;  // block-uniform
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red[group * D + lane * 4 + i] = dwa[i];
      red[group * D + D / 2 + lane * 4 + i] = dwb[i];
    }
    __syncthreads();
    if ((int)threadIdx.x < D) {
      double s = 0.0;
      for (int i = 0; i < G; ++i) s += (double)red[i * D + threadIdx.x];
      a.part[((int64_t)blockIdx.x) * D + threadIdx.x] = (float)s;
    }
  }
}

// dw of queries (blockIdx.y = 0) and keys (1), 16 columns a block: their blocks' partial sums, in a
// fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(1024)
    rope_dw_kernel(const float* part, int bq, int bk, void* dqw, void* dkw, int w_f32) {
  __shared__ double red[1024];
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  const int first = blockIdx.y ? bq : 0, n = blockIdx.y ? bk : bq;
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), y = threadIdx.x >> 4;
  double s = 0.0;
  for (int i = y; i < n; i += 8 * 64) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = i + k * 64 < n ? part[(int64_t)(first + i + k * 64) * D + c] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += (double)x[k];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (y < o) red[threadIdx.x] += red[threadIdx.x + o * 16];
    __syncthreads();
  }
  if (y == 0) {
    void* out = blockIdx.y ? dkw : dqw;
    if (!out) return;
    if (w_f32) reinterpret_cast<float*>(out)[c] = (float)red[threadIdx.x];
    else reinterpret_cast<T*>(out)[c] = from_f32<T>((float)red[threadIdx.x]);
  }
}

constexpr int kPlanBlocks = 148 * 4;  // most backward blocks

struct RopePlan {
  int bq, bk, bv;
  size_t bytes;
};

// Several heads per lane once that still leaves every multiprocessor several blocks: 4 from 2.4
// million elements on, 8 forward from 19 million on. Forward, 32 + 8 heads of 64, inputs from memory,
// 4 against 8: 5 million elements 5.7 and 6.7 us (with norm 7.9 and 6.6), 10 million 9.2 and 9.7 (12.2
// and 10.9), 21 million 17.1 and 17.1 (22.2 and 19.1), 78 million 54.6 and 51.8 (69.9 and 62.9), 168
// million 114 and 110 (145 and 130); fp32 within 1% everywhere.
int64_t elements(const ssa_qk_rope_t* p) { return (int64_t)p->B * p->S * (p->Hq + p->Hkv) * p->D; }
int heads_per_lane(const ssa_qk_rope_t* p) {
  return elements(p) >= 148 * 16384 * 8 ? 8 : elements(p) >= 148 * 16384 ? 4 : 1;
}

RopePlan rope_plan(const ssa_qk_rope_t* p) {
  RopePlan q{};
  const int kh = heads_per_lane(p) > 1 ? 4 : 1;
  const int G = kThreads / (p->D / 8);
  auto blocks = [&](int H) {
    return ((int64_t)p->B * p->S * ((H + kh - 1) / kh) + G - 1) / G;
  };
  const int64_t nq = blocks(p->Hq), nk = blocks(p->Hkv), all = nq + 2 * nk;
  auto share = [&](int64_t n) {
    if (all <= kPlanBlocks) return (int)n;
    const int64_t s = n * kPlanBlocks / all;
    return (int)(s < 1 ? 1 : s);
  };
  q.bq = share(nq), q.bk = share(nk), q.bv = share(nk);
  q.bytes = p->q_weight ? sizeof(float) * (size_t)(q.bq + q.bk) * p->D : 0;
  return q;
}

int rope_check(const ssa_qk_rope_t* p) {
  if (!p) return abi_error(SSA_ERR_NULL, "problem is NULL");
  if (p->dtype < SSA_DTYPE_F32 || p->dtype > SSA_DTYPE_BF16)
    return abi_error(SSA_ERR_UNSUPPORTED, "qk_rope: unsupported dtype %d", p->dtype);
  if (p->B <= 0 || p->S <= 0 || p->Hq <= 0 || p->Hkv <= 0 || p->table_rows <= 0)
    return abi_error(SSA_ERR_BAD_SHAPE, "qk_rope: non-positive shape B=%d S=%d Hq=%d Hkv=%d rows=%d",
                     p->B, p->S, p->Hq, p->Hkv, p->table_rows);
  if (p->D != 16 && p->D != 32 && p->D != 64 && p->D != 128)
    return abi_error(SSA_ERR_UNSUPPORTED, "qk_rope: head dim D=%d not supported (16, 32, 64, 128)",
                     p->D);
  if ((int64_t)p->B * p->S * ((int64_t)p->Hq + 2 * (int64_t)p->Hkv) > ((int64_t)1 << 32))
    return abi_error(SSA_ERR_BAD_SHAPE, "qk_rope: more than 2^32 head rows");
  if (!p->qkv.ptr || !p->cos || !p->sin)
    return abi_error(SSA_ERR_NULL, "qk_rope: qkv, cos or sin is NULL");
  if (!p->q_weight != !p->k_weight)
    return abi_error(SSA_ERR_NULL, "qk_rope: q_weight and k_weight come together or not at all");
  if (((uintptr_t)p->cos | (uintptr_t)p->sin) % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "qk_rope: cos and sin must be 16-byte aligned");
  if (p->weight_dtype != p->dtype && p->weight_dtype != SSA_DTYPE_F32)
    return abi_error(SSA_ERR_UNSUPPORTED, "qk_rope: weights are fp32 or of the inputs' dtype");
  return SSA_OK;
}

int check_rows(const ssa_tensor_t& t, int dtype, const char* name) {
  const int rc = abi_check_tensor(t, name);
  if (rc != SSA_OK) return rc;
  const int64_t es = dtype == SSA_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)t.ptr % 16 || t.sB * es % 16 || t.sH * es % 16 || t.sN * es % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "%s: base and strides must be 16-byte aligned", name);
  return SSA_OK;
}

RopeArgs rope_args(const ssa_qk_rope_t* p) {
  RopeArgs a{};
  a.B = p->B, a.S = p->S, a.Hq = p->Hq, a.Hkv = p->Hkv;
  a.qkv = TensorRef{p->qkv.ptr, p->qkv.sB, p->qkv.sH, p->qkv.sN};
  a.cos = p->cos, a.sin = p->sin, a.table_rows = p->table_rows;
  a.pos = p->positions, a.pos64 = p->positions_64, a.pos_sB = p->positions_stride;
  a.qw = p->q_weight, a.kw = p->k_weight;
  a.w_f32 = p->weight_dtype == SSA_DTYPE_F32 && p->dtype != SSA_DTYPE_F32 ? 1 : 0;
  a.eps = p->eps;
  const int64_t written = elements(p) * (p->dtype == SSA_DTYPE_F32 ? 4 : 2);
  a.stream = written > ((int64_t)96 << 20);
  return a;
}

template <typename T, int D, int kHeads, bool NORM>
int run_fwd(const RopeArgs& a, cudaStream_t st) {
  const int64_t items =
      (int64_t)a.B * a.S * ((a.Hq + kHeads - 1) / kHeads + (a.Hkv + kHeads - 1) / kHeads);
  const int G = kThreads / (D / 8);
  const cudaError_t e = sm100::launch_pdl(rope_fwd_kernel<T, D, kHeads, NORM>,
                                          dim3((unsigned)((items + G - 1) / G)), dim3(kThreads), 0, st, a);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "qk_rope_fwd: %s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

template <typename T, int D, int kHeads, bool NORM>
int run_bwd(const RopeArgs& a, void* dqw, void* dkw, cudaStream_t st) {
  cudaError_t e = sm100::launch_pdl(rope_bwd_kernel<T, D, kHeads, NORM>,
                                    dim3((unsigned)(a.bq + a.bk + a.bv)), dim3(kThreads), 0, st, a);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "qk_rope_bwd: %s", cudaGetErrorString(e));
  note_launches(1);
  if (NORM && (dqw || dkw)) {
    e = sm100::launch_pdl(rope_dw_kernel<T, D>, dim3(D / 16, 2), dim3(1024), 0, st, (const float*)a.part,
                          a.bq, a.bk, dqw, dkw, a.w_f32);
    if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "qk_rope_dw: %s", cudaGetErrorString(e));
    note_launches(1);
  }
  return SSA_OK;
}

template <typename T, int D, bool NORM>
int dispatch_norm(const RopeArgs& a, int heads, bool fwd, void* dqw, void* dkw, cudaStream_t st) {
  if (fwd)
    return heads == 8   ? run_fwd<T, D, 8, NORM>(a, st)
           : heads == 4 ? run_fwd<T, D, 4, NORM>(a, st)
                        : run_fwd<T, D, 1, NORM>(a, st);
  return heads > 1 ? run_bwd<T, D, 4, NORM>(a, dqw, dkw, st) : run_bwd<T, D, 1, NORM>(a, dqw, dkw, st);
}

template <typename T, int D>
int dispatch(const RopeArgs& a, int heads, bool fwd, void* dqw, void* dkw, cudaStream_t st) {
  return a.qw ? dispatch_norm<T, D, true>(a, heads, fwd, dqw, dkw, st)
              : dispatch_norm<T, D, false>(a, heads, fwd, dqw, dkw, st);
}

template <typename T>
int dispatch_d(int D, const RopeArgs& a, int heads, bool fwd, void* dqw, void* dkw, cudaStream_t st) {
  switch (D) {
    case 16: return dispatch<T, 16>(a, heads, fwd, dqw, dkw, st);
    case 32: return dispatch<T, 32>(a, heads, fwd, dqw, dkw, st);
    case 64: return dispatch<T, 64>(a, heads, fwd, dqw, dkw, st);
    default: return dispatch<T, 128>(a, heads, fwd, dqw, dkw, st);
  }
}

int dispatch_t(const ssa_qk_rope_t* p, const RopeArgs& a, bool fwd, void* dqw, void* dkw,
               cudaStream_t st) {
  const int heads = heads_per_lane(p);
  switch (p->dtype) {
    case SSA_DTYPE_F32: return dispatch_d<float>(p->D, a, heads, fwd, dqw, dkw, st);
    case SSA_DTYPE_F16: return dispatch_d<__half>(p->D, a, heads, fwd, dqw, dkw, st);
    default: return dispatch_d<__nv_bfloat16>(p->D, a, heads, fwd, dqw, dkw, st);
  }
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" {

int ssa_qk_rope_fwd(const ssa_qk_rope_t* p, void* q, void* k, void* stream) {
  abi_clear_error();
  int rc = rope_check(p);
  if (rc != SSA_OK) return rc;
  if ((rc = check_rows(p->qkv, p->dtype, "qkv")) != SSA_OK) return rc;
  if (!q || !k) return abi_error(SSA_ERR_NULL, "qk_rope: q or k is NULL");
  if (((uintptr_t)q | (uintptr_t)k) % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "qk_rope: q and k must be 16-byte aligned");
  if ((rc = abi_bind_device(p->qkv.ptr, "qkv")) != SSA_OK) return rc;
  RopeArgs a = rope_args(p);
  a.q = q, a.k = k;
  return dispatch_t(p, a, true, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

size_t ssa_qk_rope_bwd_workspace_size(const ssa_qk_rope_t* p) {
  abi_clear_error();
  return rope_check(p) == SSA_OK ? rope_plan(p).bytes : 0;
}

int ssa_qk_rope_bwd(const ssa_qk_rope_t* p, ssa_tensor_t dq, ssa_tensor_t dk, ssa_tensor_t dv,
                    void* dqkv, void* dq_weight, void* dk_weight, void* workspace,
                    size_t workspace_bytes, void* stream) {
  abi_clear_error();
  int rc = rope_check(p);
  if (rc != SSA_OK) return rc;
  if ((rc = check_rows(p->qkv, p->dtype, "qkv")) || (rc = check_rows(dq, p->dtype, "dq")) ||
      (rc = check_rows(dk, p->dtype, "dk")) || (rc = check_rows(dv, p->dtype, "dv")))
    return rc;
  if (!dqkv) return abi_error(SSA_ERR_NULL, "qk_rope: dqkv is NULL");
  if ((uintptr_t)dqkv % 16)
    return abi_error(SSA_ERR_BAD_STRIDE, "qk_rope: dqkv must be 16-byte aligned");
  const RopePlan q = rope_plan(p);
  if (q.bytes && (!workspace || workspace_bytes < q.bytes || (uintptr_t)workspace % 256))
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu",
                     q.bytes, workspace_bytes);
  if ((rc = abi_bind_device(p->qkv.ptr, "qkv")) != SSA_OK) return rc;
  RopeArgs a = rope_args(p);
  a.dq = TensorRef{dq.ptr, dq.sB, dq.sH, dq.sN};
  a.dk = TensorRef{dk.ptr, dk.sB, dk.sH, dk.sN};
  a.dv = TensorRef{dv.ptr, dv.sB, dv.sH, dv.sN};
  a.dqkv = dqkv;
  a.part = static_cast<float*>(workspace);
  a.bq = q.bq, a.bk = q.bk, a.bv = q.bv;
  return dispatch_t(p, a, false, dq_weight, dk_weight, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

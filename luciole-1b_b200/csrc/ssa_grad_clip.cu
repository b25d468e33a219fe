// ssa_grad_clip.cu — the 2-norm over a list of gradient tensors, and the gradients scaled by
// min(1, max_norm / (norm + 1e-6)), in place or into fp32 tensors (an optimizer's master
// gradients, which saves their separate conversion).
//
// Bound: memory. The norm reads every gradient once; the scaling needs the norm, so it reads them
// again and writes once. The tensors' addresses and sizes travel in the kernels' parameter block
// (no table copy to the device, nothing to keep alive, capturable as it is), up to kTable tensors
// per launch. Work is cut into chunks of 64 KB, one block each; the second pass walks the
// chunks from the last to the first, so that what the first pass read last is still in L2.
//
// Squares are added in fp32 over the elements of a 16-byte load and in fp64 from there on, in a fixed
// order: the norm is the same from run to run. A thread whose sum overflowed, or is so small that
// squares may have been lost, adds its elements again in fp64.
#include <algorithm>
#include <cmath>
#include <exception>
#include <vector>

#include "ssa_internal.h"
#include "ssa_sm100.cuh"

namespace ssa {
namespace {

constexpr int kThreads = 512;
constexpr int kLoads = 8;                         // 16-byte loads a thread has under way per chunk
template <typename T>
constexpr int kChunkOf = kThreads * kLoads * 16 / (int)sizeof(T);  // elements: 64 KB

struct TableEntry {
  const void* in;
  void* out;
  int64_t n;
  int32_t first;     // index of the tensor's first chunk among the launch's chunks
  int32_t vec;       // 16-byte accesses are aligned on both sides
};

template <int kTable>
struct Table {
  int32_t tensors;
  int32_t chunks;
  TableEntry t[kTable];
};

// Four elements of a thread: 8 or 16 bytes, so that a warp's accesses are contiguous on both sides when
// 16-bit gradients are written as fp32.
template <typename T>
struct Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ Four<T> load4(const T* p) {
  using W = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
  const W x = *reinterpret_cast<const W*>(p);
  return *reinterpret_cast<const Four<T>*>(&x);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const Four<T>& f) {
  using W = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
  __stcs(reinterpret_cast<W*>(p), *reinterpret_cast<const W*>(&f));  // not read again here
}

// The tensor of a chunk: the last entry whose first chunk is not past it.
template <int kTable>
__device__ __forceinline__ int find_tensor(const Table<kTable>& t, int chunk) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.t[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A thread's elements of a chunk again, in fp64 (from memory: the rare case costs no registers).
template <typename T>
__device__ __noinline__ double sum_squares_64(const T* in, int64_t first, int64_t n) {
  constexpr int E = 16 / (int)sizeof(T);
  double d = 0.0;
  for (int u = 0; u < kLoads; ++u)
    for (int i = 0; i < E; ++i) {
      const int64_t at = first + (int64_t)u * kThreads * E + i;
      if (at < n) d = fma((double)to_f32<T>(in[at]), (double)to_f32<T>(in[at]), d);
    }
  return d;
}

template <typename T, int kTable>
__global__ void __launch_bounds__(kThreads)
    sum_squares_kernel(const __grid_constant__ Table<kTable> tab, double* part) {
  constexpr int E = 16 / (int)sizeof(T);  // elements of a 16-byte load
  __shared__ double red[kThreads / 32];
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  const TableEntry& e = tab.t[find_tensor(tab, (int)blockIdx.x)];
  const int64_t base = (int64_t)((int)blockIdx.x - e.first) * kChunkOf<T>;
  const T* in = reinterpret_cast<const T*>(e.in);
  uint4 raw[kLoads];
  if (e.vec && base + kChunkOf<T> <= e.n) {
    const uint4* p = reinterpret_cast<const uint4*>(in + base) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) raw[u] = p[u * kThreads];
  } else if (e.vec) {  // a tensor's end: one load may reach past it
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t at = base + (int64_t)(u * kThreads + (int)threadIdx.x) * E;
      raw[u] = at + E <= e.n ? *reinterpret_cast<const uint4*>(in + at) : make_uint4(0u, 0u, 0u, 0u);
      if (at < e.n && at + E > e.n) {
        T* t = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
        for (int i = 0; i < E - 1; ++i)
          if (at + i < e.n) t[i] = in[at + i];
      }
    }
  } else {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int64_t at = base + (int64_t)(u * kThreads + (int)threadIdx.x) * E;
      T* t = reinterpret_cast<T*>(&raw[u]);
#pragma unroll
      for (int i = 0; i < E; ++i) t[i] = at + i < e.n ? in[at + i] : from_f32<T>(0.f);
    }
  }
  // A load's squares in pairs and fours in fp32 (4 roundings at most), the rest in fp64: gradients
  // that repeat a pattern would otherwise repeat its rounding error (factor 9.7e-8 off with all of a
  // thread's sum in fp32, 3e-8 so; 990 million elements 1179 -> 1187 us).
  double d = 0.0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const T* t = reinterpret_cast<const T*>(&raw[u]);
    float q[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float x = to_f32<T>(t[2 * i]), y = to_f32<T>(t[2 * i + 1]);
      q[i] = fmaf(x, x, y * y);
    }
#pragma unroll
    for (int o = E / 4; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < o; ++i) q[i] += q[i + o];
    d += (double)q[0];
  }
  // fp32 squares overflow above 1.8e19 and lose digits below 1e-18 or so. All zero (rows of an
  // embedding that no token reached): nothing to redo.
  if (!(d < 3.0e38) || d < 1.0e-30) {
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) any |= raw[u].x | raw[u].y | raw[u].z | raw[u].w;
    if (any) d = sum_squares_64<T>(in, base + (int64_t)threadIdx.x * E, e.n);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x < 32) {
    d = threadIdx.x < kThreads / 32 ? red[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (threadIdx.x == 0) part[blockIdx.x] = d;
  }
}

// norm = sqrt of the chunks' sums, coef = min(1, max_norm / (norm + 1e-6)); NaN stays NaN.
__global__ void __launch_bounds__(1024) norm_kernel(const double* part, int64_t n, double max_norm,
                                                    float* norm, float* coef) {
  __shared__ double red[32];
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  double s[8] = {};
  for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
    double x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = i + k * 1024 < n ? part[i + k * 1024] : 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] += x[k];
  }
  double d = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  d = red[threadIdx.x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (threadIdx.x == 0) {
    const double root = sqrt(d);
    const float r = (float)root;
    *norm = r;
    if (coef) {  // rounded once; a norm that fp32 shows as infinite gives 0 (and infinity over it NaN)
      const float c = (float)(max_norm / (isinf(r) ? (double)r : root + 1e-6));
      *coef = c > 1.f ? 1.f : c;
    }
  }
}

template <typename T, typename O, int kTable>
__global__ void __launch_bounds__(kThreads)
    scale_kernel(const __grid_constant__ Table<kTable> tab, const float* coef) {
  sm100::griddep_wait();
  sm100::griddep_launch_dependents();
  const float c = __ldg(coef);
  const int chunk = tab.chunks - 1 - (int)blockIdx.x;  // last chunk first: its data is still in L2
  const TableEntry& e = tab.t[find_tensor(tab, chunk)];
  if (c == 1.f && e.in == e.out) return;  // in place and nothing to scale
  const int64_t base = (int64_t)(chunk - e.first) * kChunkOf<T>;
  const T* in = reinterpret_cast<const T*>(e.in);
  O* out = reinterpret_cast<O*>(e.out);
  constexpr int N = kChunkOf<T> / (4 * kThreads);
  if (e.vec && base + kChunkOf<T> <= e.n) {
    Four<T> x[N];
#pragma unroll
    for (int u = 0; u < N; ++u) x[u] = load4(in + base + (u * kThreads + (int)threadIdx.x) * 4);
#pragma unroll
    for (int u = 0; u < N; ++u) {
      Four<O> y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y.v[i] = from_f32<O>(to_f32<T>(x[u].v[i]) * c);
      store4(out + base + (u * kThreads + (int)threadIdx.x) * 4, y);
    }
  } else {
    // The end of a tensor, or one no vector access fits. A batch is read before any of it is written:
    // in and out may be one, so that the compiler cannot move a read up by itself.
    constexpr int B = 8;
    const int64_t end = base + kChunkOf<T> < e.n ? base + kChunkOf<T> : e.n;
    const int64_t whole = e.vec ? base + (end - base) / 4 * 4 : base;  // in vectors of four up to here
    for (int64_t i0 = base + 4 * (int)threadIdx.x; i0 < whole; i0 += 4 * B * kThreads) {
      Four<T> x[B];
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (i0 + 4 * u * kThreads < whole) x[u] = load4(in + i0 + 4 * u * kThreads);
#pragma unroll
      for (int u = 0; u < B; ++u) {
        if (i0 + 4 * u * kThreads >= whole) break;
        Four<O> y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.v[i] = from_f32<O>(to_f32<T>(x[u].v[i]) * c);
        store4(out + i0 + 4 * u * kThreads, y);
      }
    }
    for (int64_t i0 = whole + (int)threadIdx.x; i0 < end; i0 += B * kThreads) {
      T x[B];
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (i0 + u * kThreads < end) x[u] = in[i0 + u * kThreads];
#pragma unroll
      for (int u = 0; u < B; ++u)
        if (i0 + u * kThreads < end) out[i0 + u * kThreads] = from_f32<O>(to_f32<T>(x[u]) * c);
    }
  }
}

int64_t chunks_of(int dtype, int64_t n) {
  const int64_t c = dtype == SSA_DTYPE_F32 ? kChunkOf<float> : kChunkOf<__half>;
  return (n + c - 1) / c;
}

// One launch for tensors [i0, i1) of the list.
template <typename T, typename O, int kTable, bool SCALE>
int launch_table(const ssa_grad_list_t* l, int i0, int i1, double* part, const float* coef,
                 cudaStream_t st) {
  Table<kTable> tab;
  tab.tensors = 0;
  int64_t chunks = 0;
  for (int i = i0; i < i1; ++i) {
    if (l->sizes[i] == 0) continue;
    TableEntry& e = tab.t[tab.tensors++];
    e.in = l->grads[i];
    e.out = l->outs ? l->outs[i] : const_cast<void*>(l->grads[i]);
    e.n = l->sizes[i];
    e.first = (int32_t)chunks;
    e.vec = ((uintptr_t)e.in | (SCALE ? (uintptr_t)e.out : 0)) % 16 == 0;
    chunks += chunks_of(l->dtype, e.n);
  }
  if (!chunks) return SSA_OK;
  tab.chunks = (int32_t)chunks;
  cudaError_t err;
  if constexpr (SCALE)
    err = sm100::launch_pdl(scale_kernel<T, O, kTable>, dim3((unsigned)chunks), dim3(kThreads), 0,
                            st, tab, coef);
  else
    err = sm100::launch_pdl(sum_squares_kernel<T, kTable>, dim3((unsigned)chunks), dim3(kThreads), 0,
                            st, tab, part);
  if (err != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "grad_clip: %s", cudaGetErrorString(err));
  note_launches(1);
  return SSA_OK;
}

// Walks the list in launches of at most 64 or 768 tensors (the parameter block is copied with
// every launch: a short list takes the short one).
template <typename T, typename O, bool SCALE>
int walk(const ssa_grad_list_t* l, double* part, const float* coef, cudaStream_t st) {
  const int step = l->count <= 64 ? 64 : 768;
  int64_t done = 0;
  const int groups = (l->count + step - 1) / step;
  for (int k = 0; k < groups; ++k) {
    const int g = SCALE ? groups - 1 - k : k;
    const int i0 = g * step, i1 = i0 + step < l->count ? i0 + step : l->count;
    const int rc = step == 64
                       ? launch_table<T, O, 64, SCALE>(l, i0, i1, part + done, coef, st)
                       : launch_table<T, O, 768, SCALE>(l, i0, i1, part + done, coef, st);
    if (rc != SSA_OK) return rc;
    if (!SCALE)
      for (int i = i0; i < i1; ++i) done += chunks_of(l->dtype, l->sizes[i]);
  }
  return SSA_OK;
}

template <bool SCALE>
int walk_types(const ssa_grad_list_t* l, double* part, const float* coef, cudaStream_t st) {
  const bool f32 = SCALE && l->out_dtype == SSA_DTYPE_F32;
  switch (l->dtype) {
    case SSA_DTYPE_F32:
      return walk<float, float, SCALE>(l, part, coef, st);
    case SSA_DTYPE_F16:
      return f32 ? walk<__half, float, SCALE>(l, part, coef, st)
                 : walk<__half, __half, SCALE>(l, part, coef, st);
    default:
      return f32 ? walk<__nv_bfloat16, float, SCALE>(l, part, coef, st)
                 : walk<__nv_bfloat16, __nv_bfloat16, SCALE>(l, part, coef, st);
  }
}

int64_t total_chunks(const ssa_grad_list_t* l) {
  int64_t n = 0;
  for (int i = 0; i < l->count; ++i) n += chunks_of(l->dtype, l->sizes[i]);
  return n;
}

struct Range {
  uintptr_t from, to;
  int written, index;
};

// Two blocks may not write the same element, nor one write what another reads: a written tensor
// meets no other tensor. (An output may be its own gradient.)
int check_ranges(const ssa_grad_list_t* l) {
  const size_t es = l->dtype == SSA_DTYPE_F32 ? 4 : 2;
  const size_t eo = l->outs && l->out_dtype == SSA_DTYPE_F32 ? 4 : es;
  try {
    std::vector<Range> r;
    r.reserve(2 * (size_t)l->count);
    for (int i = 0; i < l->count; ++i) {
      if (!l->sizes[i]) continue;
      const uintptr_t in = (uintptr_t)l->grads[i], out = l->outs ? (uintptr_t)l->outs[i] : in;
      r.push_back(Range{out, out + eo * (size_t)l->sizes[i], 1, i});
      if (out != in || eo != es) r.push_back(Range{in, in + es * (size_t)l->sizes[i], 0, i});
    }
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t end_written = 0, end_any = 0;
    for (const Range& x : r) {
      if (x.from < end_written || (x.written && x.from < end_any))
        return abi_error(SSA_ERR_BAD_SHAPE, "grad_clip: tensors that are written must not share "
                         "memory with another (tensor %d)", x.index);
      if (x.to > end_any) end_any = x.to;
      if (x.written && x.to > end_written) end_written = x.to;
    }
  } catch (const std::exception& e) {
    return abi_error(SSA_ERR_CUDA, "grad_clip: %s", e.what());
  }
  return SSA_OK;
}

int list_check(const ssa_grad_list_t* l, bool outs) {
  if (!l) return abi_error(SSA_ERR_NULL, "list is NULL");
  if (l->dtype < SSA_DTYPE_F32 || l->dtype > SSA_DTYPE_BF16)
    return abi_error(SSA_ERR_UNSUPPORTED, "grad_clip: unsupported dtype %d", l->dtype);
  if (l->count < 1) return abi_error(SSA_ERR_BAD_SHAPE, "grad_clip: empty list");
  if (!l->grads || !l->sizes) return abi_error(SSA_ERR_NULL, "grad_clip: grads or sizes is NULL");
  const uintptr_t es = l->dtype == SSA_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < l->count; ++i) {
    if (l->sizes[i] < 0 || l->sizes[i] > ((int64_t)1 << 40))
      return abi_error(SSA_ERR_BAD_SHAPE, "grad_clip: tensor %d has %lld elements", i,
                       (long long)l->sizes[i]);
    if (l->sizes[i] && !l->grads[i])
      return abi_error(SSA_ERR_NULL, "grad_clip: tensor %d is NULL", i);
    if ((uintptr_t)l->grads[i] % es)
      return abi_error(SSA_ERR_BAD_STRIDE, "grad_clip: tensor %d is not aligned to its type", i);
  }
  if (total_chunks(l) > INT32_MAX)
    return abi_error(SSA_ERR_BAD_SHAPE, "grad_clip: too many elements");
  if (!outs) return SSA_OK;
  if (!l->outs) return check_ranges(l);
  if (l->out_dtype != l->dtype && l->out_dtype != SSA_DTYPE_F32)
    return abi_error(SSA_ERR_UNSUPPORTED, "grad_clip: outputs are fp32 or of the gradients' dtype");
  const uintptr_t eo = l->out_dtype == SSA_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < l->count; ++i)
    if (l->sizes[i] && (!l->outs[i] || (uintptr_t)l->outs[i] % eo))
      return abi_error(SSA_ERR_NULL, "grad_clip: output %d is NULL or not aligned to its type", i);
  return check_ranges(l);
}

int first_tensor(const ssa_grad_list_t* l) {
  for (int i = 0; i < l->count; ++i)
    if (l->sizes[i]) return i;
  return -1;
}

int norm_into(const ssa_grad_list_t* l, double* part, double max_norm, float* norm, float* coef,
              cudaStream_t st) {
  int rc = walk_types<false>(l, part, nullptr, st);
  if (rc != SSA_OK) return rc;
  const cudaError_t e = sm100::launch_pdl(norm_kernel, dim3(1), dim3(1024), 0, st,
                                          (const double*)part, total_chunks(l), max_norm, norm, coef);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "grad_norm: %s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

}  // namespace
}  // namespace ssa

using namespace ssa;

extern "C" {

size_t ssa_grad_clip_workspace_size(const ssa_grad_list_t* list) {
  abi_clear_error();
  if (list_check(list, false) != SSA_OK) return 0;
  return 256 + sizeof(double) * (size_t)(total_chunks(list) + 1);
}

int ssa_grad_norm(const ssa_grad_list_t* list, float* norm, void* workspace, size_t workspace_bytes,
                  void* stream) {
  abi_clear_error();
  int rc = list_check(list, false);
  if (rc != SSA_OK) return rc;
  if (!norm) return abi_error(SSA_ERR_NULL, "grad_norm: norm is NULL");
  const size_t need = 256 + sizeof(double) * (size_t)(total_chunks(list) + 1);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu",
                     need, workspace_bytes);
  if ((rc = abi_bind_device(norm, "norm")) != SSA_OK) return rc;
  return norm_into(list, reinterpret_cast<double*>(static_cast<uint8_t*>(workspace) + 256), 0.f,
                   norm, nullptr, static_cast<cudaStream_t>(stream));
}

int ssa_grad_clip(const ssa_grad_list_t* list, double max_norm, float* norm, void* workspace,
                  size_t workspace_bytes, void* stream) {
  abi_clear_error();
  int rc = list_check(list, true);
  if (rc != SSA_OK) return rc;
  if (!norm) return abi_error(SSA_ERR_NULL, "grad_clip: norm is NULL");
  if (!(max_norm >= 0.0))
    return abi_error(SSA_ERR_BAD_SHAPE, "grad_clip: max_norm must not be negative or NaN");
  const size_t need = 256 + sizeof(double) * (size_t)(total_chunks(list) + 1);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 256)
    return abi_error(SSA_ERR_WORKSPACE, "workspace needs %zu bytes (256-byte aligned), got %zu",
                     need, workspace_bytes);
  if ((rc = abi_bind_device(norm, "norm")) != SSA_OK) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  float* coef = reinterpret_cast<float*>(ws);
  double* part = reinterpret_cast<double*>(ws + 256);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = norm_into(list, part, max_norm, norm, coef, st)) != SSA_OK) return rc;
  if (first_tensor(list) < 0) return SSA_OK;
  return walk_types<true>(list, part, coef, st);
}

}  // extern "C"

// ssa_gemm.cu — the plain products of the backward passes (dx and dW) on the core in ssa_gemm.cuh.
#include "ssa_gemm.cuh"

#include <atomic>

namespace ssa {
namespace sm100 {

int device_sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kPlanSms;
  if ((n = counts[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1)
    return kPlanSms;
  counts[dev].store(n, std::memory_order_relaxed);
  return n;
}

namespace {

// The epilogue is kept short: in the 256 x 512 form the next tile's MMAs wait for half of it. The next
// 32 columns are on their way from TMEM while the last ones are stored; 16-bit results are rounded
// before the exchange; a later piece's sum goes out as fp32 reductions, which wait for nothing (one
// addition per element and launch: the order, and so the sum, is fixed by the stream).
template <int BN, bool BF16>
struct EpiStore {
  using Args = StoreArgs;
  struct Row {
    float scale;
  };
  __device__ static __forceinline__ Row row(const Args& a, int row) {
    return Row{a.row_scale && row < a.rows ? __ldg(a.row_scale + row) : 1.f};
  }
  __device__ static __forceinline__ void tile(const Args& a, const GemmUnit& w, const Row& rw,
                                              const EpiCtx& e) {
    const float sc = (a.scale ? __ldg(a.scale) : 1.f) * rw.scale;
    const int col0 = w.nt * BN + e.half * (BN / 2);
    const int n = min(BN / 2, ((a.cols - col0 + 31) >> 5) << 5);  // columns of this warp, whole 32s
    if (n <= 0) return;
    uint32_t x[32];
    e.fetch(e.half * (BN / 2), x);
#pragma unroll 1
    for (int c = 0; c < n; c += 32) {
      const int col = col0 + c;
      float v[32];
      e.settle();
      e.values(x, v);
      if (c + 32 < n) e.fetch(e.half * (BN / 2) + c + 32, x);
      if (a.out) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= sc;
        put_row16<BF16>(e, v, 0xffffffffu);
        __syncwarp();
        const int p = e.lane & 3, my = col + 8 * p;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int r = it * 8 + (e.lane >> 2);
          const int row = e.row0 + r;
          int64_t orow = row;
          bool ok = row < a.rows && my < a.cols;
          if (a.jump_at) {
            const int in = row < a.jump_at ? row : row - a.jump_at;
            ok = ok && in < a.jump_rows;
            orow = row < a.jump_at ? row : (int64_t)a.jump + in;
          }
          if (ok)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + orow * a.ldo + my) =
                *exch16(e.exch, r, p);
        }
      } else {
#pragma unroll
        for (int p = 0; p < 8; ++p)
          *exch32(e.exch, e.lane, p) = make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
        __syncwarp();
        const int p = e.lane & 7, my = col + 4 * p;
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int r = it * 4 + (e.lane >> 3);
          const int row = e.row0 + r;
          if (row >= a.rows || my >= a.cols) continue;
          float4* to = reinterpret_cast<float4*>(a.sum + ((int64_t)w.sp * a.rows + row) * a.cols + my);
          if (a.add_prev) atomicAdd(to, *exch32(e.exch, r, p));
          else *to = *exch32(e.exch, r, p);
        }
      }
      __syncwarp();
    }
  }
};

// out[row, col] = scale * sum over splits, in split order (deterministic).
template <bool BF16>
__global__ void __launch_bounds__(256) sum_splits_kernel(const float* sum, void* out,
                                                         const float* scale, const float* row_scale,
                                                         int64_t rows, int cols, int64_t ldo,
                                                         int splits) {
  griddep_wait();
  griddep_launch_dependents();
  const float all = scale ? __ldg(scale) : 1.f;
  const int per_row = cols / 4;
  const int64_t total = rows * per_row, plane = rows * (int64_t)cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int col = (int)(i - row * per_row) * 4;
    const float* p = sum + row * cols + col;
    const float sc = row_scale ? all * __ldg(row_scale + row) : all;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(p + k * plane);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + row * ldo + col) =
        make_uint2(pack2<BF16>(s.x * sc, s.y * sc), pack2<BF16>(s.z * sc, s.w * sc));
  }
}

template <int CG, int BN, int NH, bool BF16>
int gradients(const StoreProduct* dx, const StoreProduct* dw, cudaStream_t st) {
  using Epi = EpiStore<BN, BF16>;
  auto product = [](const StoreProduct* p) { return GemmProduct<Epi>{p->a, p->b, p->g, p->ea}; };
  if (!dw) return launch_gemm<Epi, CG, BN, NH, 0, true, BF16>(product(dx), nullptr, st);
  if (!dx) return launch_gemm<Epi, CG, BN, NH, 1, true, BF16>(product(dw), nullptr, st);
  const GemmProduct<Epi> second = product(dw);
  return launch_gemm<Epi, CG, BN, NH, 2, true, BF16>(product(dx), &second, st);
}

template <bool BF16>
int gradients_form(const GemmForm& f, const StoreProduct* dx, const StoreProduct* dw,
                   cudaStream_t st) {
  if (f.wide) return gradients<2, 256, 2, BF16>(dx, dw, st);
  return f.pair ? gradients<2, 256, 1, BF16>(dx, dw, st) : gradients<1, 128, 1, BF16>(dx, dw, st);
}

}  // namespace

int launch_gradients(bool bf16, const GemmForm& form, const StoreProduct* dx, const StoreProduct* dw,
                     cudaStream_t st) {
  return bf16 ? gradients_form<true>(form, dx, dw, st) : gradients_form<false>(form, dx, dw, st);
}

int launch_sum_splits(bool bf16, const float* sum, void* out, const float* scale,
                      const float* row_scale, int64_t rows, int cols, int64_t ldo, int splits,
                      cudaStream_t st) {
  const int64_t blocks = (rows * (cols / 4) + 255) / 256;
  const int64_t most = (int64_t)device_sm_count() * 8;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  const cudaError_t e =
      bf16 ? launch_pdl(sum_splits_kernel<true>, grid, dim3(256), 0, st, sum, out, scale,
                        row_scale, rows, cols, ldo, splits)
           : launch_pdl(sum_splits_kernel<false>, grid, dim3(256), 0, st, sum, out, scale,
                        row_scale, rows, cols, ldo, splits);
  if (e != cudaSuccess) return abi_error(SSA_ERR_LAUNCH, "sum_splits: %s", cudaGetErrorString(e));
  note_launches(1);
  return SSA_OK;
}

}  // namespace sm100
}  // namespace ssa

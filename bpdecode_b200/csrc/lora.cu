// Low-rank adapters of many requests beside a projection that they share:
//
//   y[t, n] = sum_k x[t, k] W[n, k] + s_a sum_j (sum_k x[t, k] A_a[j, k]) B_a[n, j]
//
// with a = ids[t], no adapter where ids[t] is outside [0, num_adapters).
#include <algorithm>
#include <climits>

#include "common.cuh"

namespace bpd {
namespace {

constexpr int kTile = 64;   // rows and outputs of a CTA's tile
constexpr int kStep = 16;   // inner elements of one step
constexpr int kTileN = 128; // outputs of a tile of the packed B

struct LoraArgs {
  const void* x;
  int64_t x_stride;
  const void* w;
  int64_t w_stride;
  int32_t T, K, N;
  const void* a;
  const void* b;
  const float* scale;
  int32_t adapters, rank;
  const void* ids;
  int32_t ids64;
  void* out;
  int64_t out_stride;
  float* low;
};

__device__ __forceinline__ int32_t adapter_of(const LoraArgs& g, int32_t t) {
  if (t >= g.T || !g.ids) return -1;
  const int64_t id = g.ids64 ? static_cast<const int64_t*>(g.ids)[t]
                             : static_cast<const int32_t*>(g.ids)[t];
  return id >= 0 && id < g.adapters ? static_cast<int32_t>(id) : -1;
}

// low[t, j] = s_a sum_k x[t, k] A_a[j, k]: one CTA for a row, one warp for a j.
template <typename T>
__global__ void shrink_kernel(const LoraArgs g) {
  pdl_wait();
  const int32_t t = blockIdx.x, lane = threadIdx.x & 31;
  const int32_t a = adapter_of(g, t);
  if (a < 0) return;
  using Bits = typename Dt<T>::Bits;
  const Bits* x = static_cast<const Bits*>(g.x) + t * g.x_stride;
  for (int32_t j = threadIdx.x >> 5; j < g.rank; j += blockDim.x >> 5) {
    const Bits* row = static_cast<const Bits*>(g.a) + (static_cast<int64_t>(a) * g.rank + j) * g.K;
    float s = 0.0f;
    for (int32_t k = lane; k < g.K; k += 32) s += Dt<T>::to_float(x[k]) * Dt<T>::to_float(row[k]);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (lane == 0) g.low[static_cast<int64_t>(t) * g.rank + j] = s * g.scale[a];
  }
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) project_kernel(const LoraArgs g) {
  using Bits = typename Dt<T>::Bits;
  __shared__ float xs[kStep][kTile + 1], ws[kStep][kTile + 1];
  pdl_wait();
  const int32_t n0 = blockIdx.x * kTile, t0 = blockIdx.y * kTile;
  const int32_t tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int32_t k0 = 0; k0 < g.K; k0 += kStep) {
    for (int32_t i = threadIdx.x; i < kTile * kStep; i += 256) {
      const int32_t k = k0 + (i & (kStep - 1)), r = i / kStep;
      xs[i & (kStep - 1)][r] =
          t0 + r < g.T && k < g.K
              ? Dt<T>::to_float(static_cast<const Bits*>(g.x)[(t0 + r) * g.x_stride + k]) : 0.0f;
      ws[i & (kStep - 1)][r] =
          n0 + r < g.N && k < g.K
              ? Dt<T>::to_float(static_cast<const Bits*>(g.w)[(n0 + r) * g.w_stride + k]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kStep; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int32_t t = t0 + ty * 4 + i;
    if (t >= g.T) break;
    const int32_t a = adapter_of(g, t);
    for (int j = 0; j < 4; ++j) {
      const int32_t n = n0 + tx + 16 * j;
      if (n >= g.N) continue;
      float y = acc[i][j];
      if (a >= 0) {
        const Bits* tile = static_cast<const Bits*>(g.b) +
                           (static_cast<int64_t>(a) * ((g.N + kTileN - 1) / kTileN) + n / kTileN) *
                               kTileN * g.rank;
        for (int32_t r = 0; r < g.rank; ++r)
          y += g.low[static_cast<int64_t>(t) * g.rank + r] *
               Dt<T>::to_float(tile[((r >> 3) * kTileN + n % kTileN) * 8 + (r & 7)]);
      }
      static_cast<typename Dt<O>::Bits*>(g.out)[t * g.out_stride + n] = Dt<O>::from_float_dev(y);
    }
  }
}

template <typename T, typename O>
cudaError_t launch_project(const LoraArgs& g, cudaStream_t st) {
  if (g.ids) {
    const cudaError_t e = launch_pdl(shrink_kernel<T>, dim3(g.T), dim3(256), 0, st, g);
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(project_kernel<T, O>, dim3((g.N + kTile - 1) / kTile, (g.T + kTile - 1) / kTile),
                    dim3(256), 0, st, g);
}

}  // namespace
}  // namespace bpd

using namespace bpd;

extern "C" size_t bpd_lora_workspace_bytes(int32_t rows, int32_t rank) {
  return align256(static_cast<size_t>(std::max(rows, 0)) * std::max(rank, 0) * sizeof(float));
}

extern "C" bpd_status bpd_lora_project(const void* x, int64_t x_stride, const void* weight,
                                       int64_t weight_stride, int32_t dtype, int32_t rows,
                                       int32_t in_features, int32_t out_features, const void* a,
                                       const void* b, const float* scale, int32_t num_adapters,
                                       int32_t rank, const void* ids, int32_t ids_int64, void* out,
                                       int32_t out_dtype, int64_t out_stride, void* workspace,
                                       void* stream) {
  const char* what = "bpd_lora_project";
  BPD_REQUIRE(rows >= 0 && in_features > 0 && out_features > 0, "%s: bad sizes", what);
  BPD_REQUIRE(dtype == BPD_BF16 || dtype == BPD_F16, "%s: unsupported dtype %d", what, dtype);
  BPD_REQUIRE(out_dtype == dtype || out_dtype == BPD_F32, "%s: unsupported output dtype %d", what,
              out_dtype);
  if (rows == 0) return BPD_OK;
  BPD_REQUIRE(x && weight && out, "%s: null pointer", what);
  BPD_REQUIRE(in_features % 8 == 0, "%s: in_features must be a multiple of 8", what);
  BPD_REQUIRE(aligned16(x) && aligned16(weight) && x_stride % 8 == 0 && weight_stride % 8 == 0,
              "%s: rows of x and weight must start on 16-byte boundaries", what);
  BPD_REQUIRE(x_stride >= in_features && weight_stride >= in_features &&
                  out_stride >= out_features, "%s: row stride too small", what);
  if (ids) {
    BPD_REQUIRE(num_adapters >= 0, "%s: bad sizes", what);
    if (num_adapters == 0) ids = nullptr;
  }
  if (ids) {
    BPD_REQUIRE(a && b && scale && workspace, "%s: null pointer", what);
    BPD_REQUIRE(rank > 0 && rank % 16 == 0 && rank <= BPD_LORA_MAX_RANK,
                "%s: rank must be a multiple of 16, at most %d", what, BPD_LORA_MAX_RANK);
    BPD_REQUIRE(aligned16(a) && aligned16(b) && aligned16(workspace),
                "%s: adapters and workspace must be 16-byte aligned", what);
  }
  const LoraArgs g{x, x_stride, weight, weight_stride, rows, in_features, out_features, a, b,
                   scale, num_adapters, rank, ids, ids_int64, out, out_stride,
                   static_cast<float*>(workspace)};
  cudaStream_t st = as_stream(stream);
  cudaError_t e;
  if (dtype == BPD_BF16)
    e = out_dtype == BPD_F32 ? launch_project<__nv_bfloat16, float>(g, st)
                             : launch_project<__nv_bfloat16, __nv_bfloat16>(g, st);
  else
    e = out_dtype == BPD_F32 ? launch_project<__half, float>(g, st)
                             : launch_project<__half, __half>(g, st);
  return e == cudaSuccess ? BPD_OK : fail(BPD_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

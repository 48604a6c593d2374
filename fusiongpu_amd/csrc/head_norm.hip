// head_norm.hip -- layer norm over the rows of [rows][dim], forward and backward.
#include <algorithm>
#include <type_traits>

#include "head.hpp"

namespace fgpu {
namespace {

constexpr int kNormVec = 4;      // elements a lane reads at once
constexpr int kNormMaxDim = 16384;

// A row on WAVES waves, V vectors a lane, all of it in registers: dim <= WAVES * 64 * 4 * V.
template <int WAVES, int V>
struct Row {
  f32x4 v[V];
  __device__ static int col(int k) { return (k * WAVES * kWave + (int)threadIdx.x % (WAVES * kWave)) * kNormVec; }
  template <class T>
  __device__ __forceinline__ void load(const T* p, int dim) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      v[k] = f32x4{0, 0, 0, 0};
      if (col(k) < dim) v[k] = load4_n(p + col(k), dim - col(k));
    }
  }
};

// Sum over the lanes of a row (WAVES waves), the same bits in all of them.
template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float* lds) {
  x = wave_sum_f(x);
  if constexpr (WAVES > 1) {
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) x += lds[w];
  }
  return x;
}

template <class T, int WAVES, int V>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void norm_kernel(const T* x, const T* gamma, const T* beta,
                                                                                int64_t rows, int dim, float eps, T* y,
                                                                                float* mean, float* rstd) {
  __shared__ float lds[WAVES];
  constexpr int kRows = WAVES == 1 ? 4 : 1;
  const int64_t r = (int64_t)blockIdx.x * kRows + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  if (r >= rows) return;
  Row<WAVES, V> a;
  a.load(x + r * dim, dim);
  float s = 0;
#pragma unroll
  for (int k = 0; k < V; ++k) s += (a.v[k][0] + a.v[k][1]) + (a.v[k][2] + a.v[k][3]);
  const float mu = row_sum<WAVES>(s, lds) / (float)dim;
  s = 0;
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = a.col(k) + e < dim ? a.v[k][e] - mu : 0.0f;
      a.v[k][e] = d;
      s = fmaf(d, d, s);
    }
  const float rs = 1.0f / sqrtf(row_sum<WAVES>(s, lds) / (float)dim + eps);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = a.col(k), n = dim - c;
    if (n <= 0) continue;
    f32x4 o = a.v[k] * rs;
    if (gamma) o *= load4_n(gamma + c, n);
    if (beta) o += load4_n(beta + c, n);
    store4_n(y + r * dim + c, o, n);
  }
  if ((WAVES == 1 ? lane_id() : threadIdx.x) == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

// Each row group (WAVES waves) walks rows group, group + groups, ... and keeps its part of the two column sums in
// registers; part [group][2][dim].
template <class T, int WAVES, int V>
__global__ __launch_bounds__(WAVES == 1 ? 256 : WAVES * kWave) void norm_backward_kernel(
    const T* dy, const T* x, const T* gamma, const float* mean, const float* rstd, int64_t rows, int dim, T* dx, float* part) {
  __shared__ float lds[WAVES];
  constexpr int kRows = WAVES == 1 ? 4 : 1;
  const int64_t groups = (int64_t)gridDim.x * kRows;
  const int64_t g = (int64_t)blockIdx.x * kRows + (WAVES == 1 ? threadIdx.x >> 6 : 0);
  f32x4 sg[V], sb[V], ga[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = Row<WAVES, V>::col(k), n = dim - c;
    sg[k] = sb[k] = f32x4{0, 0, 0, 0};
    ga[k] = f32x4{1, 1, 1, 1};
    if (gamma && n > 0) ga[k] = load4_n(gamma + c, n);
  }
  for (int64_t r = g; r < rows; r += groups) {
    Row<WAVES, V> a, d;
    a.load(x + r * dim, dim);
    d.load(dy + r * dim, dim);
    const float mu = mean[r], rs = rstd[r];
    float s1 = 0, s2 = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      a.v[k] = (a.v[k] - mu) * rs;
      sg[k] += d.v[k] * a.v[k];  // columns beyond dim have dy = 0
      sb[k] += d.v[k];
      d.v[k] *= ga[k];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s1 += d.v[k][e];
        s2 = fmaf(d.v[k][e], a.v[k][e], s2);
      }
    }
    if (!dx) continue;
    const float m1 = row_sum<WAVES>(s1, lds) / (float)dim, m2 = row_sum<WAVES>(s2, lds) / (float)dim;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = a.col(k), n = dim - c;
      if (n <= 0) continue;
      store4_n(dx + r * dim + c, (d.v[k] - m1 - a.v[k] * m2) * rs, n);
    }
  }
  if (!part) return;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = Row<WAVES, V>::col(k), n = dim - c;
    if (n <= 0) continue;
    store4_n(part + g * 2 * dim + c, sg[k], n);
    store4_n(part + (g * 2 + 1) * dim + c, sb[k], n);
  }
}

// One row a wave up to 1024 dims, a workgroup of four or sixteen waves beyond.
template <class F>
fgpu_status by_dim(int dim, F&& f) {
  if (dim <= 256) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
  if (dim <= 512) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
  if (dim <= 1024) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  if (dim <= 2048) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
  if (dim <= 4096) return f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
}

int norm_groups(int64_t rows, int dim) {  // row groups of the backward pass, a multiple of four
  const int64_t want = dim <= 1024 ? 4096 : dim <= 4096 ? 1024 : 512;
  return (int)(std::min<int64_t>((rows + 3) / 4 * 4, want));
}

fgpu_status check_norm(int64_t rows, int dim, int dtype) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "layer norm: unknown dtype");
  FGPU_CHECK(rows >= 0 && dim >= 1, FGPU_ERR_ARG, "layer norm: rows >= 0 and dim >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && dim <= kNormMaxDim, FGPU_ERR_UNSUPPORTED,
             "layer norm: more than 2^30 rows or 16384 dims");
  return FGPU_OK;
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

fgpu_status fgpu_layer_norm(const void* d_x, const void* d_gamma, const void* d_beta, int64_t rows, int dim, int dtype,
                            float eps, void* d_y, float* d_mean, float* d_rstd, void* stream) {
  FGPU_TRY(check_norm(rows, dim, dtype));
  FGPU_CHECK(eps >= 0.0f, FGPU_ERR_ARG, "layer norm: eps must not be negative");
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_y, FGPU_ERR_ARG, "layer norm: null x or output");
  return by_dim(dim, [&](auto w, auto v) -> fgpu_status {
    constexpr int W = decltype(w)::value, V = decltype(v)::value, kRows = W == 1 ? 4 : 1, kThreads = W == 1 ? 256 : W * kWave;
    const int grid = ceil_div(rows, kRows);
    if (dtype == FGPU_DTYPE_F32)
      norm_kernel<float, W, V><<<grid, kThreads, 0, as_stream(stream)>>>(
          (const float*)d_x, (const float*)d_gamma, (const float*)d_beta, rows, dim, eps, (float*)d_y, d_mean, d_rstd);
    else
      norm_kernel<bf16, W, V><<<grid, kThreads, 0, as_stream(stream)>>>(
          (const bf16*)d_x, (const bf16*)d_gamma, (const bf16*)d_beta, rows, dim, eps, (bf16*)d_y, d_mean, d_rstd);
    FGPU_HIP(hipGetLastError());
    return FGPU_OK;
  });
}

size_t fgpu_layer_norm_backward_workspace_bytes(int64_t rows, int dim, int dtype) {
  if (check_norm(rows, dim, dtype) != FGPU_OK || rows == 0) return 0;
  return carve_bytes<float>((size_t)norm_groups(rows, dim) * 2 * dim);
}

fgpu_status fgpu_layer_norm_backward(const void* d_dy, const void* d_x, const void* d_gamma, const float* d_mean,
                                     const float* d_rstd, int64_t rows, int dim, int dtype, void* d_dx, void* d_dgamma,
                                     void* d_dbeta, void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_norm(rows, dim, dtype));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  if (rows == 0) {
    if (d_dgamma) FGPU_TRY(launch_column_finish(nullptr, 0, 0, dim, f32, d_dgamma, s));
    if (d_dbeta) FGPU_TRY(launch_column_finish(nullptr, 0, 0, dim, f32, d_dbeta, s));
    return FGPU_OK;
  }
  FGPU_CHECK(d_dy && d_x && d_mean && d_rstd, FGPU_ERR_ARG, "layer norm backward: null dy, x, mean or rstd");
  const int groups = norm_groups(rows, dim);
  float* part = nullptr;
  if (d_dgamma || d_dbeta) {
    Carve ws(d_workspace, workspace_bytes);
    part = ws.take<float>((size_t)groups * 2 * dim);
    FGPU_CHECK(ws.ok(), FGPU_ERR_WORKSPACE,
               "layer norm backward: workspace smaller than fgpu_layer_norm_backward_workspace_bytes");
  }
  FGPU_TRY(by_dim(dim, [&](auto w, auto v) -> fgpu_status {
    constexpr int W = decltype(w)::value, V = decltype(v)::value, kRows = W == 1 ? 4 : 1, kThreads = W == 1 ? 256 : W * kWave;
    const int grid = groups / kRows;
    if (f32)
      norm_backward_kernel<float, W, V><<<grid, kThreads, 0, s>>>((const float*)d_dy, (const float*)d_x, (const float*)d_gamma,
                                                                  d_mean, d_rstd, rows, dim, (float*)d_dx, part);
    else
      norm_backward_kernel<bf16, W, V><<<grid, kThreads, 0, s>>>((const bf16*)d_dy, (const bf16*)d_x, (const bf16*)d_gamma,
                                                                 d_mean, d_rstd, rows, dim, (bf16*)d_dx, part);
    FGPU_HIP(hipGetLastError());
    return FGPU_OK;
  }));
  if (d_dgamma) FGPU_TRY(launch_column_finish(part, groups, 2 * dim, dim, f32, d_dgamma, s));
  if (d_dbeta) FGPU_TRY(launch_column_finish(part + dim, groups, 2 * dim, dim, f32, d_dbeta, s));
  return FGPU_OK;
}

}  // extern "C"

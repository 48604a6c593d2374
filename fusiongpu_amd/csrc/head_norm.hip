// head_norm.hip -- layer norm over the rows of [rows][dim], forward and backward.
//
// Forward: mean and variance of a row held in registers (two passes over the registers, one over memory: the variance is
// that of the centred values), y = (x - mean) rstd gamma + beta.  Backward, with h = (x - mean) rstd and u = dy gamma:
// dx = rstd (u - mean(u) - h mean(u h)), dgamma = sum of dy h, dbeta = sum of dy over the rows.
//
// Bound by HBM: every array passes once.  Measured: forward float32 100003 x 771 130 us (4.75 TB/s; a large copy reaches
// 4.94), bf16 65536 x 1024 43 us (its output stays in the last-level cache); backward bf16 65536 x 1024 72 us + 4 us for
// the column sums (5.3 TB/s), float32 153 us.  One row of 1024 takes 2.1 us, a launch's own time.
#include <algorithm>
#include <type_traits>

#include "head.hpp"

namespace fgpu {
namespace {

constexpr int kNormMaxDim = 16384;

// 16 bytes of a row as they lie in memory, eight bf16 or four floats, held as four words (as elements, the compiler would
// unpack them where they are loaded and wait there).
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
template <class T, bool RAGGED>
struct Raw {
  static constexpr int N = 16 / sizeof(T);
  u32x4 w;
  // The first n elements at p.  RAGGED (rows that are no whole number of vectors): a row's last vector reads on into the
  // next row where there is `more`, whose elements Vec::from masks when the data is there; where the array itself ends
  // the last 16 bytes of it are read and moved down.  TINY: the array may be shorter than 16 bytes.
  template <bool TINY>
  __device__ __forceinline__ void load(const T* p, int n, bool more) {
    w = u32x4{0, 0, 0, 0};
    if (n <= 0) return;
    if (!RAGGED || n >= N || more) {
      w = *reinterpret_cast<const u32x4u*>(p);
    } else if (TINY) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (e >= n) break;
        if constexpr (N == 4) w[e] = reinterpret_cast<const uint32_t*>(p)[e];
        else w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (e % 2 * 16);
      }
    } else {
      const int by = N - n;  // elements
      u32x4 t = *reinterpret_cast<const u32x4u*>(p - by);
      const int words = by * (int)sizeof(T) / 4;
      if (words & 2) t = u32x4{t[2], t[3], 0, 0};
      if (words & 1) t = u32x4{t[1], t[2], t[3], 0};
      if (N == 8 && (by & 1)) t = u32x4{t[0] >> 16 | t[1] << 16, t[1] >> 16 | t[2] << 16, t[2] >> 16 | t[3] << 16, t[3] >> 16};
      w = t;
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (N == 4) return __uint_as_float(w[e]);
    return __uint_as_float(e % 2 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
  }
  __device__ __forceinline__ void fill_one() {
    const uint32_t one = N == 4 ? 0x3F800000u : 0x3F803F80u;
    w = u32x4{one, one, one, one};
  }
};
// The same as float32.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
  template <bool RAGGED>
  __device__ __forceinline__ void from(const Raw<T, RAGGED>& r, int n) {  // the first n, then zeros
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = r.get(e);
    if (RAGGED && n < N) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = e < n ? v[e] : 0.0f;
    }
  }
  template <bool RAGGED>
  __device__ __forceinline__ void store(T* p, int n) const {
    if constexpr (N == 8) {
      if (!RAGGED || n >= 8) {
        store8(p, f32x8{{v[0], v[1], v[2], v[3]}, {v[4], v[5], v[6], v[7]}});
        return;
      }
      if (n >= 4) store4(p, f32x4{v[0], v[1], v[2], v[3]});
    } else if (!RAGGED || n >= 4) {
      store4(p, f32x4{v[0], v[1], v[2], v[3]});
      return;
    }
    const bool high = N == 8 && n >= 4;
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      float x = v[e];
      if constexpr (N == 8) {
        const float y = v[4 + e];
        x = high ? y : x;
      }
      if (e < (n & 3)) p[(n & ~3) + e] = (T)x;
    }
  }
};

// How a row lies on the lanes: LPR lanes of one wave (16 or 64) or WAVES whole waves, V 16-byte vectors a lane, all of
// it in registers.  A workgroup of kThreads threads holds kRows rows at a time.
template <int LPR, int WAVES, int V>
struct Shape {
  static constexpr int lanes = LPR * WAVES, vecs = V;
  static constexpr int threads = WAVES == 1 ? 256 : WAVES * kWave, rows = threads / lanes;
  static_assert(WAVES == 1 || LPR == kWave, "whole waves");
  __device__ static int row_of() { return threadIdx.x / lanes; }
  __device__ static int lane_of() { return threadIdx.x % lanes; }
  template <class T>
  __device__ static int col(int k) { return (k * lanes + lane_of()) * Vec<T>::N; }
  template <class T, bool R>  // a row of `dim` at p, `left` elements from the array's end
  __device__ static __forceinline__ void load(Raw<T, R> (&a)[V], const T* p, int dim, int64_t left) {
    constexpr bool kTiny = LPR == 16 && V == 1;
    const bool next_row = left > dim;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = col<T>(k);
      a[k].template load<kTiny>(p + c, dim - c, kTiny ? left - c >= Vec<T>::N : next_row);
    }
  }
  // Sums of N values over the row's lanes, the same bits in all of them.  Across waves through `lds` [2][WAVES][N],
  // `turn` naming the half that the last call did not use: one barrier a call is then enough.
  template <int N>
  __device__ static __forceinline__ void sum(float (&x)[N], float* lds, int turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = lanes_sum<LPR>(x[i]);
    if constexpr (WAVES > 1) {
      float* at = lds + turn * WAVES * N;
      if (lane_id() == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) at[(threadIdx.x >> 6) * N + i] = x[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[i] = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) x[i] += at[w * N + i];
      }
    }
  }
};

// A row a row's lanes, no loop: many light workgroups keep more loads in flight than fewer that hold gain and offset.
template <class T, class S, bool R>
__global__ __launch_bounds__(S::threads) void norm_kernel(const T* x, const T* gamma, const T* beta, int64_t rows, int dim,
                                                          float eps, T* y, float* mean, float* rstd) {
  __shared__ float lds[2 * (S::lanes + kWave - 1) / kWave];
  constexpr int V = S::vecs, N = Vec<T>::N;
  const int64_t r = (int64_t)blockIdx.x * S::rows + S::row_of();
  if (r >= rows) return;  // a row's lanes leave together
  Raw<T, R> in[V], g[V], b[V];
  S::load(in, x + r * dim, dim, (rows - r) * dim);
  if (gamma) S::load(g, gamma, dim, dim);
  if (beta) S::load(b, beta, dim, dim);
  Vec<T> a[V];
  float s[1] = {0};
#pragma unroll
  for (int k = 0; k < V; ++k) {
    a[k].from(in[k], dim - S::template col<T>(k));
#pragma unroll
    for (int e = 0; e < N; ++e) s[0] += a[k].v[e];
  }
  S::sum(s, lds, 0);
  const float mu = s[0] / (float)dim;
  s[0] = 0;
#pragma unroll
  for (int k = 0; k < V; ++k)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = S::template col<T>(k) + e < dim ? a[k].v[e] - mu : 0.0f;
      a[k].v[e] = d;
      s[0] = fmaf(d, d, s[0]);
    }
  S::sum(s, lds, 1);
  const float rs = 1.0f / sqrtf(s[0] / (float)dim + eps);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = S::template col<T>(k), n = dim - c;
    if (n <= 0) continue;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float o = a[k].v[e] * rs;
      if (gamma) o *= g[k].get(e);
      if (beta) o += b[k].get(e);
      a[k].v[e] = o;
    }
    a[k].template store<R>(y + r * dim + c, n);
  }
  if (S::lane_of() == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

// A workgroup walks its rows blockIdx.x S::rows + row, + gridDim.x S::rows, ..., the next row's loads in flight while
// this one is worked on, keeps the two column sums in registers and joins its rows' at the end: part [workgroup][2][dim].
template <class T, class S, bool R>
__global__ __launch_bounds__(S::threads) void norm_backward_kernel(const T* dy, const T* x, const T* gamma,
                                                                   const float* mean, const float* rstd, int64_t rows,
                                                                   int dim, T* dx, float* part) {
  // With 16 waves a lane has 128 registers: too few for 16 elements' next row.
  constexpr bool kAhead = S::lanes <= 256 || S::vecs * Vec<T>::N < 16;
  constexpr int V = S::vecs, N = Vec<T>::N, kHeld = S::rows > 1 ? S::lanes * V * N : 1;
  __shared__ float lds[4 * (S::lanes + kWave - 1) / kWave];
  __shared__ float held[S::rows > 1 ? S::rows : 1][kHeld];
  const int64_t step = (int64_t)gridDim.x * S::rows;
  float sg[V][N], sb[V][N];
  Raw<T, R> ga[V];
  if (gamma) S::load(ga, gamma, dim, dim);
#pragma unroll
  for (int k = 0; k < V; ++k) {
    if (!gamma) ga[k].fill_one();
#pragma unroll
    for (int e = 0; e < N; ++e) sg[k][e] = sb[k][e] = 0;
  }
  int64_t r = (int64_t)blockIdx.x * S::rows + S::row_of();
  Vec<T> a[V], d[V];
  Raw<T, R> an[V], dn[V];
  float mu = 0, rs = 0, mun = 0, rsn = 0;
  auto fetch = [&](int64_t row) {
    S::load(an, x + row * dim, dim, (rows - row) * dim);
    S::load(dn, dy + row * dim, dim, (rows - row) * dim);
    mun = mean[row], rsn = rstd[row];
  };
  if (kAhead && r < rows) fetch(r);
  int turn = 0;
  while (r < rows) {
    if (!kAhead) fetch(r);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int n = dim - S::template col<T>(k);
      a[k].from(an[k], n), d[k].from(dn[k], n);
    }
    mu = mun, rs = rsn;
    const int64_t next = r + step;
    if (kAhead && next < rows) fetch(next);
    float s[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float h = (a[k].v[e] - mu) * rs, g = d[k].v[e];
        sg[k][e] = fmaf(g, h, sg[k][e]);  // columns beyond dim have dy = 0
        sb[k][e] += g;
        a[k].v[e] = h;
        d[k].v[e] = g * ga[k].get(e);
        s[0] += d[k].v[e];
        s[1] = fmaf(d[k].v[e], h, s[1]);
      }
    if (dx) {
      S::sum(s, lds, turn);
      turn ^= 1;
      const float m1 = s[0] / (float)dim, m2 = s[1] / (float)dim;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = S::template col<T>(k), n = dim - c;
        if (n <= 0) continue;
#pragma unroll
        for (int e = 0; e < N; ++e) d[k].v[e] = (d[k].v[e] - m1 - a[k].v[e] * m2) * rs;
        d[k].template store<R>(dx + r * dim + c, n);
      }
    }
    r = next;
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    if constexpr (S::rows > 1) {
      if (q) __syncthreads();
#pragma unroll
      for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e) held[S::row_of()][S::template col<T>(k) + e] = q ? sb[k][e] : sg[k][e];
      __syncthreads();
      for (int c = threadIdx.x; c < dim; c += S::threads) {
        float v = 0;
#pragma unroll
        for (int w = 0; w < S::rows; ++w) v += held[w][c];
        out[q * dim + c] = v;
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (S::template col<T>(k) + e < dim) out[q * dim + S::template col<T>(k) + e] = q ? sb[k][e] : sg[k][e];
    }
  }
}

// Calls f with the shape a row of `dim` takes: 16 lanes up to two vectors a lane, then a wave up to 1024 dims, 4 waves up to
// 4096, 16 beyond; at most 16 elements a lane, so the backward pass's sums, gains and two rows in flight fit the
// registers of two workgroups a CU or more.
template <class T, class F>
fgpu_status by_dim(int dim, F&& f) {
  constexpr int E = 16 / Vec<T>::N;  // vectors that hold 16 elements
  if (dim <= 16 * Vec<T>::N) return f(Shape<16, 1, 1>{});
  if (dim <= 32 * Vec<T>::N) return f(Shape<16, 1, 2>{});
  if (dim <= 64 * Vec<T>::N) return f(Shape<64, 1, 1>{});
  if (dim <= 512) return f(Shape<64, 1, 512 / 64 / Vec<T>::N>{});
  if (dim <= 1024) return f(Shape<64, 1, E>{});
  if (dim <= 2048) return f(Shape<64, 4, E / 2>{});
  if (dim <= 4096) return f(Shape<64, 4, E>{});
  if (dim <= 8192) return f(Shape<64, 16, E / 2>{});
  return f(Shape<64, 16, E>{});
}

// Workgroups of the backward pass: at most two a CU of the 256 threads' shapes (each leaves a part of the column sums),
// one of the 16 waves'.
constexpr int kNormParts = 512;
int norm_groups(int64_t rows, int shape_rows) { return (int)std::min<int64_t>(ceil_div(rows, shape_rows), kNormParts); }

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
  auto run = [&](auto type) -> fgpu_status {
    using T = decltype(type);
    return by_dim<T>(dim, [&](auto shape) -> fgpu_status {
      using S = decltype(shape);
      const auto k = dim % Vec<T>::N ? norm_kernel<T, S, true> : norm_kernel<T, S, false>;
      constexpr int64_t kMost = kLaunchThreads / S::threads * S::rows;
      for (int64_t r0 = 0; r0 < rows; r0 += kMost) {
        const int64_t n = std::min(rows - r0, kMost);
        k<<<ceil_div(n, S::rows), S::threads, 0, as_stream(stream)>>>((const T*)d_x + r0 * dim, (const T*)d_gamma,
                                                                     (const T*)d_beta, n, dim, eps, (T*)d_y + r0 * dim,
                                                                     d_mean ? d_mean + r0 : nullptr,
                                                                     d_rstd ? d_rstd + r0 : nullptr);
        FGPU_HIP(hipGetLastError());
      }
      return FGPU_OK;
    });
  };
  return dtype == FGPU_DTYPE_F32 ? run(float{}) : run(bf16{});
}

size_t fgpu_layer_norm_backward_workspace_bytes(int64_t rows, int dim, int dtype) {
  if (check_norm(rows, dim, dtype) != FGPU_OK || rows == 0) return 0;
  return carve_bytes<float>((size_t)std::min<int64_t>(rows, kNormParts) * 2 * dim);
}

fgpu_status fgpu_layer_norm_backward(const void* d_dy, const void* d_x, const void* d_gamma, const float* d_mean,
                                     const float* d_rstd, int64_t rows, int dim, int dtype, void* d_dx, void* d_dgamma,
                                     void* d_dbeta, void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_norm(rows, dim, dtype));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  if (rows == 0) {
    if (d_dgamma) FGPU_TRY(launch_zeros(dim, f32, d_dgamma, s));
    if (d_dbeta) FGPU_TRY(launch_zeros(dim, f32, d_dbeta, s));
    return FGPU_OK;
  }
  FGPU_CHECK(d_dy && d_x && d_mean && d_rstd, FGPU_ERR_ARG, "layer norm backward: null dy, x, mean or rstd");
  float* part = nullptr;
  if (d_dgamma || d_dbeta) {
    Carve ws(d_workspace, workspace_bytes);
    part = ws.take<float>((size_t)std::min<int64_t>(rows, kNormParts) * 2 * dim);
    FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE,
               "layer norm backward: workspace smaller than fgpu_layer_norm_backward_workspace_bytes");
  }
  int groups = 0;
  auto run = [&](auto type) -> fgpu_status {
    using T = decltype(type);
    return by_dim<T>(dim, [&](auto shape) -> fgpu_status {
      using S = decltype(shape);
      groups = norm_groups(rows, S::rows);
      const auto k = dim % Vec<T>::N ? norm_backward_kernel<T, S, true> : norm_backward_kernel<T, S, false>;
      k<<<groups, S::threads, 0, s>>>((const T*)d_dy, (const T*)d_x, (const T*)d_gamma, d_mean, d_rstd, rows, dim, (T*)d_dx,
                                      part);
      FGPU_HIP(hipGetLastError());
      return FGPU_OK;
    });
  };
  FGPU_TRY(f32 ? run(float{}) : run(bf16{}));
  if (part) {
    ColumnSum c;
    c.part = part, c.parts = groups, c.stride = 2 * dim, c.cols = dim, c.out = d_dgamma, c.f32 = f32;
    FGPU_TRY(launch_column_sums(c, d_dbeta, s));
  }
  return FGPU_OK;
}

}  // extern "C"

// head_ortho.hip -- an update with its singular values drawn to one, by Newton-Schulz products.
//
// X_0 = x / (|x| + eps) in the Frobenius norm; each step forms the products of the shorter side, A = X X^T (or X^T X),
// P = b A + c A^2, and X <- a X + P X (or X P): every singular value s becomes a s + b s^3 + c s^5, the vectors stay.
//
// Between the products X, A and P are held as two float16 planes, 2^10 times their value: h + l is good to 2^-23 of what
// lies above 2^-25 of one, and all of them stay below 2^6 while the singular values stay below about two.  The steps
// multiply a small singular value by up to a each, and with it whatever a rounding leaves in its directions, so X may not
// be rounded to one plane of 8 or 11 bits between them.
#include <algorithm>
#include <cmath>

#include "gated.hpp"

namespace fgpu {
namespace {

constexpr float kHeld = 1024.0f;  // what planes hold of a value of one
constexpr int kNormBlocks = 512;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Two planes of a matrix: rows of ld, a multiple of 8; columns from n to the next multiple of 8 hold zeros.
struct Planes {
  uint16_t* p = nullptr;
  int64_t ld = 0, plane = 0;
};
__device__ __forceinline__ f32x8 planes8(const Planes& a, int64_t at) {
  const f16x8 h = *reinterpret_cast<const f16x8*>(a.p + at), l = *reinterpret_cast<const f16x8*>(a.p + a.plane + at);
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v.set(e, (float)h[e] + (float)l[e]);
  return v;
}
__device__ __forceinline__ void put_planes8(const Planes& a, int64_t at, const f32x8& v) {
  f16x8 h, l;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = (_Float16)v[e];
    l[e] = (_Float16)(v[e] - (float)h[e]);
  }
  *reinterpret_cast<f16x8*>(a.p + at) = h;
  *reinterpret_cast<f16x8*>(a.p + a.plane + at) = l;
}

// ---- the start: the norm, and X_0 ----------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void norm_parts_kernel(const T* x, int64_t count, double* part) {
  __shared__ double sum[256];
  double v = 0;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < count; i += (int64_t)gridDim.x * 256 * 8) {
    const f32x8 q = load8_n(x + i, (int)min(count - i, (int64_t)8));
#pragma unroll
    for (int e = 0; e < 8; ++e) v += (double)q[e] * q[e];
  }
  sum[threadIdx.x] = v;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if ((int)threadIdx.x < h) sum[threadIdx.x] += sum[threadIdx.x + h];
    __syncthreads();
  }
  if (threadIdx.x == 0) part[blockIdx.x] = sum[0];
}

template <class T>
__global__ __launch_bounds__(256) void start_kernel(const T* x, int64_t rows, int cols, const double* part, int parts, float eps,
                                                    Planes out) {
  __shared__ double sum[256];
  double v = 0;
  for (int i = threadIdx.x; i < parts; i += 256) v += part[i];
  sum[threadIdx.x] = v;
  __syncthreads();
  for (int h = 128; h > 0; h >>= 1) {
    if ((int)threadIdx.x < h) sum[threadIdx.x] += sum[threadIdx.x + h];
    __syncthreads();
  }
  const double norm = sqrt(sum[0]) + eps;
  // Something not finite makes everything NaN; nothing but zeros stays zero.
  const double by = !(norm < INFINITY) ? (double)NAN : norm > 0 ? kHeld / norm : 0;
  const int64_t per = whole8(cols) / 8, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8;
    const f32x8 q = load8_n(x + r * cols + c, cols - c);
    f32x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.set(e, c + e < cols ? (float)(q[e] * by) : 0.0f);
    put_planes8(out, r * out.ld + c, o);
  }
}

// ---- the products ------------------------------------------------------------------
// alpha D + beta C, as planes or (out) as the result.
struct OrthoFinish {
  float alpha = 0, beta = 0;
  Planes c, to;
  void* out = nullptr;
  int m = 0, n = 0;
  template <class T>
  __device__ __forceinline__ void put(f32x8 v, int64_t row, int col) const {
    v.lo *= alpha, v.hi *= alpha;
    if (c.p) {
      const f32x8 o = planes8(c, row * c.ld + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) v.set(e, fmaf(beta, o[e], v[e]));
    }
    if (out) store8_n<false>((T*)out + row * n + col, v, n - col);
    else put_planes8(to, row * to.ld + col, v);
  }
};
template <class T>
struct OrthoEpi {
  OrthoFinish f;
  float* part;  // [split][m][n8]: the product alone, to be joined; or NULL

  template <class G>
  struct Side {
    __device__ void fetch(const OrthoEpi&, int, int, int) {}
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
    const int n8 = (f.n + 7) & ~7;
#pragma unroll
    for (int p = 0; p < G::FN / 2; ++p) {
      const int col = w.col(p);
      if (col >= n8) continue;
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        const int64_t row = w.row(j);
        if (row >= f.m) continue;
        if (part) {
          float* d = part + ((int64_t)w.sp * f.m + row) * n8 + col;
          *reinterpret_cast<f32x4*>(d) = acc[2 * p][j];
          *reinterpret_cast<f32x4*>(d + 4) = acc[2 * p + 1][j];
        } else {
          f.put<T>(f32x8{acc[2 * p][j], acc[2 * p + 1][j]}, row, col);
        }
      }
    }
  }
};
// The parts of a split product added in their order, eight columns a thread.
template <class T>
__global__ __launch_bounds__(256) void ortho_join_kernel(OrthoFinish f, const float* part, int splits) {
  const int n8 = (f.n + 7) & ~7, per = n8 / 8;
  const int64_t total = (int64_t)f.m * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    f32x8 v{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const f32x8 q = load8(part + ((int64_t)s * total + i) * 8);
      v.lo += q.lo, v.hi += q.hi;
    }
    const int64_t row = i / per;
    f.put<T>(v, row, (int)(i - row * per) * 8);
  }
}

constexpr int kPairs = 3;
Plan plan_ortho(int m, int n, int k) {
  Product p{m, n, k, false};
  p.pairs = kPairs;
  return plan_product(p, true);
}
size_t ortho_part_bytes(int m, int n, const Plan& q) {
  return q.splits > 1 ? carve_bytes<float>((size_t)q.splits * m * ((n + 7) & ~7)) : 0;
}

template <class T, bool AKC, bool BKC>
fgpu_status ortho_product(const Planes& a, const Planes& b, int k, const OrthoFinish& f, float* part, hipStream_t s) {
  const Plan q = plan_ortho(f.m, f.n, k);
  FGPU_CHECK(q.tile, FGPU_ERR_UNSUPPORTED, "orthogonalize: more tiles than one launch takes");
  const GemmArgs g{{a.p, a.ld, a.plane}, {b.p, b.ld, b.plane}, f.m, f.n, k, q.tiles_m, q.tiles_n, q.splits, q.k_per_split};
  const OrthoEpi<T> e{f, q.splits > 1 ? part : nullptr};
  const int grid = q.tiles_m * q.tiles_n * q.splits;
  if (q.tile == 256) gemm_kernel<Tile256, AKC, BKC, kPairs, OrthoEpi<T>, OfHalf><<<grid, Tile256::threads, 0, s>>>(g, e);
  else if (q.tile == 128) gemm_kernel<Tile128, AKC, BKC, kPairs, OrthoEpi<T>, OfHalf><<<grid, Tile128::threads, 0, s>>>(g, e);
  else gemm_kernel<Tile64, AKC, BKC, kPairs, OrthoEpi<T>, OfHalf><<<grid, Tile64::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  if (q.splits > 1) {
    const int blocks = (int)std::min<int64_t>(((int64_t)f.m * ((f.n + 7) / 8) + 255) / 256, 256 * 16);
    ortho_join_kernel<T><<<blocks, 256, 0, s>>>(f, part, q.splits);
    FGPU_HIP(hipGetLastError());
  }
  return FGPU_OK;
}

struct Shape {
  int rows, cols, small, large;
  bool tall;
  Shape(int r, int c) : rows(r), cols(c), small(std::min(r, c)), large(std::max(r, c)), tall(r > c) {}
  size_t x_bytes() const { return carve_bytes<uint16_t>((size_t)rows * packed_ld(cols) * 2); }
  size_t a_bytes() const { return carve_bytes<uint16_t>((size_t)small * packed_ld(small) * 2); }
  size_t part_bytes() const {
    const int m = tall ? rows : small, n = tall ? small : cols;
    return std::max({ortho_part_bytes(small, small, plan_ortho(small, small, large)),
                     ortho_part_bytes(small, small, plan_ortho(small, small, small)),
                     ortho_part_bytes(m, n, plan_ortho(m, n, small))});
  }
};
Planes planes_at(void* p, int rows, int cols) { return {(uint16_t*)p, packed_ld(cols), rows * packed_ld(cols)}; }

fgpu_status check_common(int64_t rows, int64_t cols, int dtype) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "orthogonalize: unknown dtype");
  FGPU_CHECK(rows >= 0 && cols >= 0, FGPU_ERR_ARG, "orthogonalize: rows and cols >= 0");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_DIM && cols <= FGPU_HEAD_MAX_DIM, FGPU_ERR_UNSUPPORTED, "orthogonalize: more than 2^16 rows or columns");
  return FGPU_OK;
}

template <class T>
fgpu_status run_ortho(const T* x, const Shape& sh, int steps, float a, float b, float c, float eps, T* out, Carve& ws,
                      hipStream_t s) {
  Planes xs[2] = {planes_at(ws.take<char>(sh.x_bytes()), sh.rows, sh.cols), planes_at(ws.take<char>(sh.x_bytes()), sh.rows, sh.cols)};
  const Planes ga = planes_at(ws.take<char>(sh.a_bytes()), sh.small, sh.small);
  const Planes gp = planes_at(ws.take<char>(sh.a_bytes()), sh.small, sh.small);
  float* part = (float*)ws.take<char>(sh.part_bytes());
  double* norm = ws.take<double>(kNormBlocks);
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "orthogonalize: workspace smaller than fgpu_orthogonalize_workspace_bytes");
  const int64_t count = (int64_t)sh.rows * sh.cols;
  const int blocks = (int)std::min<int64_t>((count + 2047) / 2048, kNormBlocks);
  norm_parts_kernel<T><<<blocks, 256, 0, s>>>(x, count, norm);
  start_kernel<T><<<(int)std::min<int64_t>((sh.rows * (whole8(sh.cols) / 8) + 255) / 256, 4096), 256, 0, s>>>(
      x, sh.rows, sh.cols, norm, blocks, eps, xs[0]);
  FGPU_HIP(hipGetLastError());
  const int n = sh.small;
  for (int i = 0; i < steps; ++i) {
    const Planes &from = xs[i & 1], &to = xs[i + 1 & 1];
    const bool last = i + 1 == steps;
    OrthoFinish fa, fp, fx;
    fa.alpha = 1 / kHeld, fa.to = ga, fa.m = fa.n = n;
    fp.alpha = c / kHeld, fp.beta = b, fp.c = ga, fp.to = gp, fp.m = fp.n = n;
    fx.alpha = 1 / kHeld, fx.beta = a, fx.c = from, fx.to = to, fx.m = sh.rows, fx.n = sh.cols;
    if (last) fx.out = out, fx.alpha /= kHeld, fx.beta /= kHeld;
    if (sh.tall) {
      FGPU_TRY((ortho_product<T, false, false>(from, from, sh.large, fa, part, s)));
      FGPU_TRY((ortho_product<T, true, true>(ga, ga, n, fp, part, s)));
      FGPU_TRY((ortho_product<T, true, true>(from, gp, n, fx, part, s)));
    } else {
      FGPU_TRY((ortho_product<T, true, true>(from, from, sh.large, fa, part, s)));
      FGPU_TRY((ortho_product<T, true, true>(ga, ga, n, fp, part, s)));
      FGPU_TRY((ortho_product<T, true, false>(gp, from, n, fx, part, s)));
    }
  }
  return FGPU_OK;
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

size_t fgpu_orthogonalize_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
  if (check_common(rows, cols, dtype) != FGPU_OK || rows == 0 || cols == 0) return 0;
  const Shape sh((int)rows, (int)cols);
  return 2 * (sh.x_bytes() + sh.a_bytes()) + sh.part_bytes() + carve_bytes<double>(kNormBlocks);
}

fgpu_status fgpu_orthogonalize(const void* d_x, int64_t rows, int64_t cols, int dtype, int steps, float a, float b, float c,
                               float eps, void* d_y, void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, cols, dtype));
  FGPU_CHECK(steps >= 1 && steps <= FGPU_ORTHO_MAX_STEPS, FGPU_ERR_ARG, "orthogonalize: 1 to 64 steps");
  FGPU_CHECK(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), FGPU_ERR_ARG, "orthogonalize: coefficients must be finite");
  FGPU_CHECK(eps >= 0 && std::isfinite(eps), FGPU_ERR_ARG, "orthogonalize: eps >= 0");
  if (rows == 0 || cols == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_y, FGPU_ERR_ARG, "orthogonalize: null input or output");
  FGPU_CHECK(aligned16(d_workspace), FGPU_ERR_ARG, "orthogonalize: the workspace must be 16-byte aligned");
  const Shape sh((int)rows, (int)cols);
  Carve ws(d_workspace, workspace_bytes);
  hipStream_t s = as_stream(stream);
  if (dtype == FGPU_DTYPE_F32) return run_ortho((const float*)d_x, sh, steps, a, b, c, eps, (float*)d_y, ws, s);
  return run_ortho((const bf16*)d_x, sh, steps, a, b, c, eps, (bf16*)d_y, ws, s);
}

}  // extern "C"

// head_direct.hip -- products of few tiles: fragments straight from the caller's arrays, k split over a workgroup's waves.
//
// Where a product has too few 64 x 64 tiles to fill the GPU, what counts is how soon the first bytes arrive and how many
// launches follow one another, not the rate of the matrix units.  Here eight waves share a 32 x 32 (or 16 x 16) tile, each
// with an eighth of k: a wave loads its fragments from global memory as they lie (any stride and alignment, no packed
// copy; float32 is split into its bf16 triple in registers, dz is formed from dy and the kept pre-activation as it is
// read), the partial tiles meet in LDS, and the epilogue is the product's own: one launch a product, or one for both
// gradients and a column sum.
//
// Bound by latency: one row x 1024 x 1024 in bf16 takes 4.6 us on the GPU, of which its 2 MB of weights are 0.4 at the
// rate of a copy and a launch 2: 64 workgroups, four k steps a wave, which it loads two at a time, so it waits for two rounds
// of loads and for the join; 128 x 768 x 2048 6.7 us (tiled 7.3 with the caches warm); float32 400 x 256 x 256 6.9 us
// (tiled, with its two copies, 12).  Beyond a few rounds of tiles the fragments' loads from the caches bound it (each
// element is read once a 32-wide tile) and the tiled products take over: head_linear.hip has the rule and both sides.
#include <algorithm>

#include "head_direct.hpp"

namespace fgpu {
namespace {

template <class T, int FM, int FN>
__global__ __launch_bounds__(kDirectThreads) void direct_forward_kernel(DirectJob j) {
  __shared__ __attribute__((aligned(1024))) char lds[direct_lds<T, FM, FN>(true, true)];
  direct_tile<T, FM, FN, true, true, false>(j, blockIdx.x, lds);
}

template <class T, int FM, int FN>
__global__ __launch_bounds__(kDirectThreads) void direct_gated_kernel(DirectJob j) {
  __shared__ __attribute__((aligned(1024))) char lds[direct_lds<T, FM, FN>(true, true)];
  direct_tile<T, FM, FN, true, true, false, true>(j, blockIdx.x, lds);
}

// The tiles of `x` (k contiguous x strided: an input's gradient), then those of `w` (both strided: a weight's, with the
// column sums of its first operand).
template <class T, bool DZ>
__global__ __launch_bounds__(kDirectThreads) void direct_backward_kernel(DirectJob x, int x_tiles, DirectJob w) {
  __shared__ __attribute__((aligned(1024))) char lds[direct_lds<T, 2, 2>(false, false)];
  const int b = blockIdx.x;
  if (b < x_tiles)
    direct_tile<T, 2, 2, true, false, DZ>(x, b, lds);
  else
    direct_tile<T, 2, 2, false, false, DZ>(w, b - x_tiles, lds);
}

int tiles_of(const DirectJob& j, int fm, int fn) { return ceil_div(j.m, 16 * fm) * ceil_div(j.n, 16 * fn); }

}  // namespace

fgpu_status launch_direct_forward(const DirectJob& j, bool f32, hipStream_t s) {
  const bool thin = j.m <= 16;
  const int grid = tiles_of(j, thin ? 1 : 2, thin ? 1 : 2);
  if (f32)
    thin ? direct_forward_kernel<float, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_forward_kernel<float, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  else
    thin ? direct_forward_kernel<bf16, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_forward_kernel<bf16, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_direct_gated(const DirectJob& j, bool f32, hipStream_t s) {
  const bool thin = j.m <= 16;
  const int grid = ceil_div(j.m, thin ? 16 : 32) * ceil_div(j.n, thin ? 8 : 16);
  if (f32)
    thin ? direct_gated_kernel<float, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_gated_kernel<float, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  else
    thin ? direct_gated_kernel<bf16, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_gated_kernel<bf16, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_direct_backward(const DirectJob* x, const DirectJob* w, bool f32, hipStream_t s) {
  const DirectJob none{};
  const int xt = x ? tiles_of(*x, 2, 2) : 0, wt = w ? tiles_of(*w, 2, 2) : 0;
  if (xt + wt == 0) return FGPU_OK;
  const bool dz = (x && x->a.pre) || (w && w->a.pre);
  const auto k = f32 ? (dz ? direct_backward_kernel<float, true> : direct_backward_kernel<float, false>)
                     : (dz ? direct_backward_kernel<bf16, true> : direct_backward_kernel<bf16, false>);
  k<<<xt + wt, kDirectThreads, 0, s>>>(x ? *x : none, xt, w ? *w : none);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

// Microseconds, fitted over 1 to 16384 rows and 64 to 2048 dims: a start, the k steps (32) of a wave one after the other,
// and all tiles' steps at what 256 CUs take for one each.
namespace {
int wave_steps(int64_t k) { return ceil_div(ceil_div(k, 32), kDirectWaves); }
double tile_steps(int64_t m, int64_t n, int64_t k) { return (double)ceil_div(m, 32) * ceil_div(n, 32) * wave_steps(k) / 256; }
}  // namespace
double direct_forward_estimate_us(const Product& p) {
  if (p.m <= 16) return p.f32 ? 7.5 : 4.5;
  // Rows that are not whole 16-byte groups load at half the rate or less.
  const double ragged = p.k % 8 == 0 ? 1 : p.f32 ? 1.2 : 2.4;
  return 3 + std::max<double>(wave_steps(p.k), tile_steps(p.m, p.n, p.k)) * (p.f32 ? 2.2 : 0.95) * ragged;
}
double direct_backward_estimate_us(int rows, int in_dim, int out_dim, bool f32) {
  const int longest = std::max(wave_steps(out_dim), wave_steps(rows));
  const double all = tile_steps(rows, in_dim, out_dim) + tile_steps(out_dim, in_dim, rows);
  const double ragged = in_dim % 8 || out_dim % 8 ? 1.3 : 1;
  return f32 ? 2 + (1.8 * longest + 2.2 * all) * ragged : 2.5 + (1.0 * longest + 0.6 * all) * ragged;
}

}  // namespace fgpu

// head_prep.hip -- what the products of the query head's operators need first, in one launch: operands copied where their
// rows cannot be read as they are, dz with its column sums, the rows of the contrastive loss's backward pass.
//
// Bound by HBM: dz of 16384 x 4096 in bf16 (two arrays read, one written) takes 82 us, 4.9 TB/s.  It is formed once rather
// than in both gradients' products, which read it in two orders and as many times as they have tiles beside it.
//
// In bf16 it is rounded to bf16 there, as the next layer's own gradient will be (the bias's sum takes it unrounded).  The
// gradients are then 0.0024 of their norm off the exact ones (16384 x 1024 x 4096, GELU), of which the rounding of the
// results is 0.0017; a second operand with what the first rounding leaves would double both products.
#include <algorithm>

#include "head.hpp"

namespace fgpu {
namespace {

// Four elements of an operand's row: bf16, or the three planes of float32.
template <class T>
__device__ __forceinline__ void put4(uint16_t* d, int64_t plane, const f32x4& v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<bf16x4*>(d) = __builtin_convertvector(v, bf16x4);
  } else {
    bf16x4 h, m, l;
    split4(v, h, m, l);
    *reinterpret_cast<bf16x4*>(d) = h;
    *reinterpret_cast<bf16x4*>(d + plane) = m;
    *reinterpret_cast<bf16x4*>(d + 2 * plane) = l;
  }
}

__device__ __forceinline__ bool loss_row_live(const LossRows& r, int m) {
  const int t = r.target[m];
  if ((uint32_t)t >= (uint32_t)r.nc || r.lse[m] == -INFINITY) return false;
  return !(r.bias && r.bias[t] <= FGPU_MASK_BIAS);
}

// One thread four columns of a row, the workgroups of the job in turn.
template <class T>
__device__ __forceinline__ void copy_rows(const CopyJob& j, const LossRows& loss, int block, int blocks) {
  uint16_t* dst = const_cast<uint16_t*>(j.dst.p);
  const int64_t per = whole8(j.cols) / 4, total = j.rows * per;
  for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)blocks * 256) {
    const int64_t r = i / per, c = (i - r * per) * 4;
    f32x4 v = {0, 0, 0, 0};
    const bool zero = (j.row_bias && j.row_bias[r] <= FGPU_MASK_BIAS) || (j.loss_rows && !loss_row_live(loss, (int)r));
    if (c < j.cols && !zero) v = load4_n((const T*)j.src + r * j.cols + c, (int)min(j.cols - c, (int64_t)4));
    put4<T>(dst + r * j.dst.ld + c, j.dst.plane, v);
  }
}

constexpr int kDzCols = 256;  // columns of a workgroup: 64 lanes x 4; its four waves take rows in turn

template <class T>
__device__ __forceinline__ void make_dz(const DzJob& j, int block) {
  __shared__ f32x4 sum[4][64];
  const int64_t width = j.dst.p ? whole8(j.cols) : j.cols;
  const int across = (int)((width + kDzCols - 1) / kDzCols), chunk = block / across;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = block % across * kDzCols + lane * 4, cnt = min(j.cols - c, 4);
  const int per = (j.rows + j.chunks - 1) / j.chunks, r0 = chunk * per, r1 = min(j.rows, r0 + per);
  uint16_t* dst = const_cast<uint16_t*>(j.dst.p);
  f32x4 acc = {0, 0, 0, 0};
  if (c < width) {
#pragma unroll 2
    for (int r = r0 + w; r < r1; r += 4) {
      f32x4 v = {0, 0, 0, 0};
      if (cnt > 0) {
        v = load4_n((const T*)j.dy + (int64_t)r * j.cols + c, cnt);
        if (j.act != FGPU_ACT_NONE) {
          const f32x4 z = load4_n((const T*)j.pre + (int64_t)r * j.cols + c, cnt);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= act_slope<T>(z[k], j.act);
        }
      }
      acc += v;
      if (dst) put4<T>(dst + (int64_t)r * j.dst.ld + c, j.dst.plane, v);
    }
  }
  if (!j.part) return;
  sum[w][lane] = acc;
  __syncthreads();
  if (w == 0 && cnt > 0) {
    for (int k = 1; k < 4; ++k) acc += sum[k][lane];
    for (int k = 0; k < min(cnt, 4); ++k) j.part[(int64_t)chunk * j.cols + c + k] = acc[k];
  }
}

__device__ __forceinline__ void loss_row(const LossRows& r, int m) {
  if (m >= r.nq) return;
  LossRow o{INFINITY, 0.0f, -1, 0};
  if (loss_row_live(r, m)) {
    const int t = r.target[m];
    // lse comes in natural units: the two conversions put up to |lse| 2^-23 on the exponents, as the scores' own roundings do
    o = {r.lse[m] * kLog2e, r.dloss[m], t, r.ids ? r.ids[t] : 0};
  }
  r.rows[m] = o;
  if (r.left) r.left[m] = 0;
}
__device__ __forceinline__ void clear_candidates(const LossRows& r, int block, int blocks) {
  for (int64_t c = (int64_t)block * 256 + threadIdx.x; c < r.nc; c += (int64_t)blocks * 256) r.owner[c] = INT_MAX;
}

struct Blocks {
  int dz, copy0, copy1, loss, clear;
};
template <class T>
__global__ __launch_bounds__(256) void prep_kernel(Prep p, Blocks n) {
  int b = blockIdx.x;
  if (b < n.dz)
    make_dz<T>(p.dz, b);
  else if ((b -= n.dz) < n.copy0)
    copy_rows<T>(p.copy[0], p.loss, b, n.copy0);
  else if ((b -= n.copy0) < n.copy1)
    copy_rows<T>(p.copy[1], p.loss, b, n.copy1);
  else if ((b -= n.copy1) < n.loss)
    loss_row(p.loss, b * 256 + threadIdx.x);
  else
    clear_candidates(p.loss, b - n.loss, n.clear);
}

}  // namespace

int dz_chunks(int rows, int cols) {
  const int per = std::max(16, ceil_div((int64_t)rows * ceil_div(cols, kDzCols), 2048));
  return ceil_div(rows, (per + 3) / 4 * 4);
}

fgpu_status launch_prep(const Prep& p, bool f32, hipStream_t s) {
  auto copy_blocks = [](const CopyJob& j) {
    return j.src ? (int)std::min<int64_t>(ceil_div(j.rows * (whole8(j.cols) / 4), 256), 8192) : 0;
  };
  Blocks n{0, copy_blocks(p.copy[0]), copy_blocks(p.copy[1]), 0, 0};
  if (p.dz.dy) n.dz = ceil_div(p.dz.cols, kDzCols) * p.dz.chunks;
  if (p.loss.rows) n.loss = ceil_div(p.loss.nq, 256);
  if (p.loss.owner) n.clear = std::min(ceil_div(p.loss.nc, 1024), 1024);
  const int total = n.dz + n.copy0 + n.copy1 + n.loss + n.clear;
  if (total == 0) return FGPU_OK;
  if (f32)
    prep_kernel<float><<<total, 256, 0, s>>>(p, n);
  else
    prep_kernel<bf16><<<total, 256, 0, s>>>(p, n);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

}  // namespace fgpu

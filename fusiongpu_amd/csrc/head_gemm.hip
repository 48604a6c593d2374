// head_gemm.hip -- products with a fused epilogue, the packing of their operands and the last step of column sums.
#include <algorithm>

#include "head.hpp"

namespace fgpu {
namespace {

// out = act(alpha D + bias) + residual for four consecutive columns n .. n + 3 of row m (cnt of them inside).
template <class T>
__device__ __forceinline__ void finish4(const Finish& f, f32x4 v, int64_t at, int n, int cnt) {
  v *= f.alpha;
  if (f.bias) v += load4_n((const T*)f.bias + n, cnt);
  if (f.pre) store4_n((T*)f.pre + at, v, cnt);
  if (f.act != FGPU_ACT_NONE) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = act_value(v[r], f.act);
  }
  if (f.residual) v += load4_n((const T*)f.residual + at, cnt);
  store4_n((T*)f.out + at, v, cnt);
}

template <class T, int ACT>
struct ProductEpi {
  Finish f;
  float* part;  // [split][m][n4] in place of the result, or NULL
  int m, n;

  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*) const {
    if (w.first_col() + G::FN * 16 <= n)
      whole(acc, w);
    else
      ragged(acc, w);
  }
  // Every column of the wave lies inside: straight from the accumulators, 16 bytes of bf16 a store.
  template <class G>
  __device__ __forceinline__ void whole(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    constexpr int P = G::FN / 2;
    if (part) {
      const int n4 = (n + 3) & ~3;
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        if (w.row(j) >= m) continue;
        float* d = part + ((int64_t)w.sp * m + w.row(j)) * n4 + w.col(0);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          *reinterpret_cast<f32x4*>(d + 32 * p) = acc[2 * p][j];
          *reinterpret_cast<f32x4*>(d + 32 * p + 4) = acc[2 * p + 1][j];
        }
      }
      return;
    }
    f32x8 bias[P];
#pragma unroll
    for (int p = 0; p < P; ++p) bias[p] = f.bias ? load8((const T*)f.bias + w.col(p)) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      if (w.row(j) >= m) continue;
      const int64_t at = (int64_t)w.row(j) * n + w.col(0);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.set(e, fmaf(acc[2 * p + e / 4][j][e % 4], f.alpha, bias[p][e]));
        if (f.pre) store8((T*)f.pre + at + 32 * p, v);
        if (ACT != FGPU_ACT_NONE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v.set(e, act_value(v[e], ACT));
        }
        if (f.residual) {
          const f32x8 r = load8((const T*)f.residual + at + 32 * p);
          v.lo += r.lo, v.hi += r.hi;
        }
        store8((T*)f.out + at + 32 * p, v);
      }
    }
  }
  // The wave holds the last columns: through LDS, four columns a lane, so the code that minds the edge stands once.
  template <class G>
  __device__ __forceinline__ void ragged(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    constexpr int kCols = G::FN * 16, kPass = GemmWave<G>::lds_bytes / (16 * kCols * 4) < G::FM
                                                  ? GemmWave<G>::lds_bytes / (16 * kCols * 4) : G::FM;
    static_assert(kPass > 0 && G::FM % kPass == 0, "whole passes");
    float* lds = reinterpret_cast<float*>(w.lds);
    const int n4 = (n + 3) & ~3;
#pragma unroll
    for (int j0 = 0; j0 < G::FM; j0 += kPass) {
      wave_lds_sync();
#pragma unroll
      for (int j = 0; j < kPass; ++j)
#pragma unroll
        for (int i = 0; i < G::FN; ++i) {
          const int row = j * 16 + (w.lane & 15), c4 = (w.col(i / 2) - w.first_col()) / 4 + (i & 1);
          *reinterpret_cast<f32x4*>(lds + row * kCols + 4 * (c4 ^ (row & (kCols / 4 - 1)))) = acc[i][j0 + j];
        }
      wave_lds_sync();
#pragma unroll 1
      for (int t = w.lane; t < kPass * 16 * kCols / 4; t += kWave) {
        const int row = t / (kCols / 4), c4 = t % (kCols / 4), col = w.first_col() + 4 * c4;
        const int gm = w.m0 + (w.wm * G::FM + j0) * 16 + row;
        if (gm >= m || col >= n) continue;
        const f32x4 v = *reinterpret_cast<const f32x4*>(lds + row * kCols + 4 * (c4 ^ (row & (kCols / 4 - 1))));
        if (part)
          *reinterpret_cast<f32x4*>(part + ((int64_t)w.sp * m + gm) * n4 + col) = v;
        else
          finish4<T>(f, v, (int64_t)gm * n + col, col, n - col);
      }
    }
  }
};

// Adds the parts of a split product in order and finishes it: one thread four columns.
template <class T>
__global__ __launch_bounds__(256) void split_finish_kernel(const float* part, int m, int n, int splits, Finish f) {
  const int n4 = (n + 3) >> 2;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, total = (int64_t)m * n4;
  if (i >= total) return;
  const int64_t row = i / n4;
  const int col = (int)(i - row * n4) * 4;
  f32x4 v = {0, 0, 0, 0};
  if (f.add) v = *reinterpret_cast<const f32x4*>(f.add + i * 4);
  for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(part + ((int64_t)s * total + i) * 4);
  if (f.sum)
    *reinterpret_cast<f32x4*>(f.sum + i * 4) = v;
  else
    finish4<T>(f, v, row * n + col, col, n - col);
}

struct Plan {
  int tile, tiles_m, tiles_n, splits, k_per_split;
};
Plan plan_of(const Product& p) {
  Plan q;
  auto tiles = [&](int t) { return (int64_t)ceil_div(p.m, t) * ceil_div(p.n, t); };
  q.tile = tiles(256) >= 192 ? 256 : tiles(128) >= 256 ? 128 : 64;
  q.tiles_m = ceil_div(p.m, q.tile);
  q.tiles_n = ceil_div(p.n, q.tile);
  const int64_t t = (int64_t)q.tiles_m * q.tiles_n;
  const int steps = ceil_div(p.k, kGemmBK);
  int64_t want = q.tile == 256 ? 1 : std::max<int64_t>(1, 512 / t);
  want = std::min<int64_t>(want, std::max(1, steps / 4));
  q.k_per_split = ceil_div(steps, want) * kGemmBK;
  q.splits = ceil_div(p.k, q.k_per_split);
  return q;
}

template <class T, bool AKC, bool BKC, int PAIRS, class E>
fgpu_status run(const GemmArgs& g, const E& e, hipStream_t s) {
  gemm_kernel<T, AKC, BKC, PAIRS, E><<<g.tiles_m * g.tiles_n * g.splits, T::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}
template <bool AKC, bool BKC, int PAIRS, class E>
fgpu_status run_tile(int tile, const GemmArgs& g, const E& e, hipStream_t s) {
  if (tile == 256) return run<Tile256, AKC, BKC, PAIRS>(g, e, s);
  if (tile == 128) return run<Tile128, AKC, BKC, PAIRS>(g, e, s);
  return run<Tile64, AKC, BKC, PAIRS>(g, e, s);
}
// The activation is part of the kernel's type where the product finishes it (the forward product alone has one).
template <int PAIRS, class T>
fgpu_status run_form(bool a_kc, bool b_kc, int tile, const GemmArgs& g, const Finish& f, float* part, hipStream_t s) {
  const ProductEpi<T, FGPU_ACT_NONE> plain{f, part, g.m, g.n};
  if (a_kc && !b_kc) return run_tile<true, false, PAIRS>(tile, g, plain, s);
  if (!a_kc) return run_tile<false, false, PAIRS>(tile, g, plain, s);
  if (part || f.act == FGPU_ACT_NONE) return run_tile<true, true, PAIRS>(tile, g, plain, s);
  if (f.act == FGPU_ACT_RELU) return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_RELU>{f, part, g.m, g.n}, s);
  if (f.act == FGPU_ACT_GELU) return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_GELU>{f, part, g.m, g.n}, s);
  return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_SILU>{f, part, g.m, g.n}, s);
}

template <class T>
__device__ __forceinline__ bool row_is_zero(int64_t r, const float* zb, const int32_t* zt, int nc) {
  return (zb && zb[r] <= FGPU_MASK_BIAS) || (zt && (uint32_t)zt[r] >= (uint32_t)nc);
}

// One thread four columns of a row.
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(const T* src, int64_t rows, int64_t cols, int64_t ldp, int64_t plane,
                                                   uint16_t* dst, const float* zb, const int32_t* zt, int nc) {
  const int64_t per = ldp / 4, total = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per, c = (i - r * per) * 4;
    f32x4 v = {0, 0, 0, 0};
    if (c < cols && !row_is_zero<T>(r, zb, zt, nc)) v = load4_n(src + r * cols + c, (int)min(cols - c, (int64_t)4));
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<bf16x4*>(dst + r * ldp + c) = __builtin_convertvector(v, bf16x4);
    } else {
      bf16x4 h, m, l;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        bf16 a, b, d;
        split_f32(v[k], a, b, d);
        h[k] = a, m[k] = b, l[k] = d;
      }
      *reinterpret_cast<bf16x4*>(dst + r * ldp + c) = h;
      *reinterpret_cast<bf16x4*>(dst + plane + r * ldp + c) = m;
      *reinterpret_cast<bf16x4*>(dst + 2 * plane + r * ldp + c) = l;
    }
  }
}

// 16 columns x 64 groups of parts a workgroup; blockIdx.y: which of two sums.
constexpr int kFinishCols = 16, kFinishGroups = 64;
template <class T>
__global__ __launch_bounds__(1024) void column_finish_kernel(const float* part, int parts, int64_t stride, int64_t cols,
                                                             T* out0, T* out1) {
  __shared__ float sum[kFinishGroups][kFinishCols + 1];
  T* out = blockIdx.y ? out1 : out0;
  if (!out) return;
  const int cl = threadIdx.x % kFinishCols, g = threadIdx.x / kFinishCols;
  const int64_t c = (int64_t)blockIdx.x * kFinishCols + cl;
  part += blockIdx.y * cols;
  float v = 0;
  if (c < cols)
    for (int p = g; p < parts; p += kFinishGroups) v += part[(int64_t)p * stride + c];
  sum[g][cl] = v;
  __syncthreads();
  // one wave a column: its 64 groups across the lanes
  const int w = threadIdx.x >> 6;
  v = lanes_sum<64>(sum[threadIdx.x & 63][w]);
  if ((threadIdx.x & 63) == 0 && (int64_t)blockIdx.x * kFinishCols + w < cols) out[(int64_t)blockIdx.x * kFinishCols + w] = (T)v;
}

}  // namespace

size_t product_workspace_bytes(const Product& p) {
  const Plan q = plan_of(p);
  return q.splits > 1 || p.chunked ? carve_bytes<float>((size_t)q.splits * p.m * ((p.n + 3) & ~3)) : 0;
}

fgpu_status launch_product(const Product& p, const GemmOperand& a, bool a_kc, const GemmOperand& b, bool b_kc,
                           const Finish& f, void* ws, hipStream_t s) {
  const Plan q = plan_of(p);
  const GemmArgs g{a, b, p.m, p.n, p.k, q.tiles_m, q.tiles_n, q.splits, q.k_per_split};
  float* part = q.splits > 1 || p.chunked ? static_cast<float*>(ws) : nullptr;
  if (p.f32)
    FGPU_TRY((run_form<6, float>(a_kc, b_kc, q.tile, g, f, part, s)));
  else
    FGPU_TRY((run_form<1, bf16>(a_kc, b_kc, q.tile, g, f, part, s)));
  if (part) {
    const int64_t total = (int64_t)p.m * ((p.n + 3) / 4);
    if (p.f32)
      split_finish_kernel<float><<<ceil_div(total, 256), 256, 0, s>>>(part, p.m, p.n, q.splits, f);
    else
      split_finish_kernel<bf16><<<ceil_div(total, 256), 256, 0, s>>>(part, p.m, p.n, q.splits, f);
    FGPU_HIP(hipGetLastError());
  }
  return FGPU_OK;
}

fgpu_status launch_pack(const void* src, int64_t rows, int64_t cols, bool f32, const GemmOperand& dst,
                        const float* zero_bias, const int32_t* zero_target, int nc, hipStream_t s) {
  const int64_t total = rows * (dst.ld / 4);
  const int grid = (int)std::min<int64_t>(ceil_div(total, 256), 8192);
  uint16_t* d = const_cast<uint16_t*>(dst.p);
  if (f32)
    pack_kernel<float><<<grid, 256, 0, s>>>((const float*)src, rows, cols, dst.ld, dst.plane, d, zero_bias, zero_target, nc);
  else
    pack_kernel<bf16><<<grid, 256, 0, s>>>((const bf16*)src, rows, cols, dst.ld, dst.plane, d, zero_bias, zero_target, nc);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_column_finish2(const float* part, int parts, int64_t stride, int64_t cols, bool f32_out, void* out0,
                                  void* out1, hipStream_t s) {
  const dim3 grid(ceil_div(cols, kFinishCols), out1 ? 2 : 1);
  if (f32_out)
    column_finish_kernel<float><<<grid, 1024, 0, s>>>(part, parts, stride, cols, (float*)out0, (float*)out1);
  else
    column_finish_kernel<bf16><<<grid, 1024, 0, s>>>(part, parts, stride, cols, (bf16*)out0, (bf16*)out1);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_column_finish(const float* part, int parts, int64_t stride, int64_t cols, bool f32_out, void* out,
                                 hipStream_t s) {
  return launch_column_finish2(part, parts, stride, cols, f32_out, out, nullptr, s);
}

}  // namespace fgpu

// head_gemm.hip -- products with a fused epilogue, and what joins split ones and column sums.
//
// Bound by the matrix units, and where k is short by the epilogue: 8192^3 in bf16 takes 0.82 ms (1.35 PFLOP/s; the library's
// plain product 1.44 to 1.6), 65536 x 4096 x 1024 with bias, GELU and the kept pre-activation 0.64 ms (0.86 PFLOP/s, 1.1 GB
// of stores), 8192 x 4096 x 4096 in float32 214 TFLOP/s (the library's float32 product 127 to 154).
#include <algorithm>
#include <type_traits>

#include "head.hpp"

namespace fgpu {
namespace {

// REST: with Finish::rest.
template <class T, int ACT, bool REST = false>
struct ProductEpi {
  Finish f;
  float* part;  // [split][m][n4] in place of the result, or NULL
  int m, n;

  template <class G>
  struct Side {
    __device__ void fetch(const ProductEpi&, int, int, int) {}
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
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
    f.stream ? rows<true>(acc, w) : rows<false>(acc, w);
  }
  // STREAM: results past the caches.  (A test at each store would be merged away, and the hint with it.)
  template <bool STREAM, class G>
  __device__ __forceinline__ void rows(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    constexpr int P = G::FN / 2;
    f32x8 bias[P];
#pragma unroll
    for (int p = 0; p < P; ++p) bias[p] = f.bias ? load8((const T*)f.bias + w.col(p)) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
    int head[G::FM];
    if constexpr (REST) {
#pragma unroll
      for (int j = 0; j < G::FM; ++j) head[j] = w.row(j) < m ? f.rest.row_of(w.row(j)) : -1;
    }
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      if (w.row(j) >= m) continue;
      const int64_t at = (int64_t)w.row(j) * n + w.col(0);
      f32x8 rest[P];
      if constexpr (REST) {
#pragma unroll
        for (int p = 0; p < P; ++p) rest[p] = f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
        if (f.rest.any(head[j])) {
          const float c = f.rest.coef_of(w.row(j), head[j]);
#pragma unroll
          for (int p = 0; p < P; ++p) {
            const f32x8 x = load8(f.rest.row(head[j]) + w.col(p));
            rest[p] = f32x8{x.lo * c, x.hi * c};
          }
        }
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float d = acc[2 * p + e / 4][j][e % 4];
          if constexpr (REST) d += rest[p][e];
          v.set(e, fmaf(d, f.alpha, bias[p][e]));
        }
        if (f.pre) put<STREAM>((T*)f.pre + at + 32 * p, v);
        if (ACT != FGPU_ACT_NONE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v.set(e, act_value<T>(v[e], ACT));
        }
        if (f.residual) {
          const f32x8 r = load8((const T*)f.residual + at + 32 * p);
          v.lo += r.lo, v.hi += r.hi;
        }
        put<STREAM>((T*)f.out + at + 32 * p, v);
      }
    }
  }
  template <bool STREAM>
  __device__ static __forceinline__ void put(T* p, const f32x8& v) {
    if constexpr (STREAM) stream8(p, v);
    else store8(p, v);
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
        f32x4 v = *reinterpret_cast<const f32x4*>(lds + row * kCols + 4 * (c4 ^ (row & (kCols / 4 - 1))));
        if (REST && !part) f.rest.add4(v, gm, col);
        if (part)
          *reinterpret_cast<f32x4*>(part + ((int64_t)w.sp * m + gm) * n4 + col) = v;
        else
          finish4<T>(f, v, (int64_t)gm * n + col, col, n - col);
      }
    }
  }
};

// Adds the parts of a split product in a fixed order and finishes it: a thread four columns, or, of many parts, sixteen
// threads four columns (each a sixteenth of the parts), so that few outputs of many parts are not one long chain of loads.
constexpr int kManyParts = 32;
template <class T>
__device__ __forceinline__ void split_finish(const SplitJob& j, int block) {
  __shared__ f32x4 sums[16][17];
  const bool many = j.splits >= kManyParts;
  const int n4 = (j.n + 3) >> 2, out = many ? threadIdx.x & 15 : threadIdx.x, group = many ? threadIdx.x >> 4 : 0;
  const int64_t i = (int64_t)block * (many ? 16 : 256) + out, total = (int64_t)j.m * n4;
  f32x4 v = {0, 0, 0, 0};
  if (i < total) {
    if (j.f.add && group == 0) v = *reinterpret_cast<const f32x4*>(j.f.add + i * 4);
#pragma unroll 4
    for (int s = group; s < j.splits; s += many ? 16 : 1)
      v += *reinterpret_cast<const f32x4*>(j.part + ((int64_t)s * total + i) * 4);
  }
  if (many) {
    sums[group][out] = v;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int s = 1; s < 16; ++s) v += sums[s][out];
  }
  if (i >= total) return;
  const int64_t row = i / n4;
  const int col = (int)(i - row * n4) * 4;
  if (j.f.sum) {
    *reinterpret_cast<f32x4*>(j.f.sum + i * 4) = v;
    return;
  }
  j.f.rest.add4(v, (int)row, col);
  finish4<T>(j.f, v, row * j.n + col, col, j.n - col);
}

// 16 columns x 16 groups of parts a workgroup.
constexpr int kSumCols = 16, kSumGroups = 16;
__device__ __forceinline__ void column_sum(const ColumnSum& c, const float* part, void* out, int block) {
  __shared__ float sum[kSumGroups][kSumCols + 1];
  const int cl = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
  const int64_t col = (int64_t)block * kSumCols + cl;
  float v = 0;
  if (col < c.cols)
#pragma unroll 4
    for (int p = g; p < c.parts; p += kSumGroups) v += part[(int64_t)p * c.stride + col];
  sum[g][cl] = v;
  __syncthreads();
  if (g == 0 && col < c.cols) {
#pragma unroll
    for (int k = 1; k < kSumGroups; ++k) v += sum[k][cl];
    if (c.f32) ((float*)out)[col] = v;
    else ((bf16*)out)[col] = (bf16)v;
  }
}
__global__ __launch_bounds__(256) void column_sum_kernel(ColumnSum c, void* out1) {
  void* out = blockIdx.y ? out1 : c.out;
  if (out) column_sum(c, c.part + blockIdx.y * c.cols, out, blockIdx.x);
}

// Zeros: 16 bytes a thread and step, the `rest` (fewer than 16, a whole number of elements) by the first workgroup.
__global__ __launch_bounds__(256) void zeros_kernel(char* out, int64_t vecs, int64_t rest) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < vecs; i += (int64_t)gridDim.x * 256)
    reinterpret_cast<u32x4u*>(out)[i] = u32x4u{0, 0, 0, 0};
  if (blockIdx.x == 0 && threadIdx.x < rest / 2) reinterpret_cast<uint16_t*>(out + vecs * 16)[threadIdx.x] = 0;
}

// What is left after the products, in one launch: the joining of up to two split ones, and column sums.  WALK: the grid does
// not hold all blocks (for the others the loop would cost 0.6 us a launch).
template <class T, bool WALK>
__global__ __launch_bounds__(256) void join_kernel(SplitJob a, int a_blocks, SplitJob b, int b_blocks, ColumnSum c, int blocks) {
  for (int k = blockIdx.x; k < blocks; k += gridDim.x) {
    if (k < a_blocks)
      split_finish<T>(a, k);
    else if (k < a_blocks + b_blocks)
      split_finish<T>(b, k - a_blocks);
    else
      column_sum(c, c.part, c.out, k - a_blocks - b_blocks);
    if (!WALK) return;
    __syncthreads();  // the LDS sums are read
  }
}
constexpr int kJoinGrid = 1 << 16;  // workgroups at most: a block's result is the same whichever takes it

// Microseconds of a product on `tile` tiles with k in `splits` parts.  A workgroup's k step takes `alone` while few share
// a CU and `shared` for each that does (measured: 256 x 256 1.6 / 1.6 at one a CU, 128 x 128 0.64 / 0.5 at two, 64 x 64
// 0.35 / 0.21 at five; float32's six plane products six times that, but 1.2 / 0.63 at three for 64 x 64, which holds all
// planes), its start and epilogue `fixed`; the parts of a split product are written and read once more.
Plan plan_at(const Product& p, int tile, int splits) {
  Plan q{tile, ceil_div(p.m, tile), ceil_div(p.n, tile), splits, 0, 0};
  const int steps = ceil_div(p.k, kGemmBK), per = ceil_div(steps, splits);
  q.k_per_split = per * kGemmBK;
  q.splits = ceil_div(p.k, q.k_per_split);
  const double alone = tile == 256 ? 1.6 : tile == 128 ? 0.64 : p.f32 ? 0.2 : 0.35;
  const double shared = tile == 256 ? 1.6 : tile == 128 ? 0.5 : p.f32 ? 0.105 : 0.21;
  const double fixed = tile == 256 ? 8 : tile == 128 ? 4 : 3;
  const int most = tile == 256 ? 1 : tile == 128 ? 2 : p.f32 ? 3 : 5;
  const int64_t wgs = (int64_t)q.tiles_m * q.tiles_n * q.splits, full = wgs / (256 * most), rest = wgs % (256 * most);
  const double k = (double)per * (p.f32 ? 6 : 1);
  q.us = full * (k * std::max(alone, most * shared) + fixed);
  if (rest) q.us += k * std::max(alone, ceil_div(rest, 256) * shared) + fixed;
  if (q.splits > 1) q.us += 3 + 8.0 * q.splits * p.m * ((p.n + 3) & ~3) / 6e6;
  return q;
}
int64_t plan_threads(const Plan& q) {
  const int threads = q.tile == 256 ? Tile256::threads : q.tile == 128 ? Tile128::threads : Tile64::threads;
  return (int64_t)q.tiles_m * q.tiles_n * q.splits * threads;
}
// Of the plans that are one launch (2^30 rows of up to 64 columns on 64 x 64 tiles are not).
Plan plan_of(const Product& p, int only = 0, bool may_split = true) {
  Plan best{};
  for (int tile : {256, 128, 64}) {
    if (only && tile != only) continue;
    for (int splits : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (splits > 1 && (!may_split || splits > ceil_div(p.k, 2 * kGemmBK))) break;
      const Plan q = plan_at(p, tile, splits);
      if (plan_threads(q) >= 2 * kLaunchThreads) continue;
      if (!best.tile || q.us < best.us) best = q;
    }
  }
  return best;
}
// Two products run in one launch, with one tile for both, where that costs less than their own tiles and a launch more.
constexpr double kLaunchUs = 3;
int plans_of(const Product* p, int count, Plan* q) {
  for (int i = 0; i < count; ++i) q[i] = plan_of(p[i]);
  if (count == 1) return 0;
  double us = q[0].us + q[1].us;
  int pair = 0;
  for (int tile : {128, 64}) {
    const Plan a = plan_of(p[0], tile), b = plan_of(p[1], tile);
    if (!a.tile || !b.tile || plan_threads(a) + plan_threads(b) >= 2 * kLaunchThreads) continue;
    if (a.us + b.us - kLaunchUs < us) us = a.us + b.us - kLaunchUs, pair = tile, q[0] = a, q[1] = b;
  }
  return pair;
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
  if constexpr (PAIRS == 1) {
    const ProductEpi<T, FGPU_ACT_NONE, true> rest{f, part, g.m, g.n};
    if (f.rest.head && !part && !b_kc)
      return a_kc ? run_tile<true, false, PAIRS>(tile, g, rest, s) : run_tile<false, false, PAIRS>(tile, g, rest, s);
  }
  if (a_kc && !b_kc) return run_tile<true, false, PAIRS>(tile, g, plain, s);
  if (!a_kc) return run_tile<false, false, PAIRS>(tile, g, plain, s);
  if (part || f.act == FGPU_ACT_NONE) return run_tile<true, true, PAIRS>(tile, g, plain, s);
  if (f.act == FGPU_ACT_RELU) return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_RELU>{f, part, g.m, g.n}, s);
  if (f.act == FGPU_ACT_GELU) return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_GELU>{f, part, g.m, g.n}, s);
  return run_tile<true, true, PAIRS>(tile, g, ProductEpi<T, FGPU_ACT_SILU>{f, part, g.m, g.n}, s);
}

size_t parts_bytes(const Product& p, const Plan& q) {
  return q.splits > 1 || p.chunked ? carve_bytes<float>((size_t)q.splits * p.m * ((p.n + 3) & ~3)) : 0;
}

template <int PAIRS, class O>
fgpu_status run_products(const ProductJob* jobs, int count, const Plan* q, int pair, float* const* part, const ColumnSum* sums,
                         hipStream_t s) {
  GemmArgs g[2];
  Finish f[2];
  for (int i = 0; i < count; ++i) {
    const ProductJob& j = jobs[i];
    g[i] = {j.a, j.b, j.p.m, j.p.n, j.p.k, q[i].tiles_m, q[i].tiles_n, q[i].splits, q[i].k_per_split};
    f[i] = j.f;
    // Results of more than the last-level cache's 256 MB go past it: what is written would only push the operands out
    // (65536 x 4096 x 1024 with its pre-activation 731 -> 624 us; at 134 MB it would cost 102 -> 128 us).
    f[i].stream = (int64_t)j.p.m * j.p.n * (int64_t)sizeof(O) * (j.f.pre ? 2 : 1) > (int64_t)256 << 20;
  }
  if (pair && jobs[0].asked && jobs[1].asked) {
    auto both = [&](auto rest) -> fgpu_status {
      using E = ProductEpi<O, FGPU_ACT_NONE, decltype(rest)::value>;
      const E ex{f[0], part[0], g[0].m, g[0].n}, ew{f[1], part[1], g[1].m, g[1].n};
      const int nx = g[0].tiles_m * g[0].tiles_n * g[0].splits, nw = g[1].tiles_m * g[1].tiles_n * g[1].splits;
      if (pair == 128)
        gemm_pair_kernel<Tile128, PAIRS><<<nx + nw, Tile128::threads, 0, s>>>(g[0], ex, nx, g[1], ew);
      else
        gemm_pair_kernel<Tile64, PAIRS><<<nx + nw, Tile64::threads, 0, s>>>(g[0], ex, nx, g[1], ew);
      FGPU_HIP(hipGetLastError());
      return FGPU_OK;
    };
    bool rest = false;
    for (int i = 0; i < 2; ++i) rest |= f[i].rest.head && !part[i];
    if constexpr (PAIRS == 1)
      FGPU_TRY(rest ? both(std::true_type{}) : both(std::false_type{}));
    else
      FGPU_TRY(both(std::false_type{}));
  } else {
    for (int i = 0; i < count; ++i)
      if (jobs[i].asked) FGPU_TRY((run_form<PAIRS, O>(jobs[i].a_kc, jobs[i].b_kc, q[i].tile, g[i], f[i], part[i], s)));
  }
  SplitJob sj[2];
  for (int i = 0; i < count; ++i)
    if (part[i]) sj[i].part = part[i], sj[i].m = g[i].m, sj[i].n = g[i].n, sj[i].splits = g[i].splits, sj[i].f = f[i];
  return launch_join(sj[0], sj[1], sums, sizeof(O) == 4, s);
}

}  // namespace

fgpu_status launch_join(const SplitJob& a, const SplitJob& b, const ColumnSum* sums, bool f32, hipStream_t s) {
  auto blocks = [](const SplitJob& j) {
    return j.part ? ceil_div((int64_t)j.m * ((j.n + 3) / 4), j.splits >= kManyParts ? 16 : 256) : 0;
  };
  const int na = blocks(a), nb = blocks(b), nc = sums ? ceil_div(sums->cols, kSumCols) : 0;
  const int all = na + nb + nc, grid = std::min(all, kJoinGrid);
  if (all == 0) return FGPU_OK;
  const auto k = f32 ? (all > grid ? join_kernel<float, true> : join_kernel<float, false>)
                     : (all > grid ? join_kernel<bf16, true> : join_kernel<bf16, false>);
  k<<<grid, 256, 0, s>>>(a, na, b, nb, sums ? *sums : ColumnSum{}, all);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

Plan plan_whole(const Product& p, int only_tile) { return plan_of(p, only_tile, false); }

size_t products_workspace_bytes(const Product* p, int count) {
  Plan q[2];
  plans_of(p, count, q);
  size_t b = 0;
  for (int i = 0; i < count; ++i) b += parts_bytes(p[i], q[i]);
  return b;
}
double products_estimate_us(const Product* p, int count) {
  Plan q[2];
  const int pair = plans_of(p, count, q);
  double us = 0;
  for (int i = 0; i < count; ++i) us += q[i].us;
  return pair ? us - kLaunchUs : us;
}

int products_tile(const Product* p, int count, int which) {
  Plan q[2];
  return plans_of(p, count, q) ? q[which].tile + FGPU_TILE_PAIR : q[which].tile;
}

fgpu_status launch_products(const ProductJob* jobs, int count, const ColumnSum* sums, void* ws, hipStream_t s) {
  Product p[2];
  Plan q[2];
  for (int i = 0; i < count; ++i) p[i] = jobs[i].p;
  const int pair = plans_of(p, count, q);
  for (int i = 0; i < count; ++i)
    FGPU_CHECK(q[i].tile, FGPU_ERR_UNSUPPORTED, "product: more tiles than one launch takes (2^39 results)");
  float* part[2] = {nullptr, nullptr};
  char* at = static_cast<char*>(ws);
  for (int i = 0; i < count; ++i) {
    const size_t b = jobs[i].asked ? parts_bytes(p[i], q[i]) : 0;
    if (b) part[i] = reinterpret_cast<float*>(at);
    at += b;
  }
  if (p[0].f32) return run_products<6, float>(jobs, count, q, pair, part, sums, s);
  return run_products<1, bf16>(jobs, count, q, pair, part, sums, s);
}

fgpu_status launch_zeros(int64_t count, bool f32, void* out, hipStream_t s) {
  const int64_t vecs = count / (f32 ? 4 : 8);
  zeros_kernel<<<(int)std::min<int64_t>(vecs / 256 + 1, 4096), 256, 0, s>>>((char*)out, vecs, count * (f32 ? 4 : 2) - vecs * 16);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_column_sums(const ColumnSum& c, void* out1, hipStream_t s) {
  const dim3 grid(ceil_div(c.cols, kSumCols), out1 ? 2 : 1);
  column_sum_kernel<<<grid, 256, 0, s>>>(c, out1);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

}  // namespace fgpu

// head_gated.hip -- the gated layer h = act(x Wg^T + bg) (x Wu^T + bu) and its gradients.
//
// Both projections are one product against the stacked weight [Wg; Wu]: a tile's B operand takes 32 rows of Wg and then the
// 32 of Wu that belong to the same hidden columns (GatedTileLoad), so a lane's accumulators hold g and u of the same
// columns and act(g) u is formed before anything is stored.  The gradients are those of one linear layer of 2 hidden columns
// once dz = [dh u act'(g) | dh act(g)] is there, which a launch of its own forms with its column sums (head_prep.hip).
//
// 65536 x 1024 -> 4096 in bfloat16 with both factors kept takes 1.06 to 1.10 ms (1.0 PFLOP/s), the matrix units busy 46 % of
// its cycles: sixteen steps of k, then an epilogue with its part of 1.6 GB of stores that nothing overlaps, as a 256 x 256 tile
// fills its CU (two workgroups of 128 x 128 a CU 1.15 ms, of 256 x 128 with k in steps of 32 through three buffers 1.17 to
// 1.23, starts set apart no gain).  Its gradients over 16384 rows 0.57 to 0.59 ms: dz 0.13 (670 MB, 5.0 TB/s), two products at
// 1.2 PFLOP/s (the matrix units busy 55 %).  One row 4.8 us, a launch and two rounds of loads (eight columns of each half a
// workgroup, so that 2048 hidden ones are a workgroup a CU).
#include <algorithm>
#include <cmath>

#include "gated.hpp"
#include "head_direct.hpp"

namespace fgpu {
namespace {

constexpr int kMaxHidden = FGPU_HEAD_MAX_DIM / 2;

// ---- float32, planes formed on the way to LDS -----------------------------------------
// Mid-size float32 layers: a launch that copies both operands into planes first costs as much as a third of the product,
// and what it wrote comes back through other XCDs' caches.  Here a thread loads eight values of a row as they lie (any
// alignment), two steps ahead, splits them in registers and writes the three planes; each value is split once a tile
// instead of once.  1000 x 385 -> 771: 17.0 us, thirteen steps of 0.95 us: LDS, conversions and matrix instructions of a
// step take 0.5, 0.3 and 0.3 and overlap little behind its one barrier.
struct SplitJob32 {
  const float* x;
  const float* w;
  int m, n, k;
  int tiles_n;
};
struct Eight {
  f32x8 v;
  // Eight values of row `row` from k on; zeros outside.
  __device__ __forceinline__ void load(const float* p, int64_t row, bool in, int k, int nk) {
    v = f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (in && k < nk) v = load8_n(p + row * nk + k, nk - k);
  }
};
template <class T, int ACT>
__global__ __launch_bounds__(T::threads, 2) void gated_split_kernel(SplitJob32 j, GatedEpi<float, ACT> epi) {
  // Chunks of eight values: a thread takes one of each operand, or two of one; of fewer chunks than threads, the first waves.
  constexpr int B = kPlanesBK, pa = T::BM * B * 2, pb = T::BN * B * 2;
  constexpr int ka = (T::BM * 4 + T::threads - 1) / T::threads, kb = (T::BN * 4 + T::threads - 1) / T::threads;
  constexpr int ta = T::BM * 4 < T::threads ? T::BM * 4 : T::threads, tb = T::BN * 4 < T::threads ? T::BN * 4 : T::threads;
  static_assert(ka * ta == T::BM * 4 && kb * tb == T::BN * 4, "whole chunks a thread");
  __shared__ __attribute__((aligned(1024))) char s0[3 * (pa + pb)];
  __shared__ __attribute__((aligned(1024))) char s1[3 * (pa + pb)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  GemmArgs g{};
  g.tiles_n = j.tiles_n, g.tiles_m = gridDim.x / j.tiles_n;
  int tm, tn, sp;
  gemm_tile_of(g, blockIdx.x, gridDim.x, tm, tn, sp);
  const int m0 = tm * T::BM, n0 = tn * (T::BN / 2), chunk = tid & 3, row = tid >> 2;
  TileRead<T::BM, true, false, B> ra;
  TileRead<T::BN, true, true, B> rb;
  ra.init(lane, wm * (T::BM / T::WM));
  rb.init(lane, wn * (T::BN / T::WN));
  struct Stage {
    Eight a[ka], b[kb];
  };
  const bool has_a = ta == T::threads || wave < ta / kWave, has_b = tb == T::threads || wave < tb / kWave;
  auto load = [&](Stage& t, int k) {
#pragma unroll
    for (int i = 0; i < ka; ++i) {
      const int r = row + i * (ta / 4);
      t.a[i].load(j.x, m0 + r, has_a && m0 + r < j.m, k + chunk * 8, j.k);
    }
#pragma unroll
    for (int i = 0; i < kb; ++i) {
      const int r = row + i * (tb / 4), h = n0 + (r >> 6) * 32 + (r & 31);
      t.b[i].load(j.w, (r & 32) ? (int64_t)h + j.n : h, has_b && h < j.n, k + chunk * 8, j.k);
    }
  };
  auto put = [&](char* at, int plane, const Eight& e) {
    bf16x8 p[3];
    split8(e.v, p[0], p[1], p[2]);
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(at + q * plane) = p[q];
  };
  auto store = [&](const Stage& t, char* s) {
#pragma unroll
    for (int i = 0; i < ka; ++i) {
      const int r = row + i * (ta / 4);
      if (has_a) put(s + r * (B * 2) + (chunk ^ tile_swizzle<true, false, 4>(r)) * 16, pa, t.a[i]);
    }
#pragma unroll
    for (int i = 0; i < kb; ++i) {
      const int r = row + i * (tb / 4);
      if (has_b) put(s + 3 * pa + r * (B * 2) + (chunk ^ tile_swizzle<true, true, 4>(r)) * 16, pb, t.b[i]);
    }
  };
  f32x4 acc[T::FN][T::FM];
#pragma unroll
  for (int i = 0; i < T::FN; ++i)
#pragma unroll
    for (int q = 0; q < T::FM; ++q) acc[i][q] = f32x4{0, 0, 0, 0};
  auto work = [&](const char* s) {
    bf16x8 a[T::FM][3], b[T::FN][3];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int i = 0; i < T::FN; ++i) b[i][p] = rb.get((const lds_char*)s + 3 * pa + p * pb, i, 0);
#pragma unroll
      for (int q = 0; q < T::FM; ++q) a[q][p] = ra.get((const lds_char*)s + p * pa, q, 0);
    }
#pragma unroll
    for (int q = 0; q < T::FM; ++q)
#pragma unroll
      for (int i = 0; i < T::FN; ++i)
#pragma unroll
        for (int c = 0; c < 6; ++c) acc[i][q] = OfBf16::mma(b[i][pair_b(c)], a[q][pair_a(c)], acc[i][q]);
  };
  // Behind the barrier of step i its planes are in `cur`, nobody reads `other`, and the values of i + 1 and i + 2 are on the
  // way. The next step's planes are formed between this one's matrix instructions.
  auto step = [&](char* cur, char* other, Stage& next, int k) {
    __syncthreads();
    work(cur);
    store(next, other);
    load(next, k + 3 * B);
#pragma unroll
    for (int i = 0; i < T::FM * T::FN * 6; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // and four others
    }
  };
  Stage t0, t1;
  load(t0, 0);
  load(t1, B);
  store(t0, s0);
  load(t0, 2 * B);
  int k = 0;
  for (; k + B < j.k; k += 2 * B) {
    step(s0, s1, t1, k);
    step(s1, s0, t0, k + B);
  }
  if (k < j.k) {
    __syncthreads();
    work(s0);
  }
  const GemmWave<T> w{m0, n0, tm, tn, 0, wm, wn, lane, s1};
  epi.template finish<T>(acc, w, s1, typename GatedEpi<float, ACT>::template Side<T>{});
}
using WideSplitTile = GemmTile<64, 128, 4, 2>;
template <class T>
fgpu_status run_split(SplitJob32 j, const Finish& f, hipStream_t s) {
  j.tiles_n = ceil_div(j.n, T::BN / 2);
  auto go = [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    const GatedEpi<float, ACT> epi{f, {}, j.m, j.n};
    gated_split_kernel<T, ACT><<<ceil_div(j.m, T::BM) * j.tiles_n, T::threads, 0, s>>>(j, epi);
  };
  using std::integral_constant;
  switch (f.act) {
    case FGPU_ACT_NONE: go(integral_constant<int, FGPU_ACT_NONE>{}); break;
    case FGPU_ACT_RELU: go(integral_constant<int, FGPU_ACT_RELU>{}); break;
    case FGPU_ACT_GELU: go(integral_constant<int, FGPU_ACT_GELU>{}); break;
    default: go(integral_constant<int, FGPU_ACT_SILU>{});
  }
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}
// Microseconds, fitted over 100 to 8000 rows, 96 to 2048 hidden and 96 to 2048 k: a step of 32 k of a workgroup alone on its
// CU, and of each of several.
double split_us(int m, int n, int k, int width) {
  const int64_t each = ceil_div((int64_t)ceil_div(m, 64) * ceil_div(n, width / 2), 256);
  const double alone = width == 64 ? 0.66 : 0.98, shared = width == 64 ? 0.54 : 0.86;
  return 3.3 + ceil_div(k, kPlanesBK) * (each == 1 ? alone : each * shared);
}

fgpu_status check_common(int64_t rows, int in_dim, int hidden, int dtype, int act) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "gated linear: unknown dtype");
  FGPU_CHECK(act >= FGPU_ACT_NONE && act <= FGPU_ACT_SILU, FGPU_ERR_ARG, "gated linear: unknown activation");
  FGPU_CHECK(rows >= 0 && in_dim >= 1 && hidden >= 1, FGPU_ERR_ARG, "gated linear: rows >= 0, in_dim and hidden >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && in_dim <= FGPU_HEAD_MAX_DIM && hidden <= kMaxHidden, FGPU_ERR_UNSUPPORTED,
             "gated linear: more than 2^30 rows, 2^16 input dims or 2^15 hidden ones");
  return FGPU_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Which kernel a forward call takes, by estimates: that of few tiles, tiles whose planes are formed on the way (float32), or
// tiles of operands as they are or packed (a launch more).  us, few / on the way / packed: float32 1000 x 771 x 385 (rows,
// hidden, in) - / 17.2 / 25.9, 2000 x 771 x 385 - / 25.9 / 42.7, 300 x 771 x 1024 20.6 / 23.9 / -, 4000 x 2048 x 1024 - / 197
// / 167.
struct Choice {
  bool direct = false;
  int split = 0;  // the width of its tiles
  Plan plan;
};
Choice choose(int m, int n, int k, bool f32) {
  const Product p{m, 2 * n, k, f32};
  Choice c;
  c.plan = plan_whole(p, f32 ? 256 : 0);  // smaller packed tiles of float32 are slower than those formed on the way
  double us = c.plan.tile ? c.plan.us : INFINITY;
  if (needs_pack(k, f32)) us += 5.7 + ((double)p.m + p.n) * k * (f32 ? 10 : 4) / 4e6;
  if (f32 && (int64_t)ceil_div(m, 64) * ceil_div(n, 32) * GatedTile64::threads < kLaunchThreads) {
    for (int width : {64, 128}) {
      const double t = split_us(m, n, k, width);
      if (t < us) us = t, c.split = width;
    }
  }
  const bool one_launch = (int64_t)ceil_div(m, 32) * ceil_div(n, 16) * kDirectThreads < kLaunchThreads;
  if (one_launch && direct_forward_estimate_us(p) < us) c.direct = true, c.split = 0;
  return c;
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

int fgpu_gated_linear_tile(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return -1;
  const Choice c = choose((int)rows, hidden, in_dim, dtype == FGPU_DTYPE_F32);
  return c.direct ? 0 : c.split ? c.split + FGPU_TILE_SPLIT : c.plan.tile ? c.plan.tile : -1;
}

size_t fgpu_gated_linear_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  if (!needs_pack(in_dim, f32)) return 0;
  const Choice c = choose((int)rows, hidden, in_dim, f32);
  if (c.direct || c.split) return 0;
  return packed_bytes(rows, in_dim, f32) + packed_bytes(2 * hidden, in_dim, f32);
}

fgpu_status fgpu_gated_linear(const void* d_x, const void* d_w, const void* d_bias, int64_t rows, int in_dim, int hidden,
                              int dtype, int act, void* d_h, void* d_pre, void* d_workspace, size_t workspace_bytes,
                              void* stream) {
  FGPU_TRY(check_common(rows, in_dim, hidden, dtype, act));
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_w && d_h, FGPU_ERR_ARG, "gated linear: null x, weight or output");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "gated linear: x, weight and workspace must be 16-byte aligned");
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  const int m = (int)rows;
  const Choice c = choose(m, hidden, in_dim, f32);
  Finish f;
  f.bias = d_bias, f.out = d_h, f.pre = d_pre, f.act = act;
  if (c.direct) {
    const DirectOperand x{d_x, in_dim, rows * in_dim, nullptr}, w{d_w, in_dim, (int64_t)2 * hidden * in_dim, nullptr, hidden};
    const DirectJob j{x, w, m, hidden, in_dim, 0, f, nullptr};
    return launch_direct_gated(j, f32, s);
  }
  if (c.split) {
    const SplitJob32 j{(const float*)d_x, (const float*)d_w, m, hidden, in_dim, 0};
    return c.split == 64 ? run_split<GatedTile64>(j, f, s) : run_split<WideSplitTile>(j, f, s);
  }
  FGPU_CHECK(c.plan.tile, FGPU_ERR_UNSUPPORTED, "gated linear: more tiles than one launch takes (2^39 results)");
  Carve ws(d_workspace, workspace_bytes);
  GemmOperand a = as_is(d_x, in_dim), b = as_is(d_w, in_dim);
  Prep prep;
  if (needs_pack(in_dim, f32)) {
    a = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    b = packed(ws.take<char>(packed_bytes(2 * hidden, in_dim, f32)), 2 * hidden, in_dim);
    prep.copy[0] = {d_x, rows, in_dim, a};
    prep.copy[1] = {d_w, 2 * hidden, in_dim, b};
  }
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "gated linear: workspace smaller than fgpu_gated_linear_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  if (f32) return run_gated<6, OfBf16, float>(a, b, hidden * b.ld, m, hidden, in_dim, c.plan, f, {}, s);
  return run_gated<1, OfBf16, bf16>(a, b, hidden * b.ld, m, hidden, in_dim, c.plan, f, {}, s);
}

size_t fgpu_gated_linear_backward_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const int out = 2 * hidden;
  const Product p[2] = {{(int)rows, in_dim, out, f32}, {out, in_dim, (int)rows, f32}};
  size_t b = packed_bytes(rows, out, f32) + carve_bytes<float>((size_t)dz_chunks((int)rows, hidden) * out);
  if (needs_pack(in_dim, f32)) b += packed_bytes(rows, in_dim, f32) + packed_bytes(out, in_dim, f32);
  return b + products_workspace_bytes(p, 2);
}

fgpu_status fgpu_gated_linear_backward(const void* d_dh, const void* d_x, const void* d_w, const void* d_pre, int64_t rows,
                                       int in_dim, int hidden, int dtype, int act, void* d_dx, void* d_dw, void* d_db,
                                       void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, in_dim, hidden, dtype, act));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const int m = (int)rows, out = 2 * hidden;
  hipStream_t s = as_stream(stream);
  FGPU_CHECK(rows == 0 || (d_dh && d_pre), FGPU_ERR_ARG, "gated linear backward: null dh or kept halves");
  FGPU_CHECK(rows == 0 || ((!d_dx || d_w) && (!d_dw || d_x)), FGPU_ERR_ARG,
             "gated linear backward: dx needs the weight, dw needs x");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "gated linear backward: x, weight and workspace must be 16-byte aligned");
  if (rows == 0) {
    if (d_dw) FGPU_TRY(launch_zeros((int64_t)out * in_dim, f32, d_dw, s));
    if (d_db) FGPU_TRY(launch_zeros(out, f32, d_db, s));
    return FGPU_OK;
  }
  if (!d_dx && !d_dw && !d_db) return FGPU_OK;
  const Product px{m, in_dim, out, f32}, pw{out, in_dim, m, f32};
  const bool products = d_dx || d_dw, pk = needs_pack(in_dim, f32);
  Carve ws(d_workspace, workspace_bytes);
  Prep prep;
  GemmOperand z{}, w = as_is(d_w, in_dim), x = as_is(d_x, in_dim);
  if (products) z = packed(ws.take<char>(packed_bytes(rows, out, f32)), rows, out);
  ColumnSum sums;
  if (d_db) {
    sums.parts = dz_chunks(m, hidden), sums.stride = sums.cols = out, sums.out = d_db, sums.f32 = f32;
    sums.part = ws.take<float>((size_t)sums.parts * out);
  }
  prep.dz = {d_dh, d_pre, act, m, hidden, dz_chunks(m, hidden), z, const_cast<float*>(sums.part), true};
  if (pk && d_dx) {
    w = packed(ws.take<char>(packed_bytes(out, in_dim, f32)), out, in_dim);
    prep.copy[0] = {d_w, out, in_dim, w};
  }
  if (pk && d_dw) {
    x = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    prep.copy[1] = {d_x, rows, in_dim, x};
  }
  Finish fx, fw;
  fx.out = d_dx, fw.out = d_dw;
  const ProductJob jobs[2] = {{px, z, w, true, false, fx, d_dx != nullptr}, {pw, z, x, false, false, fw, d_dw != nullptr}};
  const Product ps[2] = {px, pw};
  void* parts = ws.take<char>(products_workspace_bytes(ps, 2));
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE,
             "gated linear backward: workspace smaller than fgpu_gated_linear_backward_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  if (!products) return launch_column_sums(sums, nullptr, s);
  return launch_products(jobs, 2, d_db ? &sums : nullptr, parts, s);
}

}  // extern "C"

// head_loss.hip -- the softmax contrastive loss of queries against candidate vectors, and its gradient.
//
// s_ij = scale q_i.c_j + bias_j over the candidates j that row i keeps; lse_i = log sum_j exp s_ij and
// loss_i = lse_i - s_i,t(i).  Up to 128 dims the kernels of head_narrow.hip serve; here are the wider ones and the entry
// points.  Neither pass holds the score matrix: the forward pass keeps a running maximum and sum a
// (row, column tile) in the product's epilogue and joins them; the backward pass forms the product again, turns it
// into G_ij = g_i (exp(s_ij - lse_i) - [j = t(i)]) in the epilogue and takes dq = scale G c and dc = scale G^T q from it
// in column chunks that bound the workspace.  Scores live in units of log 2 (s log2 e), so an exponential is one
// instruction.
//
// In bfloat16 G enters the two products rounded.  A target's element is about as large as its row's others together, and its
// rounding would be on the whole result: what it leaves is added to the two results past the products, in float32 in their
// epilogues, left_i c_t(i) to dq_i and left_i q_i to dc_j for the first row i with target j (rows that share a target are
// few in training; a list of them would cost a classifier's thousands more than the whole).  In norm the gradients are then
// as far from the exact ones as their own rounding puts them, 0.0017, instead of 0.0021 to 0.0025 (300 x 1500 x 200, both
// gradients, 17.9 -> 20.2 us, 8192 x 65536 x 768 2474 -> 2485).
//
// Above 128 dims a row's gradient no longer fits the registers beside its vector, and reading G back costs less than a
// third product.  8192 x 65536 x 768 in bf16: statistics 0.88 ms (0.94 PFLOP/s), G 0.98 ms, dq and dc 0.68 each (1.2
// PFLOP/s): the two score products have twelve k steps a tile only, and their epilogues (an exponential an element; G's
// stores) are not hidden, because a 256 x 256 tile leaves a CU room for one workgroup.
#include <algorithm>
#include <type_traits>

#include "loss_scores.hpp"

namespace fgpu {
namespace {

// What the epilogues need of a tile's rows and columns: fetched a row or column a thread while the products run, laid out
// in LDS after them.  grad: the rows' (lse, weight) too.
template <class G, bool GRAD>
struct LossSide {
  static_assert(G::threads >= G::BM + G::BN, "a thread a row and column");
  int t = -1, id = 0;  // a row's target (-1: none) and its document, or a column's bias in units of log 2 and document
  float bias2 = -INFINITY;
  f32x2 row = {INFINITY, 0.0f};
  struct Lds {
    int t[G::BM], row_id[G::BM];
    f32x2 row[GRAD ? G::BM : 1];
    float bias2[G::BN];
    int col_id[G::BN];
  };
  static_assert(sizeof(Lds) <= G::stage_bytes / 2, "beside the epilogue's own buffers");

  __device__ __forceinline__ void fetch(const LossArgs& a, const LossRow* rows, int m0, int n, int tid) {
    if (tid < G::BM) {
      const int m = m0 + tid;
      if (m >= a.nq) return;
      if constexpr (GRAD) {
        const LossRow r = rows[m];
        row = f32x2{r.lse2, r.weight};
        t = r.target, id = r.id;
      } else {
        t = a.target[m];
        if ((uint32_t)t >= (uint32_t)a.nc) t = -1;
        if (a.ids && t >= 0) id = a.ids[t];
      }
    } else if (tid < G::BM + G::BN) {
      n += tid - G::BM;
      if (n >= a.nc) return;
      const float b = a.bias ? a.bias[n] : 0.0f;
      bias2 = b <= FGPU_MASK_BIAS ? -INFINITY : b * kLog2e;
      if (a.ids) id = a.ids[n];
    }
  }
  __device__ __forceinline__ Lds& put(char* lds, int tid) const {
    Lds& l = *reinterpret_cast<Lds*>(lds);
    if (tid < G::BM) {
      l.t[tid] = t, l.row_id[tid] = id;
      if (GRAD) l.row[tid] = row;
    } else if (tid < G::BM + G::BN) {
      l.bias2[tid - G::BM] = bias2, l.col_id[tid - G::BM] = id;
    }
    __syncthreads();
    return l;
  }
};
// Forward, of the columns from c0 on: per row and column tile (maximum, sum of exp2(s - maximum)), and the target's score.
struct StatsEpi {
  LossArgs a;
  f32x2* part;     // [tiles_n][nq]
  float* target2;  // [nq]
  int c0;

  template <class G>
  struct Side : LossSide<G, false> {
    __device__ __forceinline__ void fetch(const StatsEpi& e, int m0, int n0, int tid) {
      LossSide<G, false>::fetch(e.a, nullptr, m0, e.c0 + n0, tid);
    }
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char* lds, const Side<G>& side) const {
    constexpr int P = G::FN / 2;
    const auto& l = side.put(lds, threadIdx.x);
    f32x2* sh = reinterpret_cast<f32x2*>(lds + G::stage_bytes / 2);  // [WN][BM]
    ColumnSide cs[P];
#pragma unroll
    for (int p = 0; p < P; ++p) cs[p].load(l, w.col(p) - w.n0);
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      const int m = w.row(j);
      const RowSide rs{l.t[m - w.m0], l.row_id[m - w.m0]};
      f32x8 v[P];
      float top = -INFINITY;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        v[p] = f32x8{acc[2 * p][j], acc[2 * p + 1][j]};
        uint32_t at;
        const bool here = scores8(a, v[p], cs[p], rs, c0 + w.col(p), at);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, v[p][e]);  // a NaN score makes the sum NaN
        if (here) {
          float x = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) x = at == e ? v[p][e] : x;
          target2[m] = x;
        }
      }
      top = fmaxf(top, __int_as_float(xchg<16>(__float_as_int(top))));
      top = fmaxf(top, __int_as_float(xchg<32>(__float_as_int(top))));
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += fast_exp2(v[p][e] - base);
      sum += __int_as_float(xchg<16>(__float_as_int(sum)));
      sum += __int_as_float(xchg<32>(__float_as_int(sum)));
      if (w.lane < 16) sh[w.wn * G::BM + m - w.m0] = f32x2{top, sum};
    }
    __syncthreads();
    for (int ml = threadIdx.x; ml < G::BM; ml += G::threads) {
      if (w.m0 + ml >= a.nq) continue;
      float top = -INFINITY, sum = 0;
#pragma unroll
      for (int k = 0; k < G::WN; ++k) top = fmaxf(top, sh[k * G::BM + ml][0]);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int k = 0; k < G::WN; ++k) sum += sh[k * G::BM + ml][1] * fast_exp2(sh[k * G::BM + ml][0] - base);
      part[(int64_t)w.tn * a.nq + w.m0 + ml] = f32x2{top, sum};
    }
  }
};

// Joins a row's parts: 16 rows a workgroup, 64 groups of parts.  `carry` ([nq], may be the first of the parts; NULL: these
// are the last columns): gets the joined part in place of the loss.
constexpr int kJoinRows = 16, kJoinGroups = 64;
__device__ __forceinline__ void join_stats(float& top, float& sum, float t, float s) {
  const float both = fmaxf(top, t);
  sum = both == -INFINITY ? sum + s : sum * fast_exp2(top - both) + s * fast_exp2(t - both);  // nothing yet: zero, or NaN
  top = both;
}
__global__ __launch_bounds__(1024) void loss_join_kernel(LossArgs a, const f32x2* part, int parts, const float* target2,
                                                         float* loss, float* lse, f32x2* carry) {
  __shared__ f32x2 sh[kJoinRows][kJoinGroups + 1];
  const int r = threadIdx.x % kJoinRows, g = threadIdx.x / kJoinRows;
  {
    const int m = blockIdx.x * kJoinRows + r;
    float top = -INFINITY, sum = 0;
    if (m < a.nq)
      for (int p = g; p < parts; p += kJoinGroups) {
        const f32x2 v = part[(int64_t)p * a.nq + m];
        join_stats(top, sum, v[0], v[1]);
      }
    sh[r][g] = f32x2{top, sum};
  }
  __syncthreads();
  // a wave a row
  const int w = threadIdx.x >> 6, m = blockIdx.x * kJoinRows + w;
  const f32x2 v = sh[w][threadIdx.x & 63];
  const float top = wave_max_f(v[0]), base = top == -INFINITY ? 0.0f : top;
  const float sum = lanes_sum<64>(v[1] * fast_exp2(v[0] - base));
  if (threadIdx.x % kWave || m >= a.nq) return;
  if (carry) {
    carry[m] = f32x2{top, sum};
    return;
  }
  const float l2 = base + __builtin_amdgcn_logf(sum);  // log2; of 0: -inf
  lse[m] = l2 * kLn2;
  const int t = a.target[m];
  const bool live = (uint32_t)t < (uint32_t)a.nc && l2 != -INFINITY;
  loss[m] = live ? (l2 - target2[m]) * kLn2 : 0.0f;
}

template <bool STREAM>
__device__ __forceinline__ void store_g(uint16_t* d, const bf16x8& v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<bf16x8*>(d));
  else *reinterpret_cast<bf16x8*>(d) = v;
}

// Backward: G of the columns c0 .. c0 + n - 1, as an operand [nq][ldg], and its column sums a tile row.
// STREAM: past the caches (a G larger than the last-level cache comes back from memory anyway).
template <bool F32, bool STREAM>
struct GradEpi {
  LossArgs a;
  const LossRow* rows;
  uint16_t* g;
  int64_t ldg, plane;
  float* dbias_part;  // [tiles_m][n] or NULL
  int c0, n;          // the chunk's columns
  float* left;        // bfloat16: what its rounding takes from each row's target element
  int* owner;         // and the first row of each target, [nc] (NULL: not wanted)

  template <class G>
  struct Side : LossSide<G, true> {
    __device__ __forceinline__ void fetch(const GradEpi& e, int m0, int n0, int tid) {
      LossSide<G, true>::fetch(e.a, e.rows, m0, e.c0 + n0, tid);
    }
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char* lds, const Side<G>& side) const {
    constexpr int P = G::FN / 2;
    const auto& l = side.put(lds, threadIdx.x);
    ColumnSide cs[P];
    f32x8 col[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      cs[p].load(l, w.col(p) - w.n0);
      col[p] = f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
    }
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      const int m = w.row(j);
      const RowSide rs{l.t[m - w.m0], l.row_id[m - w.m0]};
      const f32x2 row = l.row[m - w.m0];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int nl = w.col(p);
        f32x8 v{acc[2 * p][j], acc[2 * p + 1][j]};
        uint32_t at;
        const bool here = scores8(a, v, cs[p], rs, c0 + nl, at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v.set(e, fast_exp2(v[e] - row[0]));
        if (here) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v.set(e, at == e ? v[e] - 1.0f : v[e]);
        }
        v.lo *= row[1], v.hi *= row[1];
        if (!F32 && here) {
          float x = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) x = at == e ? v[e] : x;
          left[m] = x - (float)(bf16)x;
          if (owner && owner[rs.t] > m) atomicMin(owner + rs.t, m);  // the test: few of many rows with one target go on
        }
        col[p].lo += v.lo, col[p].hi += v.hi;
        if (m < a.nq && nl < ldg) {  // the padding's columns are zero
          uint16_t* d = g + (int64_t)m * ldg + nl;
          if constexpr (!F32) {
            store_g<STREAM>(d, to_bf16x8(v));
          } else {
            bf16x8 h, mi, l;
            split8(v, h, mi, l);
            store_g<STREAM>(d, h);
            store_g<STREAM>(d + plane, mi);
            store_g<STREAM>(d + 2 * plane, l);
          }
        }
      }
    }
    if (!dbias_part) return;
    float* sh = reinterpret_cast<float*>(lds + G::stage_bytes / 2);  // [WM][BN]
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = col[p][e];
        v = lanes_sum<16>(v);
        if ((w.lane & 15) == 0) sh[w.wm * G::BN + w.col(p) - w.n0 + e] = v;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < G::BN; c += G::threads) {
      if (w.n0 + c >= n) continue;
      float v = 0;
#pragma unroll
      for (int k = 0; k < G::WM; ++k) v += sh[k * G::BN + c];
      dbias_part[(int64_t)w.tm * n + w.n0 + c] = v;
    }
  }
};

struct ScorePlan {
  int tile, tiles_m, tiles_n;
};
ScorePlan score_plan(int nq, int nc) {
  auto tiles = [&](int t) { return (int64_t)ceil_div(nq, t) * ceil_div(nc, t); };
  const int t = tiles(256) >= 192 ? 256 : tiles(128) >= 192 ? 128 : 64;
  return {t, ceil_div(nq, t), ceil_div(nc, t)};
}

template <int PAIRS, class E>
fgpu_status launch_scores(const ScorePlan& p, const GemmOperand& q, const GemmOperand& c, int nq, int nc, int dim, const E& e,
                          hipStream_t s) {
  const GemmArgs g{q, c, nq, nc, dim, p.tiles_m, p.tiles_n, 1, (dim + kGemmBK - 1) / kGemmBK * kGemmBK};
  const int grid = p.tiles_m * p.tiles_n;
  if (p.tile == 256)
    gemm_kernel<Tile256, true, true, PAIRS, E><<<grid, Tile256::threads, 0, s>>>(g, e);
  else if (p.tile == 128)
    gemm_kernel<Tile128, true, true, PAIRS, E><<<grid, Tile128::threads, 0, s>>>(g, e);
  else
    gemm_kernel<Tile64, true, true, PAIRS, E><<<grid, Tile64::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_loss_join(const LossArgs& a, const f32x2* part, int parts, const float* target2, float* loss, float* lse,
                             f32x2* carry, hipStream_t s) {
  loss_join_kernel<<<ceil_div(a.nq, kJoinRows), 1024, 0, s>>>(a, part, parts, target2, loss, lse, carry);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status check_loss(int nq, int nc, int dim, int dtype) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "contrastive loss: unknown dtype");
  FGPU_CHECK(nq >= 0 && nc >= 1 && dim >= 1, FGPU_ERR_ARG, "contrastive loss: nq >= 0, nc and dim >= 1");
  FGPU_CHECK(nq <= FGPU_LOSS_MAX_QUERIES && nc <= FGPU_HEAD_MAX_ROWS && dim <= FGPU_HEAD_MAX_DIM, FGPU_ERR_UNSUPPORTED,
             "contrastive loss: more than 2^20 queries, 2^30 candidates or 2^16 dims");
  return FGPU_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Columns of G held at a time at most: 2^31 elements of G, whole tiles, and at most 2^20 columns, which keeps a tile's rows
// within 32-bit offsets.
int64_t most_columns(int nq, int nc) {
  const int64_t most = std::min<int64_t>((int64_t)1 << 20, ((int64_t)1 << 31) / std::max(1, nq));
  return std::min<int64_t>(nc, most / 256 * 256);
}
// Room for the products of a chunk of `step` columns and of the last, shorter one.
size_t chunk_products_bytes(int nq, int nc, int dim, bool f32, int step) {
  size_t most = 0;
  for (int n : {step, nc % step}) {
    if (n == 0) continue;
    const Product p[2] = {{nq, dim, n, f32, step < nc}, {n, dim, nq, f32}};
    most = std::max(most, products_workspace_bytes(p, 2));
  }
  return most;
}
// The rows' constants and the cleaned copies.
size_t common_bytes(int nq, int nc, int dim, bool f32) {
  return carve_bytes<LossRow>(nq) + packed_bytes(nq, dim, f32) + packed_bytes(nc, dim, f32);
}
// The forward pass above 128 dims: columns a launch, so that its parts (8 bytes a row and column tile) take at most 512 MB
// however many candidates there are, and its grid stays far below 2^32 threads.  65536 x 262144 are still one launch.
int stats_columns(int nq, int nc) {
  const int64_t most = ((int64_t)1 << 34) / nq;
  return (int)std::min<int64_t>(nc, most / 256 * 256);
}
// Its parts a row: a launch's tiles and, where there are several launches, what the ones before came to.
int stats_parts(int nq, int nc) {
  const int step = stats_columns(nq, nc);
  return score_plan(nq, step).tiles_n + (step < nc);
}
constexpr int kMostSplits = 256;
// The backward pass's workspace when it holds `step` columns of G.
size_t backward_bytes(int nq, int nc, int dim, bool f32, int step) {
  const bool chunked = step < nc;
  size_t b = f32 ? 0 : carve_bytes<float>(nq) + carve_bytes<int>(nc);  // the targets' remainders
  b += common_bytes(nq, nc, dim, f32) + packed_bytes(nq, step, f32) + carve_bytes<float>((size_t)ceil_div(nq, 64) * step);
  if (chunked) b += carve_bytes<float>((size_t)nq * ((dim + 3) & ~3));
  return b + chunk_products_bytes(nq, nc, dim, f32, step);
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

int fgpu_contrastive_loss_tile(int nq, int nc, int dim, int dtype) {
  if (check_loss(nq, nc, dim, dtype) != FGPU_OK || nq == 0) return -1;
  return dim <= kNarrowDim ? 0 : score_plan(nq, stats_columns(nq, nc)).tile;
}

size_t fgpu_contrastive_loss_workspace_bytes(int nq, int nc, int dim, int dtype) {
  if (check_loss(nq, nc, dim, dtype) != FGPU_OK || nq == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const int parts = dim <= kNarrowDim ? narrow_stats_splits(nq, nc, f32) : stats_parts(nq, nc);
  size_t b = carve_bytes<f32x2>((size_t)parts * nq) + carve_bytes<float>(nq);
  if (needs_pack(dim, f32)) b += packed_bytes(nq, dim, f32) + packed_bytes(nc, dim, f32);
  return b;
}

fgpu_status fgpu_contrastive_loss(const void* d_q, const void* d_c, const int32_t* d_target, const float* d_bias,
                                  const int32_t* d_ids, int nq, int nc, int dim, int dtype, float scale, float* d_loss,
                                  float* d_lse, void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_loss(nq, nc, dim, dtype));
  if (nq == 0) return FGPU_OK;
  FGPU_CHECK(d_q && d_c && d_target && d_loss && d_lse, FGPU_ERR_ARG, "contrastive loss: null argument");
  FGPU_CHECK(aligned16(d_q) && aligned16(d_c) && aligned16(d_workspace), FGPU_ERR_ARG,
             "contrastive loss: queries, candidates and workspace must be 16-byte aligned");
  const bool f32 = dtype == FGPU_DTYPE_F32, pk = needs_pack(dim, f32);
  const bool narrow = dim <= kNarrowDim;
  const int parts = narrow ? narrow_stats_splits(nq, nc, f32) : stats_parts(nq, nc);
  Carve ws(d_workspace, workspace_bytes);
  f32x2* part = ws.take<f32x2>((size_t)parts * nq);
  float* target2 = ws.take<float>(nq);
  char* qp = pk ? ws.take<char>(packed_bytes(nq, dim, f32)) : nullptr;
  char* cp = pk ? ws.take<char>(packed_bytes(nc, dim, f32)) : nullptr;
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "contrastive loss: workspace smaller than fgpu_contrastive_loss_workspace_bytes");
  hipStream_t s = as_stream(stream);
  GemmOperand q = as_is(d_q, dim), c = as_is(d_c, dim);
  if (pk) {
    q = packed(qp, nq, dim);
    c = packed(cp, nc, dim);
    Prep prep;
    prep.copy[0] = {d_q, nq, dim, q};
    prep.copy[1] = {d_c, nc, dim, c};
    FGPU_TRY(launch_prep(prep, f32, s));
  }
  const LossArgs a{d_bias, d_ids, d_target, scale * kLog2e, nq, nc};
  if (narrow) {
    FGPU_TRY(launch_narrow_stats(a, q, c, dim, f32, parts, part, target2, s));
    return launch_loss_join(a, part, parts, target2, d_loss, d_lse, nullptr, s);
  }
  const int step = stats_columns(nq, nc), later = step < nc;  // later: the parts begin with the columns before
  ScorePlan sp = score_plan(nq, step);
  for (int c0 = 0; c0 < nc; c0 += step) {
    const int n = std::min(step, nc - c0);
    sp.tiles_n = ceil_div(n, sp.tile);
    const StatsEpi e{a, part + (int64_t)later * nq, target2, c0};
    const GemmOperand cc{c.p + (int64_t)c0 * c.ld, c.ld, c.plane};
    FGPU_TRY(f32 ? launch_scores<6>(sp, q, cc, nq, n, dim, e, s) : launch_scores<1>(sp, q, cc, nq, n, dim, e, s));
    FGPU_TRY(launch_loss_join(a, c0 ? part : e.part, sp.tiles_n + (c0 > 0), target2, d_loss, d_lse,
                              c0 + n < nc ? part : nullptr, s));
  }
  return FGPU_OK;
}

size_t fgpu_contrastive_loss_backward_workspace_bytes(int nq, int nc, int dim, int dtype) {
  if (check_loss(nq, nc, dim, dtype) != FGPU_OK || nq == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  if (dim <= kNarrowDim) return common_bytes(nq, nc, dim, f32) + narrow_backward_bytes(nq, nc, dim, f32, kMostSplits);
  return backward_bytes(nq, nc, dim, f32, (int)most_columns(nq, nc));
}

fgpu_status fgpu_contrastive_loss_backward(const float* d_dloss, const void* d_q, const void* d_c, const int32_t* d_target,
                                           const float* d_lse, const float* d_bias, const int32_t* d_ids, int nq, int nc,
                                           int dim, int dtype, float scale, void* d_dq, void* d_dc, float* d_dbias,
                                           void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_loss(nq, nc, dim, dtype));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  if (nq == 0) {
    if (d_dc) FGPU_TRY(launch_zeros((int64_t)nc * dim, f32, d_dc, s));
    if (d_dbias) FGPU_TRY(launch_zeros(nc, true, d_dbias, s));
    return FGPU_OK;
  }
  FGPU_CHECK(d_dloss && d_q && d_c && d_target && d_lse, FGPU_ERR_ARG, "contrastive loss backward: null argument");
  FGPU_CHECK(aligned16(d_q) && aligned16(d_c) && aligned16(d_workspace), FGPU_ERR_ARG,
             "contrastive loss backward: queries, candidates and workspace must be 16-byte aligned");
  const bool narrow = dim <= kNarrowDim, copy_c = d_bias || needs_pack(dim, f32);
  int step = (int)most_columns(nq, nc), splits = kMostSplits;
  if (narrow) {
    while (splits > 1 && common_bytes(nq, nc, dim, f32) + narrow_backward_bytes(nq, nc, dim, f32, splits) > workspace_bytes)
      splits /= 2;
  } else {
    while (step > 256 && backward_bytes(nq, nc, dim, f32, step) > workspace_bytes) step = std::max(256, step / 2 / 256 * 256);
  }
  Carve ws(d_workspace, workspace_bytes);
  LossRow* rows = ws.take<LossRow>(nq);
  char* qp = ws.take<char>(packed_bytes(nq, dim, f32));
  char* cp = copy_c ? ws.take<char>(packed_bytes(nc, dim, f32)) : nullptr;
  char *np = nullptr, *gp = nullptr, *pw = nullptr;
  float *dbias_part = nullptr, *dq_sum = nullptr, *left = nullptr;
  int* owner = nullptr;
  if (narrow) {
    np = ws.take<char>(narrow_backward_bytes(nq, nc, dim, f32, splits));
  } else {
    if (!f32) left = ws.take<float>(nq);
    // Where candidates have more than four rows each, their first one's remainder is little of it, and thousands of rows
    // that ask who is first take longer than the products (8192 x 3 x 256, both gradients, 17 us; 28 with them).
    if (!f32 && d_dc && nq <= 4 * (int64_t)nc) owner = ws.take<int>(nc);
    gp = ws.take<char>(packed_bytes(nq, step, f32));
    if (d_dbias) dbias_part = ws.take<float>((size_t)ceil_div(nq, 64) * step);
    if (step < nc && d_dq) dq_sum = ws.take<float>((size_t)nq * ((dim + 3) & ~3));
    pw = ws.take<char>(chunk_products_bytes(nq, nc, dim, f32, step));
  }
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE,
             "contrastive loss backward: workspace too small for 256 columns of the score gradient (up to 128 dims: for the "
             "copies of queries and candidates)");
  const LossArgs a{d_bias, d_ids, d_target, scale * kLog2e, nq, nc};
  // Rows without a gradient and masked candidates become zero vectors: their G is zero, and what they hold (infinities
  // and NaN included) must not reach the products.
  Prep prep;
  prep.loss = {d_bias, d_target, d_lse, d_dloss, d_ids, nq, nc, rows, left, owner};
  const GemmOperand q = packed(qp, nq, dim);
  prep.copy[0] = {d_q, nq, dim, q, nullptr, true};
  GemmOperand c = as_is(d_c, dim);
  if (copy_c) {
    c = packed(cp, nc, dim);
    prep.copy[1] = {d_c, nc, dim, c, d_bias, false};
  }
  FGPU_TRY(launch_prep(prep, f32, s));
  if (narrow) return launch_narrow_backward({a, rows, q, c, dim, f32, scale, d_dq, d_dc, d_dbias}, splits, np, s);
  for (int c0 = 0; c0 < nc; c0 += step) {
    const int n = std::min(step, nc - c0);
    const GemmOperand g = packed(gp, nq, n), cc{c.p + (int64_t)c0 * c.ld, c.ld, c.plane};
    const ScorePlan sp = score_plan(nq, n);
    auto grad = [&](auto f, auto stream) -> fgpu_status {
      constexpr bool F = decltype(f)::value;
      const GradEpi<F, decltype(stream)::value> e{a, rows, const_cast<uint16_t*>(g.p), g.ld, g.plane, dbias_part, c0, n,
                                                     left, owner};
      return launch_scores<F ? 6 : 1>(sp, q, cc, nq, n, dim, e, s);
    };
    const bool past = (int64_t)nq * n * (f32 ? 6 : 2) > (int64_t)256 << 20;
    const std::true_type yes;
    const std::false_type no;
    FGPU_TRY(f32 ? (past ? grad(yes, yes) : grad(yes, no)) : (past ? grad(no, yes) : grad(no, no)));
    ColumnSum sums;
    sums.part = dbias_part, sums.parts = sp.tiles_m, sums.stride = sums.cols = n, sums.out = d_dbias ? d_dbias + c0 : nullptr;
    Finish fq, fc;
    fq.out = d_dq, fq.alpha = scale;
    fq.add = c0 > 0 ? dq_sum : nullptr;
    fq.sum = c0 + n < nc ? dq_sum : nullptr;
    if (d_dc) fc.out = static_cast<char*>(d_dc) + (int64_t)c0 * dim * (f32 ? 4 : 2);
    fc.alpha = scale;
    if (left) fq.rest = {&rows->target, sizeof(LossRow) / sizeof(int), false, left, c.p, c.ld, nc};
    if (owner) fc.rest = {owner + c0, 1, true, left, q.p, q.ld, nq};
    const ProductJob jobs[2] = {{{nq, dim, n, f32, step < nc}, g, cc, true, false, fq, d_dq != nullptr},
                                {{n, dim, nq, f32}, g, q, false, false, fc, d_dc != nullptr}};
    if (d_dq || d_dc)
      FGPU_TRY(launch_products(jobs, 2, d_dbias ? &sums : nullptr, pw, s));
    else if (d_dbias)
      FGPU_TRY(launch_column_sums(sums, nullptr, s));
  }
  return FGPU_OK;
}

}  // extern "C"

// head.hpp -- what the query head's operators share: products with a fused epilogue, packed operands, column sums.
#pragma once

#include "mfma_gemm.hpp"

namespace fgpu {

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
// HIP counts a launch's threads in 32 bits: of 2^32 and more, what passes a multiple of 2^32 runs and no error comes back
// (exact multiples are refused).  What may need that many goes out in launches of up to half of it.
constexpr int64_t kLaunchThreads = (int64_t)1 << 31;

// ---- activations -------------------------------------------------------------
// gelu(z) = z Phi(z).  The tail 1 - Phi(|z|) = erfc(x) / 2, x = |z| / sqrt(2), is t P(t) exp(-x^2) with t = 1 / (1 + c x):
// t runs through (0, 1] and erfc(x) exp(x^2) / t is smooth there, so a polynomial fitted to its least largest relative error
// up to |z| = 13 holds the tail's digits all the way out: of degree 8, c = 0.4, to 5.7e-8, a float32 last place and a half
// with its roundings; of degree 6, c = 0.51, to 7.2e-7, for bfloat16 results (2^-9 at best; degree 8 there would take 646 us
// instead of 639 at 65536 x 4096 x 1024).  Squaring z for the exponential adds 1.5 z^2 2^-24 of it.  A sum with the tail
// subtracted from one, z (1 + erf(x)) / 2, would lose the negative side's digits.  The exponential is the one that the
// derivative needs too.
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

template <class T>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  e = fast_exp2(z * z * (-0.5f * kLog2e));  // exp(-z^2 / 2)
  float p, t;
  if constexpr (sizeof(T) == 4) {
    t = fast_rcp(fmaf(0.282842726f, fabsf(z), 1.0f));
    p = fmaf(0.0200270936f, t, -0.0672089234f);
    p = fmaf(p, t, 0.0358143561f);
    p = fmaf(p, t, 0.05115458f);
    p = fmaf(p, t, 0.0348447599f);
    p = fmaf(p, t, 0.0988777131f);
    p = fmaf(p, t, 0.100375392f);
    p = fmaf(p, t, 0.113302819f);
    p = fmaf(p, t, 0.112812243f);
  } else {
    t = fast_rcp(fmaf(0.360624462f, fabsf(z), 1.0f));
    p = fmaf(0.047742594f, t, -0.181245252f);
    p = fmaf(p, t, 0.181495771f);
    p = fmaf(p, t, 0.0259678476f);
    p = fmaf(p, t, 0.140100196f);
    p = fmaf(p, t, 0.141972914f);
    p = fmaf(p, t, 0.143966064f);
  }
  const float tail = p * t * e;
  return z < 0 ? tail : 1.0f - tail;
}
__device__ __forceinline__ float sigmoid(float z) { return fast_rcp(1.0f + fast_exp2(-kLog2e * z)); }

// Of results (act_value) or operands and results (act_slope) of type T.
template <class T>
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == FGPU_ACT_RELU) return z < 0 ? 0.0f : z;
  if (act == FGPU_ACT_GELU) {
    float e;
    return z * normal_cdf<T>(z, e);
  }
  if (act == FGPU_ACT_SILU) return z * sigmoid(z);
  return z;
}
template <class T>
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == FGPU_ACT_RELU) return z > 0 ? 1.0f : 0.0f;
  if (act == FGPU_ACT_GELU) {
    float e;
    const float c = normal_cdf<T>(z, e);
    return fmaf(z * 0.39894228040143268f, e, c);
  }
  if (act == FGPU_ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return 1.0f;
}

// Both at once: the exponential is the same.
template <class T>
__device__ __forceinline__ void act_both(float z, int act, float& value, float& slope) {
  value = z, slope = 1.0f;
  if (act == FGPU_ACT_RELU) value = z < 0 ? 0.0f : z, slope = z > 0 ? 1.0f : 0.0f;
  if (act == FGPU_ACT_GELU) {
    float e;
    const float c = normal_cdf<T>(z, e);
    value = z * c, slope = fmaf(z * 0.39894228040143268f, e, c);
  }
  if (act == FGPU_ACT_SILU) {
    const float s = sigmoid(z);
    value = z * s, slope = s * fmaf(z, 1.0f - s, 1.0f);
  }
}

// ---- sums across lanes -----------------------------------------------------------
// Sum over aligned groups of N lanes (16, 32 or 64), the same bits in all of them.  Four exchanges inside a row of 16
// lanes (pairs, quads, then the mirrored half and the mirrored row, whose sums are already alike), two swaps beyond.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __int_as_float(dpp_mov<0xB1>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x4E>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x141>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x140>(__float_as_int(v)));
  if constexpr (N >= 32) v += __int_as_float(xchg<16>(__float_as_int(v)));
  if constexpr (N >= 64) v += __int_as_float(xchg<32>(__float_as_int(v)));
  return v;
}

// ---- products (head_gemm.hip) -------------------------------------------------
// What the rounding of a product's bfloat16 operand left out, added to rows of D: to row m coef[c] times row r = head[m] of
// `src` (bfloat16, rows of ld, n of it wanted), c = m, or r with `by_source`; nothing where r is not among its `rows`.  heads
// lie `step` ints apart.  head NULL: nothing at all.
struct Remainder {
  const int* head = nullptr;
  int step = 1;
  bool by_source = false;
  const float* coef = nullptr;
  const uint16_t* src = nullptr;
  int64_t ld = 0;
  int rows = 0;
  __device__ __forceinline__ int row_of(int m) const { return head ? head[(int64_t)m * step] : -1; }
  __device__ __forceinline__ bool any(int r) const { return (uint32_t)r < (uint32_t)rows; }
  __device__ __forceinline__ float coef_of(int m, int r) const { return coef[by_source ? r : m]; }
  __device__ __forceinline__ const bf16* row(int r) const { return (const bf16*)src + r * ld; }
  __device__ __forceinline__ void add4(f32x4& v, int m, int col) const {
    const int r = row_of(m);
    if (!any(r)) return;
    const float c = coef_of(m, r);
    const f32x4 x = load4(row(r) + col);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fmaf(c, x[e], v[e]);
  }
};
// What becomes of D: out = act(alpha D + bias) + residual, with the value before act in `pre`; out and residual [m][n].
struct Finish {
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* out = nullptr;
  void* pre = nullptr;
  float alpha = 1.0f;
  int act = FGPU_ACT_NONE;
  bool stream = false;  // results past the caches (launch_products decides)
  // Products added up over several calls (Product::chunked): D += add before the rest, and `sum` takes D in place of the
  // result; both [m][n rounded up to 4] float32.
  const float* add = nullptr;
  float* sum = nullptr;
  Remainder rest;  // of bfloat16 products without an activation
};

// out = act(alpha D + bias) + residual for four consecutive columns n .. n + 3 of row m (cnt of them inside).
template <class T>
__device__ __forceinline__ void finish4(const Finish& f, f32x4 v, int64_t at, int n, int cnt) {
  v *= f.alpha;
  if (f.bias) v += load4_n((const T*)f.bias + n, cnt);
  if (f.pre) store4_n((T*)f.pre + at, v, cnt);
  if (f.act != FGPU_ACT_NONE) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = act_value<T>(v[r], f.act);
  }
  if (f.residual) v += load4_n((const T*)f.residual + at, cnt);
  store4_n((T*)f.out + at, v, cnt);
}

// h = act(g) u with g and u = D's two halves + bias [2 n], for four consecutive columns col .. col + 3 of a row (cnt of
// them inside); both halves kept in `pre` [m][2 n] where wanted, h in `out` [m][n].
template <class T>
__device__ __forceinline__ void finish4_gated(const Finish& f, f32x4 g, f32x4 u, int64_t row, int n, int col, int cnt) {
  if (f.bias) {
    g += load4_n((const T*)f.bias + col, cnt);
    u += load4_n((const T*)f.bias + n + col, cnt);
  }
  if (f.pre) {
    T* pre = (T*)f.pre + row * 2 * n + col;
    store4_n(pre, g, cnt);
    store4_n(pre + n, u, cnt);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) u[r] *= act_value<T>(g[r], f.act);
  store4_n((T*)f.out + row * n + col, u, cnt);
}

// A product of m x n over k, of bf16 operands and results, or (f32) of split planes and float32 results.
struct Product {
  int m, n, k;
  bool f32;
  bool chunked = false;
};
// How a product is cut: tiles of `tile` squared, k in `splits` parts.
struct Plan {
  int tile, tiles_m, tiles_n, splits, k_per_split;
  double us;
};
// In one part; tile 0: no cut is one launch.
Plan plan_whole(const Product& p, int only_tile = 0);
// One product and where its result goes.
struct ProductJob {
  Product p;
  GemmOperand a, b;
  bool a_kc, b_kc;
  Finish f;
  bool asked = true;  // false: only planned, so that the other's plan does not depend on what is asked for
};
// out[c] = sum over the parts of part[p * stride + c], c < cols, added in a fixed order; f32 0: rounded to bf16.
struct ColumnSum {
  const float* part = nullptr;
  int parts = 0;
  int64_t stride = 0, cols = 0;
  void* out = nullptr;
  int f32 = 1;
};
// A product in parts [split][m][n rounded up to 4], to be added up and finished.
struct SplitJob {
  const float* part = nullptr;
  int m = 0, n = 0, splits = 0;
  Finish f;
};
// Up to two such products (part NULL: none) and column sums (NULL: none), in one launch.
fgpu_status launch_join(const SplitJob& a, const SplitJob& b, const ColumnSum* sums, bool f32, hipStream_t s);

// The products (one, or an input's gradient followed by a weight's, either not asked for), then what joins split products
// and the column sums (NULL: none): one launch for the products where they are small, one to join where there is something
// to join.
size_t products_workspace_bytes(const Product* p, int count);
fgpu_status launch_products(const ProductJob* jobs, int count, const ColumnSum* sums, void* ws, hipStream_t s);
double products_estimate_us(const Product* p, int count);  // the time that the rule between kernels goes by
int products_tile(const Product* p, int count, int which);  // the width of its tiles, + FGPU_TILE_PAIR if both are one launch

// An array as an operand: itself where its rows can be read as they are (bf16, cols % 8 == 0), otherwise a copy with
// rows of packed_ld(cols) elements, float32 as three planes.
__host__ __device__ inline int64_t whole8(int64_t cols) { return (cols + 7) / 8 * 8; }
// Rows begin on whole lines of 128 bytes, of which a tile's step takes one a row, where short rows' longer copies do not
// cost more than that gives (float32 gradients of a gated layer 8192 x 1000 x 1500 995 -> 767 us, 20000 x 300 x 600 355 ->
// 297, 8192 x 200 x 1030 218 -> 190, but 65536 x 72 x 100 119 -> 145; of a linear one 65536 x 385 x 771 1086 -> 851).  Rows of
// 130 to 180, padded by up to half, still gain (float32: 65536 x 130 -> 256 70 -> 64, 8192 x 180 -> 1024 39 -> 35, gradients 77
// -> 75 and 78 -> 76, a loss's over 30000 x 130 to 180 630 to 650 -> 580) but for gradients of very many rows and few columns
// (65536 x 130 -> 130 137 -> 152, -> 256 165 -> 170).  Rows a multiple of 4 KB apart fall on the same memory channels:
// 128 bytes more between them (the score gradient of 8192 x 65536 with its two products at 768 dims 2.73 -> 2.52 ms; float32
// 4096 x 2048 x 2048 forward 295 -> 279 us; 16384 x 1024 x 4096 bf16 backward 343 -> 343).
inline int64_t packed_ld(int64_t cols) {
  const int64_t ld = cols > 128 ? (cols + 63) / 64 * 64 : whole8(cols);
  return ld % 2048 ? ld : ld + 64;
}
inline bool needs_pack(int64_t cols, bool f32) { return f32 || cols % 8 != 0; }
inline size_t packed_bytes(int64_t rows, int64_t cols, bool f32) {
  return carve_bytes<uint16_t>((size_t)rows * packed_ld(cols) * (f32 ? 3 : 1));
}
inline GemmOperand as_is(const void* p, int64_t cols) { return {static_cast<const uint16_t*>(p), cols, 0}; }
inline GemmOperand packed(void* p, int64_t rows, int64_t cols) {
  return {static_cast<uint16_t*>(p), packed_ld(cols), rows * packed_ld(cols)};
}
// ---- what comes before the products, in one launch (head_prep.hip) ---------------------
// What the contrastive loss's backward pass needs of a row: lse in units of log 2, its weight, target and the target's
// document; a row without a gradient (no target, a masked one, nothing left) has weight 0, an infinite lse, so that its
// score gradient is zero, and target -1.
struct LossRow {
  float lse2, weight;
  int target, id;
};
struct LossRows {
  const float* bias;
  const int32_t* target;
  const float* lse;
  const float* dloss;
  const int32_t* ids;
  int nq, nc;
  LossRow* rows;
  // What head_loss.hip keeps of the targets' score gradients (NULL: nothing): gets zeros [nq], and INT_MAX [nc].
  float* left = nullptr;
  int* owner = nullptr;
};
// A copy of src [rows][cols] as an operand; rows that a mask takes out become zero.
struct CopyJob {
  const void* src = nullptr;
  int64_t rows = 0, cols = 0;
  GemmOperand dst{};
  const float* row_bias = nullptr;  // zero: rows whose bias masks them
  bool loss_rows = false;           // zero: rows without a gradient
};
// dz = dy act'(pre) as an operand (dst.p NULL: not stored) and the column sums of dz, part [chunk][cols] (NULL: none).
struct DzJob {
  const void* dy = nullptr;
  const void* pre = nullptr;
  int act = 0, rows = 0, cols = 0, chunks = 0;
  GemmOperand dst{};
  float* part = nullptr;
  // Of a gated layer h = act(g) u: dy is dh [rows][cols], pre [g | u] [rows][2 cols], and dz [dh u act'(g) | dh act(g)]
  // with its sums [chunk][2 cols].
  bool gated = false;
};
int dz_chunks(int rows, int cols);
struct Prep {
  CopyJob copy[2];
  DzJob dz;
  LossRows loss{};
};
fgpu_status launch_prep(const Prep& p, bool f32, hipStream_t s);

// ---- products of few tiles (head_direct.hip) ---------------------------------------
// An operand as the caller's array holds it: rows of ld elements, `count` elements in all.  With `pre`, each element is
// multiplied by the activation's slope at pre's (dz from dy).
struct DirectOperand {
  const void* p;
  int64_t ld, count;
  const void* pre;
  int up = 0;  // gated products: rows from one of the operand to the one that its product goes with
};
struct DirectJob {
  DirectOperand a, b;
  int m, n, k;
  int act;           // of `pre`
  Finish f;
  void* column_sum;  // both operands strided: gets the sums of a over k, [m] (NULL: not wanted)
};
// D = A B^T, both with k contiguous.
fgpu_status launch_direct_forward(const DirectJob& j, bool f32, hipStream_t s);
// A gated layer's: n hidden columns, b.up = n.
fgpu_status launch_direct_gated(const DirectJob& j, bool f32, hipStream_t s);
// In one launch: x (A with k contiguous, B strided), w (both strided); either may be NULL.
fgpu_status launch_direct_backward(const DirectJob* x, const DirectJob* w, bool f32, hipStream_t s);
// The times that the rule between these and the tiled products goes by.
double direct_forward_estimate_us(const Product& p);
double direct_backward_estimate_us(int rows, int in_dim, int out_dim, bool f32);

// ---- the contrastive loss of up to 128 dims (head_narrow.hip) ---------------------------
struct LossArgs {
  const float* bias;       // [nc] or NULL
  const int32_t* ids;      // [nc] or NULL
  const int32_t* target;   // [nq]
  float scale2;            // scale * log2(e)
  int nq, nc;
};
constexpr int kNarrowDim = 128;
// Forward: parts [split][nq] of (maximum, sum of exp2(s - maximum)) in units of log 2, and the targets' scores.
int narrow_stats_splits(int nq, int nc, bool f32);
fgpu_status launch_narrow_stats(const LossArgs& a, const GemmOperand& q, const GemmOperand& c, int dim, bool f32, int splits,
                                f32x2* part, float* target2, hipStream_t s);
// Backward, without holding the score gradient: each gradient forms the scores again.  dc and dbias may be NULL.
struct NarrowBackward {
  LossArgs a;
  const LossRow* rows;
  GemmOperand q, c;
  int dim;
  bool f32;
  float scale;
  void* dq;
  void* dc;
  float* dbias;
};
size_t narrow_backward_bytes(int nq, int nc, int dim, bool f32, int most_splits);
fgpu_status launch_narrow_backward(const NarrowBackward& b, int most_splits, void* ws, hipStream_t s);

// ---- column sums ---------------------------------------------------------------
// Two sums of the same length, the second one's parts `cols` after the first one's; either result may be NULL.
fgpu_status launch_column_sums(const ColumnSum& c, void* out1, hipStream_t s);
// Zeros: the sums over no rows, gradients without rows.
fgpu_status launch_zeros(int64_t count, bool f32, void* out, hipStream_t s);

}  // namespace fgpu

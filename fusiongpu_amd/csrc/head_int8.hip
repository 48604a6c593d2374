// head_int8.hip -- rows as 8-bit integers with a scale each, and the linear and the gated layer on weights held so.
//
// A row x becomes the whole numbers q = x 127 / max|x| to the nearest, ties to even, and the scale max|x| / 127: products
// of two such rows are exact in 32 bits (up to 2^16 dims), so a layer's only error is the rounding of its operands.
#include <algorithm>

#include "gated.hpp"

namespace fgpu {
namespace {

inline int int8_row(int dim) { return FGPU_INT8_ROW(dim); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---- rounding ------------------------------------------------------------------
// The quotient is rounded as the real number it is: n = rint of an approximate one, then compared with the borders, x 127
// against (n +- 1/2) max, in terms that are exact.  Both are scaled by the maximum's power of two first, so that nothing
// overflows; of float32 operands the products' low parts (t) are kept.  With n right or one beside, d = 127 x - n max is
// exact, and so is |d| - max / 2 where the two are close.
template <class T>
struct Rounder {
  float top, per;  // the maximum scaled to [1/2, 1); 127 / top
  int exp;         // its power of two
  float scale;     // what q is multiplied by to stand for x
  bool live;       // not all zeros, nothing infinite or NaN
  // bits: those of the largest magnitude.  A row that holds something not finite has a NaN scale and zeros.
  __device__ __forceinline__ explicit Rounder(uint32_t bits) {
    const float most = __uint_as_float(bits);
    live = bits != 0 && bits < 0x7f800000u;
    scale = bits < 0x7f800000u ? most / 127.0f : __uint_as_float(0x7fc00000u);
    exp = __builtin_amdgcn_frexp_expf(most);
    top = live ? ldexpf(most, -exp) : 1.0f;
    per = 127.0f / top;
  }
  __device__ __forceinline__ int round(float x) const {
    const float v = ldexpf(x, -exp), h = 127.0f * v;
    float n = rintf(v * per);
    const float p = n * top, d = h - p;
    float over = fabsf(d) - 0.5f * top;
    if constexpr (sizeof(T) == 4) {
      const float t = fmaf(127.0f, v, -h) - fmaf(n, top, -p);
      over += d < 0 ? -t : t;
    }
    const int i = (int)n;
    const bool move = over > 0 || (over == 0 && (i & 1));
    return live ? i + (move ? (d < 0 ? -1 : 1) : 0) : 0;
  }
  __device__ __forceinline__ uint32_t round4(float a, float b, float c, float d) const {
    return (uint32_t)(round(a) & 255) | (uint32_t)(round(b) & 255) << 8 | (uint32_t)(round(c) & 255) << 16 |
           (uint32_t)round(d) << 24;
  }
};
__device__ __forceinline__ uint32_t most_bits(uint32_t m, const f32x8& v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  return m;
}
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  v = max(v, (uint32_t)dpp_mov<0xB1>((int)v));
  v = max(v, (uint32_t)dpp_mov<0x4E>((int)v));
  v = max(v, (uint32_t)dpp_mov<0x141>((int)v));
  v = max(v, (uint32_t)dpp_mov<0x140>((int)v));
  if constexpr (N >= 32) v = max(v, (uint32_t)xchg<16>((int)v));
  if constexpr (N >= 64) v = max(v, (uint32_t)xchg<32>((int)v));
  return v;
}

// G threads a row (64 or a workgroup's 256), eight values each at a time; the first kHeld times stay in registers between
// the maximum and the rounding, what is behind them is read again.
constexpr int kHeld = 4;
template <class T, int G>
__global__ __launch_bounds__(256) void quantize_kernel(const T* x, int64_t rows, int dim, int8_t* q, float* scale) {
  __shared__ uint32_t part[4];
  const int at = threadIdx.x % G, width = (dim + 15) / 16 * 16, lane = threadIdx.x & 63;
  for (int64_t r = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; r < rows; r += (int64_t)gridDim.x * (256 / G)) {
    const T* row = x + r * dim;
    f32x8 held[kHeld];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int c = (at + i * G) * 8;
      held[i] = c < dim ? load8_n(row + c, dim - c) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = most_bits(most, held[i]);
    for (int c = (at + kHeld * G) * 8; c < dim; c += G * 8) most = most_bits(most, load8_n(row + c, dim - c));
    most = lanes_max<64>(most);
    if constexpr (G > 64) {
      __syncthreads();  // the last row's are read
      if (lane == 0) part[threadIdx.x / 64] = most;
      __syncthreads();
      most = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    const Rounder<T> k(most);
    if (at == 0) scale[r] = k.scale;
    int8_t* to = q + r * width;
    auto put = [&](int c, const f32x8& v) {
      *reinterpret_cast<u32x2*>(to + c) = u32x2{k.round4(v[0], v[1], v[2], v[3]), k.round4(v[4], v[5], v[6], v[7])};
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int c = (at + i * G) * 8;
      if (c < width) put(c, held[i]);
    }
    for (int c = (at + kHeld * G) * 8; c < width; c += G * 8)
      put(c, c < dim ? load8_n(row + c, dim - c) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}});
  }
}

template <class T>
fgpu_status quantize(const void* x, int64_t rows, int dim, int8_t* q, float* scale, hipStream_t s) {
  // A wave a row while what it holds covers the row and there are rows for all waves.
  const bool wave = dim <= 512 || (dim <= 64 * 8 * kHeld && rows >= 2048);
  const int grid = (int)std::min<int64_t>(wave ? (rows + 3) / 4 : rows, 256 * 32);
  if (wave) quantize_kernel<T, 64><<<grid, 256, 0, s>>>((const T*)x, rows, dim, q, scale);
  else quantize_kernel<T, 256><<<grid, 256, 0, s>>>((const T*)x, rows, dim, q, scale);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}
fgpu_status quantize(const void* x, int64_t rows, int dim, bool f32, int8_t* q, float* scale, hipStream_t s) {
  return f32 ? quantize<float>(x, rows, dim, q, scale, s) : quantize<bf16>(x, rows, dim, q, scale, s);
}

// ---- the linear layer's epilogue --------------------------------------------------
template <class T, int ACT>
struct Int8Epi {
  Finish f;
  Scales s;
  int m, n;

  template <class G>
  struct Side {
    __device__ void fetch(const Int8Epi&, int, int, int) {}
  };
  template <class G>
  __device__ __forceinline__ void finish(i32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
    f.stream ? rows<true>(acc, w) : rows<false>(acc, w);
  }
  template <bool STREAM, class G>
  __device__ __forceinline__ void rows(i32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
#pragma unroll
    for (int p = 0; p < G::FN / 2; ++p) {
      const int c = w.col(p), cnt = n - c;
      if (cnt <= 0) continue;
      const f32x8 sc = load8_n(s.col + c, cnt);
      f32x8 bias{{0, 0, 0, 0}, {0, 0, 0, 0}};
      if (f.bias) bias = load8_n((const T*)f.bias + c, cnt);
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        const int64_t row = w.row(j);
        if (row >= m) continue;
        f32x8 v = eight(acc[2 * p][j], acc[2 * p + 1][j], s.row[row], sc);
        v.lo += bias.lo, v.hi += bias.hi;
        if (ACT != FGPU_ACT_NONE) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v.set(e, act_value<T>(v[e], ACT));
        }
        if (f.residual) {
          const f32x8 r = load8_n((const T*)f.residual + row * n + c, cnt);
          v.lo += r.lo, v.hi += r.hi;
        }
        store8_n<STREAM>((T*)f.out + row * n + c, v, cnt);
      }
    }
  }
};
template <class T, int ACT>
fgpu_status run_linear(const GemmArgs& g, int tile, const Int8Epi<T, ACT>& e, hipStream_t s) {
  const int grid = g.tiles_m * g.tiles_n;
  using E = Int8Epi<T, ACT>;
  if (tile == 256) gemm_kernel<Tile256, true, true, 1, E, OfInt8><<<grid, Tile256::threads, 0, s>>>(g, e);
  else if (tile == 128) gemm_kernel<Tile128, true, true, 1, E, OfInt8><<<grid, Tile128::threads, 0, s>>>(g, e);
  else gemm_kernel<Tile64, true, true, 1, E, OfInt8><<<grid, Tile64::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

// ---- up to 16 rows: one launch ------------------------------------------------------
// A workgroup of eight waves forms 16 columns (gated: eight of each half), each wave an eighth of k, 64 a step, straight
// from the caller's arrays; with QUANT it finds the rows' maxima itself and rounds the values as they enter the products.
struct FewJob {
  const void* x;  // [m][k] of T, or 8-bit [m][ld]
  const int8_t* w;
  int m, n, k, ld;
  Scales s;
  Finish f;
};
constexpr int kFewWaves = 8, kFewThreads = kFewWaves * kWave, kFewRows = 16, kFewHeld = 2;
constexpr int kFewStep = 64;

template <class T, bool GATED, bool QUANT>
__global__ __launch_bounds__(kFewThreads) void few_rows_kernel(FewJob j) {
  __shared__ i32x4 join[kFewWaves][64];
  __shared__ uint32_t most[kFewWaves][16];
  __shared__ float row_scale[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * (GATED ? 8 : 16), i = lane & 15, kc = (lane >> 4) * 16;
  const int steps = (j.ld + kFewStep - 1) / kFewStep, per = (steps + kFewWaves - 1) / kFewWaves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  const i32x4 none = {0, 0, 0, 0};
  const int col = n0 + (GATED ? i & 7 : i);
  const int8_t* wrow = j.w + (int64_t)(GATED && (i & 8) ? col + j.n : col) * j.ld;
  auto weight = [&](int s) {
    const int k = s * kFewStep + kc;
    return col < j.n && s < s1 && k < j.ld ? *reinterpret_cast<const i32x4*>(wrow + k) : none;
  };
  i32x4 b[kFewHeld];
#pragma unroll
  for (int h = 0; h < kFewHeld; ++h) b[h] = weight(s0 + h);
  i32x4 acc = none;
  if constexpr (QUANT) {
    const T* xrow = (const T*)j.x + (int64_t)i * j.k;
    auto value = [&](int s, f32x8 (&v)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = s * kFewStep + kc + 8 * h;
        v[h] = i < j.m && s < s1 && k < j.k ? load8_n(xrow + k, j.k - k) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
      }
    };
    f32x8 a[kFewHeld][2];
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) value(s0 + h, a[h]);
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) top = most_bits(most_bits(top, a[h][0]), a[h][1]);
    for (int s = s0 + kFewHeld; s < s1; ++s) {
      f32x8 v[2];
      value(s, v);
      top = most_bits(most_bits(top, v[0]), v[1]);
    }
    top = max(top, (uint32_t)xchg<16>((int)top));
    top = max(top, (uint32_t)xchg<32>((int)top));
    if (lane < 16) most[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) top = max(top, most[w][i]);
    const Rounder<T> q(top);
    if (tid < 16) row_scale[tid] = q.scale;
    auto whole = [&](const f32x8 (&v)[2]) {
      i32x4 r;
#pragma unroll
      for (int h = 0; h < 4; ++h)
        r[h] = (int)q.round4(v[h / 2][h % 2 * 4], v[h / 2][h % 2 * 4 + 1], v[h / 2][h % 2 * 4 + 2], v[h / 2][h % 2 * 4 + 3]);
      return r;
    };
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[h], whole(a[h]), acc, 0, 0, 0);
    for (int s = s0 + kFewHeld; s < s1; ++s) {
      f32x8 v[2];
      value(s, v);
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(weight(s), whole(v), acc, 0, 0, 0);
    }
  } else {
    const int8_t* xrow = (const int8_t*)j.x + (int64_t)i * j.ld;
    auto value = [&](int s) {
      const int k = s * kFewStep + kc;
      return i < j.m && s < s1 && k < j.ld ? *reinterpret_cast<const i32x4*>(xrow + k) : none;
    };
    if (tid < 16) row_scale[tid] = tid < j.m ? j.s.row[tid] : 0.0f;
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[h], value(s0 + h), acc, 0, 0, 0);
    for (int s = s0 + kFewHeld; s < s1; ++s)
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(weight(s), value(s), acc, 0, 0, 0);
  }
  join[wave][lane] = acc;
  __syncthreads();
  // A thread four columns of a row (gated: of both halves, from the lanes 32 apart).
  if (tid >= (GATED ? 32 : 64) || (lane & 15) >= j.m) return;
  const int m = lane & 15, c = n0 + (lane >> 4) * 4, cnt = j.n - c;
  if (cnt <= 0) return;
  auto sum = [&](int l) {
    i32x4 v = join[0][l];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v += join[w][l];
    return v;
  };
  auto scaled = [&](const i32x4& v, const float* sc) {
    const f32x4 by = load4_n(sc, cnt);
    const float r = row_scale[m];
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)v[e] * r * by[e];
    return o;
  };
  if constexpr (GATED)
    finish4_gated<T>(j.f, scaled(sum(lane), j.s.col + c), scaled(sum(lane + 32), j.s.col + j.n + c), m, j.n, c, cnt);
  else
    finish4<T>(j.f, scaled(sum(lane), j.s.col + c), (int64_t)m * j.n + c, c, cnt);
}
template <class T>
fgpu_status few_rows(const FewJob& j, bool gated, bool quant, hipStream_t s) {
  const int grid = ceil_div(j.n, gated ? 8 : 16);
  if (gated)
    quant ? few_rows_kernel<T, true, true><<<grid, kFewThreads, 0, s>>>(j) : few_rows_kernel<T, true, false><<<grid, kFewThreads, 0, s>>>(j);
  else
    quant ? few_rows_kernel<T, false, true><<<grid, kFewThreads, 0, s>>>(j) : few_rows_kernel<T, false, false><<<grid, kFewThreads, 0, s>>>(j);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status check_common(int64_t rows, int in_dim, int64_t out, int dtype, int act) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "8-bit linear: unknown dtype");
  FGPU_CHECK(act >= FGPU_ACT_NONE && act <= FGPU_ACT_SILU, FGPU_ERR_ARG, "8-bit linear: unknown activation");
  FGPU_CHECK(rows >= 0 && in_dim >= 1 && out >= 1, FGPU_ERR_ARG, "8-bit linear: rows >= 0, dims >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && in_dim <= FGPU_HEAD_MAX_DIM && out <= FGPU_HEAD_MAX_DIM, FGPU_ERR_UNSUPPORTED,
             "8-bit linear: more than 2^30 rows or 2^16 dims");
  return FGPU_OK;
}
// out: weight rows.
size_t workspace_bytes_of(int64_t rows, int in_dim, int64_t out, int dtype, bool quant) {
  if (check_common(rows, in_dim, out, dtype, 0) != FGPU_OK || rows <= kFewRows || !quant) return 0;
  return carve_bytes<int8_t>((size_t)rows * int8_row(in_dim)) + carve_bytes<float>(rows);
}

template <class T>
fgpu_status run_layer(const void* x, const float* x_scale, const int8_t* w, const float* w_scale, int64_t rows, int k, int n,
                      bool gated, Finish f, void* d_ws, size_t ws_bytes, hipStream_t s) {
  const int ld = int8_row(k), out = gated ? 2 * n : n;
  const bool quant = !x_scale;
  if (rows <= kFewRows) return few_rows<T>({x, w, (int)rows, n, k, ld, {x_scale, w_scale}, f}, gated, quant, s);
  Carve ws(d_ws, ws_bytes);
  if (quant) {
    int8_t* q = ws.take<int8_t>((size_t)rows * ld);
    float* scale = ws.take<float>(rows);
    FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "8-bit linear: workspace smaller than its _workspace_bytes");
    FGPU_TRY(quantize(x, rows, k, sizeof(T) == 4, q, scale, s));
    x = q, x_scale = scale;
  }
  // Operands in units of two integers.
  const Product p{(int)rows, out, ld / 2, false};
  const Plan q = plan_product(p, false);
  FGPU_CHECK(q.tile, FGPU_ERR_UNSUPPORTED, "8-bit linear: more tiles than one launch takes (2^39 results)");
  const GemmOperand a{(const uint16_t*)x, ld / 2, 0}, b{(const uint16_t*)w, ld / 2, 0};
  const Scales sc{x_scale, w_scale};
  if (gated) return run_gated<1, OfInt8, T>(a, b, (int64_t)n * b.ld, p.m, n, p.k, q, f, sc, s);
  const GemmArgs g{a, b, p.m, n, p.k, q.tiles_m, q.tiles_n, 1, ceil_div(p.k, kGemmBK) * kGemmBK};
  f.stream = past_caches(rows * n * (int64_t)sizeof(T));
  switch (f.act) {
    case FGPU_ACT_NONE: return run_linear(g, q.tile, Int8Epi<T, FGPU_ACT_NONE>{f, sc, p.m, n}, s);
    case FGPU_ACT_RELU: return run_linear(g, q.tile, Int8Epi<T, FGPU_ACT_RELU>{f, sc, p.m, n}, s);
    case FGPU_ACT_GELU: return run_linear(g, q.tile, Int8Epi<T, FGPU_ACT_GELU>{f, sc, p.m, n}, s);
    default: return run_linear(g, q.tile, Int8Epi<T, FGPU_ACT_SILU>{f, sc, p.m, n}, s);
  }
}

fgpu_status layer(const void* d_x, const float* d_x_scale, const void* d_w, const float* d_w_scale, const void* d_bias,
                  const void* d_residual, int64_t rows, int in_dim, int n, bool gated, int dtype, int act, void* d_y,
                  void* d_ws, size_t ws_bytes, void* stream) {
  FGPU_TRY(check_common(rows, in_dim, gated ? 2 * (int64_t)n : n, dtype, act));
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_w && d_w_scale && d_y, FGPU_ERR_ARG, "8-bit linear: null x, weight, scales or output");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_ws), FGPU_ERR_ARG,
             "8-bit linear: x, weight and workspace must be 16-byte aligned");
  Finish f;
  f.bias = d_bias, f.residual = d_residual, f.out = d_y, f.act = act;
  const int8_t* w = (const int8_t*)d_w;
  hipStream_t s = as_stream(stream);
  if (dtype == FGPU_DTYPE_F32) return run_layer<float>(d_x, d_x_scale, w, d_w_scale, rows, in_dim, n, gated, f, d_ws, ws_bytes, s);
  return run_layer<bf16>(d_x, d_x_scale, w, d_w_scale, rows, in_dim, n, gated, f, d_ws, ws_bytes, s);
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

fgpu_status fgpu_quantize_rows(const void* d_x, int64_t rows, int dim, int dtype, int8_t* d_q, float* d_scale, void* stream) {
  FGPU_TRY(check_common(rows, dim, 1, dtype, 0));
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_q && d_scale, FGPU_ERR_ARG, "quantize: null x, values or scales");
  FGPU_CHECK(aligned16(d_q), FGPU_ERR_ARG, "quantize: the values must be 16-byte aligned");
  return quantize(d_x, rows, dim, dtype == FGPU_DTYPE_F32, d_q, d_scale, as_stream(stream));
}

size_t fgpu_linear_int8_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype, int quantized_x) {
  return workspace_bytes_of(rows, in_dim, out_dim, dtype, !quantized_x);
}
fgpu_status fgpu_linear_int8(const void* d_x, const float* d_x_scale, const int8_t* d_w, const float* d_w_scale,
                             const void* d_bias, const void* d_residual, int64_t rows, int in_dim, int out_dim, int dtype,
                             int act, void* d_y, void* d_workspace, size_t workspace_bytes, void* stream) {
  return layer(d_x, d_x_scale, d_w, d_w_scale, d_bias, d_residual, rows, in_dim, out_dim, false, dtype, act, d_y, d_workspace,
               workspace_bytes, stream);
}

size_t fgpu_gated_linear_int8_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype, int quantized_x) {
  return workspace_bytes_of(rows, in_dim, 2 * (int64_t)hidden, dtype, !quantized_x);
}
fgpu_status fgpu_gated_linear_int8(const void* d_x, const float* d_x_scale, const int8_t* d_w, const float* d_w_scale,
                                   const void* d_bias, int64_t rows, int in_dim, int hidden, int dtype, int act, void* d_h,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
  return layer(d_x, d_x_scale, d_w, d_w_scale, d_bias, nullptr, rows, in_dim, hidden, true, dtype, act, d_h, d_workspace,
               workspace_bytes, stream);
}

}  // extern "C"

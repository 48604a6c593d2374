// head_int8.hip -- rows as 8-bit integers with a scale each, and the linear and the gated layer on weights held so.
//
// A row x becomes the whole numbers q = x 127 / max|x| to the nearest, ties to even, and the scale max|x| / 127: products
// of two such rows are exact in 32 bits (up to 2^16 dims), so a layer's only error is the rounding of its operands.
//
// Rounding is bound by HBM: 100003 x 1024 in bfloat16 67 us (307 MB, 4.6 TB/s).  The gated layer on 65536 x 1024 -> 4096
// takes 0.62 to 0.65 ms, 0.05 of them rounding (the product 1.9 POP/s, the matrix units busy 39 % of its cycles; the library's
// plain product of 8192^3 2.4): eight steps of 128 k a tile, then an epilogue of two conversions, four products, an exponential
// and a reciprocal an element that nothing overlaps.  One row x 1024 -> 4096: 5.2 us, a launch, the row's
// maximum and a round of loads.
#include <algorithm>

#include "gated.hpp"

namespace fgpu {
namespace {

inline int int8_row(int dim) { return FGPU_INT8_ROW(dim); }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---- rounding ------------------------------------------------------------------
// The quotient x 127 / max is rounded as the real number it is.  n, from a product with 127 / max rounded, is the nearest whole
// number or, beside a border between two, one of both; d = 127 x - n max says which: it is exact (of float32 operands its low
// part t is kept apart), and n is right unless 2 |d| > max, or 2 |d| = max and n is odd.  Few groups of eight hold a value so
// near a border (float32: one in 2000; bfloat16, mostly ties with half the maximum: one in 30 to 300): the others take one
// multiplication, a fused one that adds 1.5 2^23 and so leaves n in the sum's low bits, and two to see that.
template <class T>
struct Rounder {
  static constexpr float kWhole = 12582912.0f;  // 1.5 2^23
  float most;   // the largest magnitude, scaled into [1/2, 1) where it lies near an end of the type
  float per;    // 127 / most
  float near;   // |d| below it: n is right
  float scale;  // what q is multiplied by to stand for x
  int exp;      // the power of two that x is scaled by
  uint32_t keep;  // zero where everything becomes zero
  // bits: those of the largest magnitude.  A row that holds something not finite has a NaN scale and zeros.
  __device__ __forceinline__ explicit Rounder(uint32_t bits) {
    const float top = __uint_as_float(bits);
    const bool live = bits != 0 && bits < 0x7f800000u;
    scale = bits < 0x7f800000u ? top / 127.0f : __uint_as_float(0x7fc00000u);
    keep = live ? ~0u : 0u;
    exp = live && (top < 0x1p-100f || top > 0x1p100f) ? -__builtin_amdgcn_frexp_expf(top) : 0;
    most = exp ? ldexpf(top, exp) : top;
    per = live ? 127.0f / most : 0.0f;
    near = sizeof(T) == 4 ? 0.4999f * most : 0.5f * most;
    if (!live) most = near = INFINITY;  // no d is looked at
  }
  __device__ __forceinline__ u32x2 round8(f32x8 x) const {
    if (exp) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x.set(e, ldexpf(x[e], exp));
    }
    float n[8], d[8], far = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      n[e] = fmaf(x[e], per, kWhole);
      d[e] = fmaf(kWhole - n[e], most, 127.0f * x[e]);
      far = fmaxf(far, fabsf(d[e]));
    }
    if (far >= near) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float over = fabsf(d[e]) - 0.5f * most;
        if constexpr (sizeof(T) == 4) {  // d again, from both parts of both products
          const float h = 127.0f * x[e], w = n[e] - kWhole, p = w * most, c = h - p;
          const float t = fmaf(127.0f, x[e], -h) - fmaf(w, most, -p);
          over = fabsf(c) - 0.5f * most + (c < 0 ? -t : t);
        }
        const bool move = over > 0 || (over == 0 && (__float_as_uint(n[e]) & 1));
        if (move) n[e] += d[e] < 0 ? -1.0f : 1.0f;
      }
    }
    u32x2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // the low bytes
      const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(n[4 * h + 1]), __float_as_uint(n[4 * h]), 0x0c0c0400u);
      const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(n[4 * h + 3]), __float_as_uint(n[4 * h + 2]), 0x04000c0cu);
      out[h] = (a | b) & keep;
    }
    return out;
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
      *reinterpret_cast<u32x2*>(to + c) = k.round8(v);
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
    if constexpr (sizeof(T) == 2 && G::FN == 4) {
      if (w.first_col() + 64 <= n) return lines<STREAM>(acc, w);
    }
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
        const f32x8 v = value(acc[2 * p][j], acc[2 * p + 1][j], s.row[row], sc, bias, row * n + c, cnt);
        store8_n<STREAM>((T*)f.out + row * n + c, v, cnt);
      }
    }
  }
  // The same where a wave's 64 columns all lie inside: whole lines a store (65536 x 2048 over k 256 138 -> 123 us,
  // 8192 x 8192 over k 1024 102 -> 96).
  template <bool STREAM, class G>
  __device__ __forceinline__ void lines(i32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    f32x8 sc[2], bias[2] = {{{0, 0, 0, 0}, {0, 0, 0, 0}}, {{0, 0, 0, 0}, {0, 0, 0, 0}}};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      sc[p] = load8(s.col + w.col(p));
      if (f.bias) bias[p] = load8((const T*)f.bias + w.col(p));
    }
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      const int64_t row = w.m0 + (w.wm * G::FM + j) * 16, mine = row + (w.lane & 15);
      const int inside = (int)min((int64_t)16, m - row);
      if (inside <= 0) break;
      f32x8 v[2] = {bias[0], bias[1]};
      if (mine < m) {
        const float scale = s.row[mine];
#pragma unroll
        for (int p = 0; p < 2; ++p)
          v[p] = value(acc[2 * p][j], acc[2 * p + 1][j], scale, sc[p], bias[p], mine * n + w.col(p), 8);
      }
      store_lines<STREAM>((T*)f.out + row * n + w.first_col(), n, w.lane, inside, v[0], v[1]);
    }
  }
  __device__ __forceinline__ f32x8 value(const i32x4& lo, const i32x4& hi, float row, const f32x8& col, const f32x8& bias,
                                         int64_t at, int cnt) const {
    f32x8 v = eight(lo, hi, row, col, bias);
    if (ACT != FGPU_ACT_NONE) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.set(e, act_value<T>(v[e], ACT));
    }
    if (f.residual) {
      const f32x8 r = load8_n((const T*)f.residual + at, cnt);
      v.lo += r.lo, v.hi += r.hi;
    }
    return v;
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
// Four columns of a row with their scales and bias, in the steps of the tiles' epilogues (`eight`): a row's bits are the same
// whichever kernel its batch takes.
struct Four {
  f32x4 by = {0, 0, 0, 0}, bias = {0, 0, 0, 0};
  template <class T>
  __device__ __forceinline__ void load(const FewJob& j, int at, int cnt) {
    by = load4_n(j.s.col + at, cnt);
    if (j.f.bias) bias = load4_n((const T*)j.f.bias + at, cnt);
  }
  __device__ __forceinline__ f32x4 of(const i32x4& v, float row) const {
    f32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf((float)v[e] * by[e], row, bias[e]);
    return o;
  }
};
// The rest of the epilogue, g and u (or the only one, g) scaled and with their bias.
template <class T, bool GATED>
__device__ __forceinline__ void finish_four(Finish f, const f32x4& g, const f32x4& u, int64_t row, int n, int col, int cnt) {
  f.bias = nullptr;
  if constexpr (GATED) finish4_gated<T>(f, g, u, row, n, col, cnt);
  else finish4<T>(f, g, row * n + col, col, cnt);
}

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
      const u32x2 lo = q.round8(v[0]), hi = q.round8(v[1]);
      return i32x4{(int)lo[0], (int)lo[1], (int)hi[0], (int)hi[1]};
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
  // A thread four columns of a row (gated: of both halves, from the lanes 32 apart).
  const int m = lane & 15, c = n0 + (lane >> 4) * 4, cnt = j.n - c;
  const bool mine = tid < (GATED ? 32 : 64) && m < j.m && cnt > 0;
  Four g4, u4;
  if (mine) {  // on the way while the waves meet
    g4.load<T>(j, c, cnt);
    if (GATED) u4.load<T>(j, j.n + c, cnt);
  }
  __syncthreads();
  if (!mine) return;
  auto sum = [&](int l) {
    i32x4 v = join[0][l];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) v += join[w][l];
    return v;
  };
  const f32x4 g = g4.of(sum(lane), row_scale[m]), u = GATED ? u4.of(sum(lane + 32), row_scale[m]) : g;
  finish_four<T, GATED>(j.f, g, u, m, j.n, c, cnt);
}
template <class T>
fgpu_status few_rows(const FewJob& j, bool gated, bool quant, hipStream_t s) {
  const int grid = ceil_div(j.n, gated ? 8 : 16);
  if (gated)
    quant ? few_rows_kernel<T, true, true><<<grid, kFewThreads, 0, s>>>(j)
          : few_rows_kernel<T, true, false><<<grid, kFewThreads, 0, s>>>(j);
  else
    quant ? few_rows_kernel<T, false, true><<<grid, kFewThreads, 0, s>>>(j)
          : few_rows_kernel<T, false, false><<<grid, kFewThreads, 0, s>>>(j);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

// ---- some hundred rows: one launch ----------------------------------------------------
// A workgroup rounds its 32 rows of x into LDS, whole, and then eight waves form 128 columns (gated: 64 of each half) from
// there and from the weight as it lies, whose first steps are on the way meanwhile.  Every column of workgroups rounds the rows
// again: up to one workgroup a CU and 512 k that takes the GPU as long as rounding in a launch of its own (float32 1000 x 385 x
// 771 9.0 us and 9.3; bfloat16 128 x 512 x 2048 9.9 and 8.2; with 1024 k 12 and 10), and the caller a launch and a workspace
// less, which is what calls of this size wait for (15 us a call and 10).
constexpr int kPanelRows = 32, kPanelK = 512, kPanelWaves = 8, kPanelThreads = kPanelWaves * kWave;
__host__ __device__ constexpr int panel_stride(int ld) { return (ld / 16 | 1) * 16; }  // rows fall on different banks

template <class T, bool GATED>
__global__ __launch_bounds__(kPanelThreads) void panel_kernel(FewJob j) {
  __shared__ __attribute__((aligned(16))) char rows[kPanelRows * panel_stride(kPanelK)];
  __shared__ float row_scale[kPanelRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int across = (j.n + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
  const int m0 = blockIdx.x / across * kPanelRows, n0 = blockIdx.x % across * (GATED ? 64 : 128);
  const int i = lane & 15, kc = (lane >> 4) * 16, stride = panel_stride(j.ld), steps = (j.ld + kFewStep - 1) / kFewStep;
  const i32x4 none = {0, 0, 0, 0};
  const int first = n0 + wave * (GATED ? 8 : 16), col = first + (GATED ? i & 7 : i);
  const int8_t* wrow = j.w + (int64_t)(GATED && (i & 8) ? col + j.n : col) * j.ld;
  auto weight = [&](int s) {
    const int k = s * kFewStep + kc;
    return col < j.n && k < j.ld ? *reinterpret_cast<const i32x4*>(wrow + k) : none;
  };
  constexpr int kAhead = 8;
  i32x4 b[kAhead];
#pragma unroll
  for (int h = 0; h < kAhead; ++h) b[h] = weight(h);
  {
    constexpr int G = kPanelThreads / kPanelRows, held = kPanelK / 8 / G;  // 16 lanes a row
    const int r = tid / G, at = tid % G, row = m0 + r;
    const T* x = (const T*)j.x + (int64_t)row * j.k;
    f32x8 v[held];
    uint32_t most = 0;
#pragma unroll
    for (int h = 0; h < held; ++h) {
      const int c = (at + h * G) * 8;
      v[h] = row < j.m && c < j.k ? load8_n(x + c, j.k - c) : f32x8{{0, 0, 0, 0}, {0, 0, 0, 0}};
    }
#pragma unroll
    for (int h = 0; h < held; ++h) most = most_bits(most, v[h]);
    const Rounder<T> q(lanes_max<16>(most));
    if (at == 0) row_scale[r] = q.scale;
    char* to = rows + r * stride;
#pragma unroll
    for (int h = 0; h < held; ++h) {
      const int c = (at + h * G) * 8;
      if (c < j.ld) *reinterpret_cast<u32x2*>(to + c) = q.round8(v[h]);
    }
  }
  __syncthreads();
  i32x4 acc[2] = {none, none};
  auto work = [&](int s, const i32x4& w) {
    const int k = s * kFewStep + kc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x4 a = k < j.ld ? *reinterpret_cast<const i32x4*>(rows + (16 * h + i) * stride + k) : none;
      acc[h] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, a, acc[h], 0, 0, 0);
    }
  };
  for (int s = 0; s < steps; s += kAhead) {
    i32x4 now[kAhead];
#pragma unroll
    for (int h = 0; h < kAhead; ++h) now[h] = b[h];
#pragma unroll
    for (int h = 0; h < kAhead; ++h) b[h] = weight(s + kAhead + h);
#pragma unroll
    for (int h = 0; h < kAhead; ++h) work(s + h, now[h]);  // past the end: zeros
  }
  const int c = first + (lane >> 4) * 4, cnt = j.n - c;
  Four g4, u4;
  if (cnt > 0 && !(GATED && lane >= 32)) {
    g4.load<T>(j, c, cnt);
    if (GATED) u4.load<T>(j, j.n + c, cnt);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int m = 16 * h + i;
    i32x4 other = none;
    if constexpr (GATED) {
#pragma unroll
      for (int e = 0; e < 4; ++e) other[e] = xchg<32>(acc[h][e]);
    }
    if (m0 + m >= j.m || cnt <= 0 || (GATED && lane >= 32)) continue;
    const f32x4 g = g4.of(acc[h], row_scale[m]), u = GATED ? u4.of(other, row_scale[m]) : g;
    finish_four<T, GATED>(j.f, g, u, m0 + m, j.n, c, cnt);
  }
}
bool takes_panel(int64_t rows, int k, int n, bool gated) {
  return k <= kPanelK && (rows + kPanelRows - 1) / kPanelRows * ceil_div(n, gated ? 64 : 128) <= 256;
}
template <class T>
fgpu_status panel(const FewJob& j, bool gated, hipStream_t s) {
  const int grid = ceil_div(j.m, kPanelRows) * ceil_div(j.n, gated ? 64 : 128);
  gated ? panel_kernel<T, true><<<grid, kPanelThreads, 0, s>>>(j) : panel_kernel<T, false><<<grid, kPanelThreads, 0, s>>>(j);
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
size_t workspace_bytes_of(int64_t rows, int in_dim, int n, bool gated, int dtype, bool quant) {
  if (check_common(rows, in_dim, gated ? 2 * (int64_t)n : n, dtype, 0) != FGPU_OK || !quant) return 0;
  if (rows <= kFewRows || takes_panel(rows, in_dim, n, gated)) return 0;
  return carve_bytes<int8_t>((size_t)rows * int8_row(in_dim)) + carve_bytes<float>(rows);
}

template <class T>
fgpu_status run_layer(const void* x, const float* x_scale, const int8_t* w, const float* w_scale, int64_t rows, int k, int n,
                      bool gated, Finish f, void* d_ws, size_t ws_bytes, hipStream_t s) {
  const int ld = int8_row(k), out = gated ? 2 * n : n;
  const bool quant = !x_scale;
  if (rows <= kFewRows) return few_rows<T>({x, w, (int)rows, n, k, ld, {x_scale, w_scale}, f}, gated, quant, s);
  if (quant && takes_panel(rows, k, n, gated)) return panel<T>({x, w, (int)rows, n, k, ld, {nullptr, w_scale}, f}, gated, s);
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
  const Plan q = plan_whole(p);
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
  if (dtype == FGPU_DTYPE_F32)
    return run_layer<float>(d_x, d_x_scale, w, d_w_scale, rows, in_dim, n, gated, f, d_ws, ws_bytes, s);
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
  return workspace_bytes_of(rows, in_dim, out_dim, false, dtype, !quantized_x);
}
fgpu_status fgpu_linear_int8(const void* d_x, const float* d_x_scale, const int8_t* d_w, const float* d_w_scale,
                             const void* d_bias, const void* d_residual, int64_t rows, int in_dim, int out_dim, int dtype,
                             int act, void* d_y, void* d_workspace, size_t workspace_bytes, void* stream) {
  return layer(d_x, d_x_scale, d_w, d_w_scale, d_bias, d_residual, rows, in_dim, out_dim, false, dtype, act, d_y, d_workspace,
               workspace_bytes, stream);
}

size_t fgpu_gated_linear_int8_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype, int quantized_x) {
  return workspace_bytes_of(rows, in_dim, hidden, true, dtype, !quantized_x);
}
fgpu_status fgpu_gated_linear_int8(const void* d_x, const float* d_x_scale, const int8_t* d_w, const float* d_w_scale,
                                   const void* d_bias, int64_t rows, int in_dim, int hidden, int dtype, int act, void* d_h,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
  return layer(d_x, d_x_scale, d_w, d_w_scale, d_bias, nullptr, rows, in_dim, hidden, true, dtype, act, d_h, d_workspace,
               workspace_bytes, stream);
}

}  // extern "C"

// head_ortho.hip -- an update with its singular values drawn to one, by Newton-Schulz products.
//
// X_0 = x / (|x| + eps) in the Frobenius norm; each step forms the products of the shorter side, A = X X^T (or X^T X),
// P = a I + b A + c A^2, and X <- P X (or X P): every singular value s becomes a s + b s^3 + c s^5, the vectors stay.
//
// Between the products X, A and P are held as two float16 planes, 2^10 times their value: h + l is good to 2^-23 of what
// lies above 2^-25 of one, and all of them stay below 2^6 while the singular values stay below about two.  The steps
// multiply a small singular value by up to a each, and with it whatever a rounding leaves in its directions, so none of them
// may be rounded to one plane of 8 or 11 bits, of bfloat16 updates either: one plane in A, and in P and X' of the first and last
// two steps, took 8192 x 1024 from 550 to 370 us and put results up to 9e-3 of their norm off at five steps and 1.8e-2 at eight
// (updates of few rows that are not zero; sparse ones 5e-3, of low rank 2e-3), where two planes leave at most 6e-5.
//
// 8192 x 1024, five steps, takes 0.55 to 0.57 ms in either type; traced, A 36 to 41 us a step as thirteen parts of its triangle
// (strided operands, the matrix units busy 30 %) and 8 to join them, P 16, X' 57 to 65 (three products, 0.8 to 0.9 PFLOP/s of
// them, the matrix units busy 38 %), norm and start 19.  128 x 771 in float32 65 us: twelve launches, a step's two 6 each: A (k
// over sixteen waves; in parts 8.3), then P and X'.
#include <algorithm>
#include <cmath>

#include "gated.hpp"

namespace fgpu {
namespace {

constexpr float kHeld = 1024.0f;  // what planes hold of a value of one
constexpr int kNormBlocks = 512;
constexpr int kPairs = 3, kPlanes = planes_of(kPairs);  // plane products of a product

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
__device__ __forceinline__ void to_planes(const f32x8& v, f16x8& h, f16x8& l) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = (_Float16)v[e];
    l[e] = (_Float16)(v[e] - (float)h[e]);
  }
}
__device__ __forceinline__ void put_planes8(const Planes& a, int64_t at, const f32x8& v) {
  f16x8 h, l;
  to_planes(v, h, l);
  *reinterpret_cast<f16x8*>(a.p + at) = h;
  *reinterpret_cast<f16x8*>(a.p + a.plane + at) = l;
}

// ---- the start: the norm, and X_0 ----------------------------------------------------
template <class T>
__global__ __launch_bounds__(256) void norm_parts_kernel(const T* x, int64_t count, double* part) {
  __shared__ double sum[256];
  double v = 0;
#pragma unroll 4
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
__global__ __launch_bounds__(256) void start_kernel(const T* x, int64_t rows, int cols, const double* part, int parts,
                                                    float eps, Planes out) {
  double v = 0;  // each wave adds all parts, in the same order
#pragma unroll 8
  for (int i = threadIdx.x & 63; i < kNormBlocks; i += kWave) v += i < parts ? part[i] : 0;
#pragma unroll
  for (int h = 32; h > 0; h >>= 1) v += __shfl_xor(v, h, kWave);
  const double norm = sqrt(v) + eps;
  // Something not finite makes everything NaN; nothing but zeros stays zero.
  const double by = !(norm < INFINITY) ? (double)NAN : norm > 0 ? kHeld / norm : 0;
  // In float32 where the factor is far from the ends of the type.
  const float by32 = by > 1e-30 && by < 1e30 ? (float)by : 0.0f;
  const uint32_t per = (uint32_t)(whole8(cols) / 8);
  const uint64_t total = rows * (uint64_t)per;
#pragma unroll 2
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const int64_t r = total < (1ull << 32) ? (uint32_t)i / per : i / per;
    const int c = (int)(i - r * (uint64_t)per) * 8;
    const f32x8 q = load8_n(x + r * cols + c, cols - c);
    f32x8 o;
    if (by32 != 0) {
      o = {q.lo * by32, q.hi * by32};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o.set(e, c + e < cols ? (float)(q[e] * by) : 0.0f);
    }
    put_planes8(out, r * out.ld + c, o);
  }
}

// ---- the products ------------------------------------------------------------------
// alpha D + beta C + diagonal I, as planes or (out) as the result.
struct OrthoFinish {
  float alpha = 0, beta = 0, diagonal = 0;
  Planes c, to;
  void* out = nullptr;
  int m = 0, n = 0;
  __device__ __forceinline__ f32x8 value(f32x8 v, int64_t row, int col, bool inside) const {
    v.lo *= alpha, v.hi *= alpha;
    if (c.p && inside) {
      const f32x8 o = planes8(c, row * c.ld + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) v.set(e, fmaf(beta, o[e], v[e]));
    }
    if (diagonal != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v.set(e, v[e] + (row == col + e ? diagonal : 0.0f));
    }
    return v;
  }
  template <class T>
  __device__ __forceinline__ void put(f32x8 v, int64_t row, int col) const {
    v = value(v, row, col, true);
    if (out) store8_n<false>((T*)out + row * n + col, v, n - col);
    else put_planes8(to, row * to.ld + col, v);
  }
};
template <class T>
struct OrthoEpi {
  OrthoFinish f;

  template <class G>
  struct Side {
    __device__ void fetch(const OrthoEpi&, int, int, int) {}
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
    const int n8 = (f.n + 7) & ~7;
    if constexpr (G::FN == 4) {
      if (w.first_col() + 64 <= f.n && (sizeof(T) == 2 || !f.out)) return lines(acc, w);
    }
#pragma unroll
    for (int p = 0; p < G::FN / 2; ++p) {
      const int col = w.col(p);
      if (col >= n8) continue;
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        const int64_t row = w.row(j);
        if (row < f.m) f.put<T>(f32x8{acc[2 * p][j], acc[2 * p + 1][j]}, row, col);
      }
    }
  }
  // The same where a wave's 64 columns all lie inside: whole lines a store.
  template <class G>
  __device__ __forceinline__ void lines(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      const int64_t row = w.m0 + (w.wm * G::FM + j) * 16, mine = row + (w.lane & 15);
      const int inside = (int)min((int64_t)16, f.m - row);
      if (inside <= 0) break;
      f32x8 v[2];
#pragma unroll
      for (int p = 0; p < 2; ++p)
        v[p] = f.value(f32x8{acc[2 * p][j], acc[2 * p + 1][j]}, mine, w.col(p), mine < f.m);
      if (sizeof(T) == 2 && f.out) {
        store_lines<false>((bf16*)f.out + row * f.n + w.first_col(), f.n, w.lane, inside, v[0], v[1]);
        continue;
      }
      f16x8 h[2], l[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) to_planes(v[p], h[p], l[p]);
      uint16_t* at = f.to.p + row * f.to.ld + w.first_col();
      store_lines<false>(at, f.to.ld, w.lane, inside, __builtin_bit_cast(u32x4, h[0]), __builtin_bit_cast(u32x4, h[1]));
      store_lines<false>(at + f.to.plane, f.to.ld, w.lane, inside, __builtin_bit_cast(u32x4, l[0]),
                         __builtin_bit_cast(u32x4, l[1]));
    }
  }
};
// A symmetric product's tiles on and below the diagonal as they are, [split][tile][row][column].
struct TriangleEpi {
  float* part;
  int tiles;

  template <class G>
  struct Side {
    __device__ void fetch(const TriangleEpi&, int, int, int) {}
  };
  template <class G>
  __device__ __forceinline__ void finish(f32x4 (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
    float* tile = part + ((int64_t)w.sp * tiles + triangle_tiles(w.tm) + w.tn) * (G::BM * G::BN);
#pragma unroll
    for (int p = 0; p < G::FN / 2; ++p)
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        float* d = tile + (w.row(j) - w.m0) * G::BN + w.col(p) - w.n0;
        *reinterpret_cast<f32x4*>(d) = acc[2 * p][j];
        *reinterpret_cast<f32x4*>(d + 4) = acc[2 * p + 1][j];
      }
  }
};
// Their parts added in their order and finished, as planes on both sides of the diagonal: a workgroup 64 x 64, which it turns
// in LDS.
__global__ __launch_bounds__(256) void triangle_join_kernel(OrthoFinish f, const float* part, int splits, int tiles, int tile) {
  __shared__ float turned[64][65];
  const int side = tile / 64, patch = blockIdx.x % (side * side), t = blockIdx.x / (side * side);
  int tm, tn;
  triangle_at(t, tm, tn);
  const int pm = patch / side, pn = patch % side, r0 = tm * tile + pm * 64, c0 = tn * tile + pn * 64;
  if (c0 > r0 || r0 >= f.n) return;  // in a tile on the diagonal; beyond the matrix
  const int n8 = (f.n + 7) & ~7, c = threadIdx.x % 8 * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = threadIdx.x / 8 + 32 * h;
    f32x8 v{{0, 0, 0, 0}, {0, 0, 0, 0}};
    const float* at = part + (int64_t)t * tile * tile + (pm * 64 + r) * tile + pn * 64 + c;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const f32x8 q = load8(at + (int64_t)s * tiles * tile * tile);
      v.lo += q.lo, v.hi += q.hi;
    }
    v = f.value(v, r0 + r, c0 + c, r0 + r < f.n && c0 + c < n8);
    if (r0 + r < f.n && c0 + c < n8) put_planes8(f.to, (int64_t)(r0 + r) * f.to.ld + c0 + c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) turned[c + e][r] = v[e];
  }
  if (c0 == r0) return;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = threadIdx.x / 8 + 32 * h;
    if (c0 + r >= f.n || r0 + c >= n8) continue;
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.set(e, turned[r][c + e]);
    put_planes8(f.to, (int64_t)(c0 + r) * f.to.ld + r0 + c, v);
  }
}

// Few tiles: eight or sixteen waves share 32 x 32, each with its part of k and its fragments straight from the planes (whose
// ends are zeros), as in head_direct.hpp; the partial tiles meet in LDS.  One launch, no parts in memory.
constexpr int kFewTile = 32, kFewBK = 32;
inline int few_waves(int k) { return k > 512 ? 16 : 8; }
// Half the rows a workgroup while that leaves CUs without one.
inline bool few_half(int m, int n) { return (int64_t)ceil_div(m, 16) * ceil_div(n, kFewTile) <= 256; }
template <bool KC, bool ISB, int F = 2>
struct FewRead {
  static constexpr int P = kPlanes, lds_bytes = KC ? 0 : P * kFewBK * F * 32;
  bf16x8 r[P][F];
  __device__ __forceinline__ void load(const Planes& o, int r0, int nr, int k0, int nk, int lane) {
#pragma unroll
    for (int i = 0; i < F; ++i) {
      int64_t at;
      bool in;
      if constexpr (KC) {
        const int l = lane & 15, row = r0 + (ISB ? 8 * (l >> 2) + 4 * i + (l & 3) : 16 * i + l), k = k0 + 8 * (lane >> 4);
        at = row * o.ld + k, in = row < nr && k < nk;
      } else {
        const int t = lane + kWave * i, k = k0 + t / (2 * F), col = r0 + t % (2 * F) * 8;
        at = k * o.ld + col, in = k < nk && col < nr;
      }
#pragma unroll
      for (int p = 0; p < P; ++p)
        r[p][i] = in ? *reinterpret_cast<const bf16x8*>(o.p + p * o.plane + at) : bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  // Strided: through the wave's own LDS and its transposing load.
  __device__ __forceinline__ void frags(bf16x8 (&f)[F][P], char* lds, int lane) const {
    if constexpr (KC) {
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < F; ++i) f[i][p] = r[p][i];
    } else {
      typedef __attribute__((address_space(3))) s16x4 lds_half;
      constexpr int row_bytes = F * 32;
      wave_lds_order();
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < F; ++i)
          *reinterpret_cast<bf16x8*>(lds + p * kFewBK * row_bytes + (lane + kWave * i) * 16) = r[p][i];
      wave_lds_order();
      const int l = lane & 15, g = lane >> 4;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < F; ++i) {
          char* at = lds + (p * kFewBK + 8 * g + (l >> 2)) * row_bytes + (ISB ? (l & 3) * 16 + i * 8 : i * 32 + (l & 3) * 8);
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds_char*)at);
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds_char*)(at + 4 * row_bytes));
          const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          f[i][p] = __builtin_bit_cast(bf16x8, v);
        }
      wave_lds_order();
    }
  }
};
template <class T, bool AKC, bool BKC, int kFewWaves, int FM>
__global__ __launch_bounds__(kFewWaves * kWave) void few_tiles_kernel(Planes a, Planes b, int k, OrthoFinish f) {
  using RA = FewRead<AKC, false, FM>;
  using RB = FewRead<BKC, true>;
  constexpr int stage = kFewWaves * (RA::lds_bytes + RB::lds_bytes), joined = kFewWaves * FM * 2 * kWave * 16;
  __shared__ __attribute__((aligned(1024))) char lds[stage > joined ? stage : joined];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int across = (f.n + kFewTile - 1) / kFewTile;
  const int m0 = blockIdx.x / across * 16 * FM, n0 = blockIdx.x % across * kFewTile;
  const int steps = (k + kFewBK - 1) / kFewBK, per = (steps + kFewWaves - 1) / kFewWaves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  char* la = lds + wave * (RA::lds_bytes + RB::lds_bytes);
  f32x4 acc[2][FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) acc[0][j] = acc[1][j] = f32x4{0, 0, 0, 0};
  auto work = [&](const RA& ra, const RB& rb) {
    bf16x8 fa[FM][RA::P], fb[2][RB::P];
    ra.frags(fa, la, lane);
    rb.frags(fb, la + RA::lds_bytes, lane);
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < kPairs; ++q)
          acc[i][j] = OfHalf::mma(fb[i][pair_b<kPairs>(q)], fa[j][pair_a<kPairs>(q)], acc[i][j]);
  };
  for (int s = s0; s < s1; s += 2) {  // two steps' loads in flight
    RA a0, a1;
    RB b0, b1;
    a0.load(a, m0, f.m, s * kFewBK, k, lane);
    b0.load(b, n0, f.n, s * kFewBK, k, lane);
    const bool two = s + 1 < s1;
    if (two) {
      a1.load(a, m0, f.m, (s + 1) * kFewBK, k, lane);
      b1.load(b, n0, f.n, (s + 1) * kFewBK, k, lane);
    }
    work(a0, b0);
    if (two) work(a1, b1);
  }
  __syncthreads();
  f32x4* join = reinterpret_cast<f32x4*>(lds);  // [wave][row fragment][column fragment][lane]
#pragma unroll
  for (int j = 0; j < FM; ++j)
#pragma unroll
    for (int i = 0; i < 2; ++i) join[((wave * FM + j) * 2 + i) * kWave + lane] = acc[i][j];
  __syncthreads();
  if (threadIdx.x >= FM * kWave) return;
  const int j = threadIdx.x / kWave, row = m0 + 16 * j + (lane & 15), col = n0 + 8 * (lane >> 4);
  f32x8 v{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w) {
    v.lo += join[((w * FM + j) * 2) * kWave + lane];
    v.hi += join[((w * FM + j) * 2 + 1) * kWave + lane];
  }
  if (row < f.m && col < ((f.n + 7) & ~7)) f.put<T>(v, row, col);
}

// A step's P and its product with X in one launch, of short sides: a workgroup of eight waves forms the rows of P that its
// 16 x 32 of the result need (P is symmetric: 16 of them where X is wide, 32 where it is tall) into LDS, a wave 16 x 32 with
// all its loads in flight at once, and then each wave takes one step of k of the product, whose part of X is on the way
// meanwhile.  Every workgroup of a row (column) forms the same rows of P: it pays while there are CUs for all and a wave's
// part is one round of loads.  us of five steps in float32, one launch / two: 64 x 256 48 / 58, 128 x 771 70 / 74, 1300 x 96
// 76 / 82, but 771 x 128 84 / 74, 192 x 500 81 / 71.
constexpr int kBothWide = 128, kBothTall = 96;
constexpr int kBothWaves = 8, kBothSteps = kBothWide / kFewBK, kBothStride = kBothWide + 8;  // rows fall on different banks
template <class T, bool TALL>
__global__ __launch_bounds__(kBothWaves * kWave) void both_kernel(Planes a, OrthoFinish fp, Planes x, OrthoFinish f) {
  using RX = FewRead<TALL, !TALL, TALL ? 1 : 2>;
  constexpr int P = kPlanes, kRows = TALL ? 32 : 16;
  constexpr int stage = kBothWaves * RX::lds_bytes, joined = kBothWaves * 2 * kWave * 16;
  __shared__ __attribute__((aligned(1024))) char lds[stage > joined ? stage : joined];
  __shared__ __attribute__((aligned(16))) uint16_t strip[P][kRows][kBothStride];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15;
  const int across = (f.n + 31) / 32, m0 = blockIdx.x / across * 16, n0 = blockIdx.x % across * 32;
  const int n = fp.n, n8 = (n + 7) & ~7, steps = (n + kFewBK - 1) / kFewBK, p0 = TALL ? n0 : m0;
  const bool mine = wave < steps;
  RX rx;
  if (mine) rx.load(x, TALL ? m0 : n0, TALL ? f.m : f.n, wave * kFewBK, n, lane);
  static_assert(kBothTall / kFewBK * 2 <= kBothWaves && kBothSteps <= kBothWaves, "a part of P a wave, a step a wave");
  if (wave < steps * (kRows / 16)) {
    const int r = wave % (kRows / 16) * 16, c0 = wave / (kRows / 16) * 32;
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    FewRead<true, false, 1> ra[kBothSteps];
    FewRead<true, true> rb[kBothSteps];
#pragma unroll
    for (int h = 0; h < kBothSteps; ++h) {  // past the end: zeros
      ra[h].load(a, p0 + r, n, h * kFewBK, n, lane);
      rb[h].load(a, c0, n, h * kFewBK, n, lane);
    }
#pragma unroll
    for (int h = 0; h < kBothSteps; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < kPairs; ++q)
          acc[i] = OfHalf::mma(rb[h].r[pair_b<kPairs>(q)][i], ra[h].r[pair_a<kPairs>(q)][0], acc[i]);
    const int row = p0 + r + l, col = c0 + 8 * (lane >> 4);
    f32x8 v{{0, 0, 0, 0}, {0, 0, 0, 0}};
    if (row < n && col < n8) v = fp.value(f32x8{acc[0], acc[1]}, row, col, true);
    f16x8 h, lo;
    to_planes(v, h, lo);
    *reinterpret_cast<f16x8*>(&strip[0][r + l][col]) = h;
    *reinterpret_cast<f16x8*>(&strip[1][r + l][col]) = lo;
  }
  __syncthreads();
  f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (mine) {
    constexpr int FX = TALL ? 1 : 2, FP = TALL ? 2 : 1;
    bf16x8 fx[FX][P], pf[FP][P];
    rx.frags(fx, lds + wave * RX::lds_bytes, lane);
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
      for (int i = 0; i < FP; ++i)
        pf[i][q] = *reinterpret_cast<const bf16x8*>(
            &strip[q][TALL ? 8 * (l >> 2) + 4 * i + (l & 3) : l][wave * kFewBK + 8 * (lane >> 4)]);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int q = 0; q < kPairs; ++q) {
        const int qa = pair_a<kPairs>(q), qb = pair_b<kPairs>(q);
        if constexpr (TALL) acc[i] = OfHalf::mma(pf[i][qb], fx[0][qa], acc[i]);
        else acc[i] = OfHalf::mma(fx[i][qb], pf[0][qa], acc[i]);
      }
  }
  __syncthreads();
  f32x4* join = reinterpret_cast<f32x4*>(lds);  // [wave][column fragment][lane]
  if (mine) join[wave * 2 * kWave + lane] = acc[0], join[(wave * 2 + 1) * kWave + lane] = acc[1];
  __syncthreads();
  if (wave) return;
  const int row = m0 + l, col = n0 + 8 * (lane >> 4);
  f32x8 v{acc[0], acc[1]};
#pragma unroll
  for (int w = 1; w < kBothSteps; ++w) {
    if (w < steps) v.lo += join[w * 2 * kWave + lane], v.hi += join[(w * 2 + 1) * kWave + lane];
  }
  if (row < f.m && col < ((f.n + 7) & ~7)) f.put<T>(v, row, col);
}
bool takes_both(int rows, int cols) {
  const int side = std::min(rows, cols), most = rows > cols ? kBothTall : kBothWide;
  return side <= most && (int64_t)ceil_div(rows, 16) * ceil_div(cols, 32) <= 256;
}

// ---- how a product is cut ------------------------------------------------------------
// Microseconds, fitted over sides of 64 to 4096 and k to 8192: a step of 32 k of a workgroup while
// it has its CU to itself, for each of those that share one, and how many do; both operands k contiguous (a strided one takes
// 1.3 times as long).
struct StepTime {
  double alone, shared;
  int most;
};
StepTime step_time(int tile) {
  return tile == 256 ? StepTime{2.0, 2.0, 1} : tile == 128 ? StepTime{0.75, 0.6, 2} : StepTime{0.26, 0.2, 3};
}
struct Cut {
  int tile = 0, splits = 1, k_per_split = 0;
  double us = 0;
};
double cut_us(const Cut& q, bool strided, int64_t tiles, double fixed) {
  const StepTime t = step_time(q.tile);
  const int steps = ceil_div(q.k_per_split, kPlanesBK), round = 256 * t.most;
  const double k = steps * (strided ? 1.3 : 1.0);
  const int64_t wgs = tiles * q.splits, full = wgs / round, rest = wgs % round;
  double us = full * (k * std::max(t.alone, t.most * t.shared) + fixed);
  if (rest) us += k * std::max(t.alone, ceil_div(rest, 256) * t.shared) + fixed;
  return us;
}
// The kernel of few tiles, whose waves take their steps one after the other; strided: how many operands are.
double few_us(int m, int n, int k, int strided) {
  const int steps = ceil_div(ceil_div(k, kFewBK), few_waves(k));
  const double all = (double)ceil_div(m, kFewTile) * ceil_div(n, kFewTile) * steps / 256;
  const double more = few_waves(k) == 16 ? 1.75 : 1;
  const double half = few_half(m, n) ? 0.7 : 1;
  const double alone = (strided == 2 ? 0.42 : strided ? 0.5 : 0.6) * more * half;
  const double shared = (strided == 2 ? 0.65 : strided ? 0.83 : 1.09) * more;
  return 2.6 + std::max(steps * alone, all * shared) * 1.9;
}
// A product of m x n over k, whole: tile 32 for the kernel of few tiles.
Cut cut_product(int m, int n, int k, int strided) {
  Cut best{kFewTile, 1, 0, few_us(m, n, k, strided)};
  for (int tile : {256, 128, 64}) {
    const int64_t tiles = (int64_t)ceil_div(m, tile) * ceil_div(n, tile);
    Cut q{tile, 1, ceil_div(k, kGemmBK) * kGemmBK};
    q.us = cut_us(q, strided == 2, tiles, tile == 256 ? 9 : tile == 128 ? 5 : 3);
    if (q.us < best.us) best = q;
  }
  return best;
}
// A symmetric product of n x n over k: whole, or (splits > 0 in `part`) its triangle in parts, joined by a launch more.
struct SymmetricCut {
  Cut whole, part;
  bool joined;
  size_t part_bytes(int n) const {
    const size_t tiles = triangle_tiles(ceil_div(n, part.tile));
    return joined ? carve_bytes<float>(part.splits * tiles * part.tile * part.tile) : 0;
  }
};
SymmetricCut cut_symmetric(int n, int k, bool strided) {
  SymmetricCut c;
  c.whole = cut_product(n, n, k, strided ? 2 : 0);
  for (int tile : {256, 128, 64}) {
    const int64_t tiles = triangle_tiles(ceil_div(n, tile));
    for (int splits = 1; splits <= 64; ++splits) {
      if (splits > 1 && (splits > ceil_div(k, 2 * kGemmBK) || tiles * splits > 2048)) break;
      Cut q{tile, splits, ceil_div(ceil_div(k, kGemmBK), splits) * kGemmBK};
      if (ceil_div(k, q.k_per_split) != splits) continue;
      q.us = cut_us(q, strided, tiles, tile == 256 ? 6 : tile == 128 ? 3.5 : 2.5);
      q.us += 4 + tiles * splits * tile * tile * 8.0 / 5e6;  // the join
      if (!c.part.tile || q.us < c.part.us) c.part = q;
    }
  }
  c.joined = c.part.us < c.whole.us;
  return c;
}

template <bool AKC, bool BKC, int FORM, class E>
fgpu_status run_cut(const GemmArgs& g, int tile, int grid, const E& e, hipStream_t s) {
  if (tile == 256) gemm_kernel<Tile256, AKC, BKC, kPairs, E, OfHalf, FORM><<<grid, Tile256::threads, 0, s>>>(g, e);
  else if (tile == 128) gemm_kernel<Tile128, AKC, BKC, kPairs, E, OfHalf, FORM><<<grid, Tile128::threads, 0, s>>>(g, e);
  else gemm_kernel<Tile64, AKC, BKC, kPairs, E, OfHalf, FORM><<<grid, Tile64::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}
template <class T, bool AKC, bool BKC>
fgpu_status run_whole(const Planes& a, const Planes& b, int k, const OrthoFinish& f, const Cut& q, hipStream_t s) {
  if (q.tile == kFewTile) {
    const int across = ceil_div(f.n, kFewTile);
    const bool half = few_half(f.m, f.n), many = few_waves(k) == 16;
    auto go = [&](auto waves, auto fm) {
      constexpr int W = decltype(waves)::value, FM = decltype(fm)::value;
      few_tiles_kernel<T, AKC, BKC, W, FM><<<ceil_div(f.m, 16 * FM) * across, W * kWave, 0, s>>>(a, b, k, f);
    };
    const std::integral_constant<int, 1> w1{};
    const std::integral_constant<int, 2> w2{};
    const std::integral_constant<int, 8> w8{};
    const std::integral_constant<int, 16> w16{};
    if (many) half ? go(w16, w1) : go(w16, w2);
    else half ? go(w8, w1) : go(w8, w2);
    FGPU_HIP(hipGetLastError());
    return FGPU_OK;
  }
  const GemmArgs g{{a.p, a.ld, a.plane}, {b.p, b.ld, b.plane}, f.m, f.n, k, ceil_div(f.m, q.tile), ceil_div(f.n, q.tile), 1,
                   q.k_per_split};
  return run_cut<AKC, BKC, kPlain>(g, q.tile, g.tiles_m * g.tiles_n, OrthoEpi<T>{f}, s);
}
// a a^T of n rows (KC: k contiguous).
template <class T, bool KC>
fgpu_status run_symmetric(const Planes& a, int k, const OrthoFinish& f, float* part, hipStream_t s) {
  const SymmetricCut c = cut_symmetric(f.n, k, !KC);
  if (!c.joined) return run_whole<T, KC, KC>(a, a, k, f, c.whole, s);
  const Cut& q = c.part;
  const int t = ceil_div(f.n, q.tile), tiles = triangle_tiles(t);
  const GemmArgs g{{a.p, a.ld, a.plane}, {a.p, a.ld, a.plane}, f.n, f.n, k, t, t, q.splits, q.k_per_split};
  FGPU_TRY((run_cut<KC, KC, kTriangle>(g, q.tile, tiles * q.splits, TriangleEpi{part, tiles}, s)));
  triangle_join_kernel<<<tiles * (q.tile / 64) * (q.tile / 64), 256, 0, s>>>(f, part, q.splits, tiles, q.tile);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

struct Shape {
  int rows, cols, small, large;
  bool tall;
  Shape(int r, int c) : rows(r), cols(c), small(std::min(r, c)), large(std::max(r, c)), tall(r > c) {}
  // Where the kernels of few tiles work rows lie close, but those a multiple of 128 bytes apart 16 bytes further: their loads
  // take 64 bytes of sixteen rows at once (us, float32, apart / not: 128 x 771 65 / 70, 128 x 1024 72 / 81, 512 x 256 70 / 75,
  // 257 x 700 83 / 92, 500 x 700 130 / 139; X's rows of tall matrices 75 / 70).  Larger tiles take whole lines (2048 x 1024
  // 345 / 281).
  int64_t apart(int c, bool more) const {
    if (small > 512 || large > 1024) return packed_ld(c);
    return whole8(c) + (more && whole8(c) % 64 == 0 ? 8 : 0);
  }
  int64_t x_ld() const { return apart(cols, !tall); }
  int64_t a_ld() const { return apart(small, true); }
  size_t x_bytes() const { return carve_bytes<uint16_t>((size_t)rows * x_ld() * 2); }
  size_t a_bytes() const { return carve_bytes<uint16_t>((size_t)small * a_ld() * 2); }
  size_t part_bytes() const {
    return std::max(cut_symmetric(small, large, tall).part_bytes(small),
                    cut_symmetric(small, small, false).part_bytes(small));
  }
};
Planes planes_at(void* p, int rows, int64_t ld) { return {(uint16_t*)p, ld, rows * ld}; }

fgpu_status check_common(int64_t rows, int64_t cols, int dtype) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "orthogonalize: unknown dtype");
  FGPU_CHECK(rows >= 0 && cols >= 0, FGPU_ERR_ARG, "orthogonalize: rows and cols >= 0");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_DIM && cols <= FGPU_HEAD_MAX_DIM, FGPU_ERR_UNSUPPORTED,
             "orthogonalize: more than 2^16 rows or columns");
  return FGPU_OK;
}

// A = X X^T, P = b A + c A^2 + a I and P X (of tall X: X^T X and X P).
template <class T>
fgpu_status gram(const Planes& x, const Shape& sh, const OrthoFinish& f, float* part, hipStream_t s) {
  if (sh.tall) return run_symmetric<T, false>(x, sh.large, f, part, s);
  return run_symmetric<T, true>(x, sh.large, f, part, s);
}
template <class T>
fgpu_status step(const Planes& x, const Planes& p, const Shape& sh, const OrthoFinish& f, hipStream_t s) {
  const Cut q = cut_product(f.m, f.n, sh.small, sh.tall ? 0 : 1);
  if (sh.tall) return run_whole<T, true, true>(x, p, sh.small, f, q, s);
  return run_whole<T, true, false>(p, x, sh.small, f, q, s);
}
template <class T>
fgpu_status both(const Planes& a, const OrthoFinish& fp, const Planes& x, const Shape& sh, const OrthoFinish& f,
                 hipStream_t s) {
  const int grid = ceil_div(f.m, 16) * ceil_div(f.n, 32);
  if (sh.tall) both_kernel<T, true><<<grid, kBothWaves * kWave, 0, s>>>(a, fp, x, f);
  else both_kernel<T, false><<<grid, kBothWaves * kWave, 0, s>>>(a, fp, x, f);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

template <class T>
fgpu_status run_ortho(const T* x, const Shape& sh, int steps, float a, float b, float c, float eps, T* out, Carve& ws,
                      hipStream_t s) {
  Planes xs[2];
  for (Planes& x2 : xs) x2 = planes_at(ws.take<char>(sh.x_bytes()), sh.rows, sh.x_ld());
  const Planes ga = planes_at(ws.take<char>(sh.a_bytes()), sh.small, sh.a_ld());
  const Planes gp = planes_at(ws.take<char>(sh.a_bytes()), sh.small, sh.a_ld());
  float* part = (float*)ws.take<char>(sh.part_bytes());
  double* norm = ws.take<double>(kNormBlocks);
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "orthogonalize: workspace smaller than fgpu_orthogonalize_workspace_bytes");
  const int64_t count = (int64_t)sh.rows * sh.cols;
  const int blocks = (int)std::min<int64_t>((count + 2047) / 2048, kNormBlocks);
  norm_parts_kernel<T><<<blocks, 256, 0, s>>>(x, count, norm);
  start_kernel<T><<<(int)std::min<int64_t>((sh.rows * (whole8(sh.cols) / 8) + 255) / 256, 1024), 256, 0, s>>>(
      x, sh.rows, sh.cols, norm, blocks, eps, xs[0]);
  FGPU_HIP(hipGetLastError());
  const int n = sh.small;
  for (int i = 0; i < steps; ++i) {
    const Planes &from = xs[i & 1], &to = xs[i + 1 & 1];
    OrthoFinish fa, fp, fx;
    fa.alpha = 1 / kHeld, fa.to = ga, fa.m = fa.n = n;
    fp.alpha = c / kHeld, fp.beta = b, fp.c = ga, fp.diagonal = kHeld * a, fp.to = gp, fp.m = fp.n = n;
    fx.alpha = 1 / kHeld, fx.to = to, fx.m = sh.rows, fx.n = sh.cols;
    if (i + 1 == steps) fx.out = out, fx.alpha /= kHeld;
    FGPU_TRY(gram<T>(from, sh, fa, part, s));
    if (takes_both(sh.rows, sh.cols)) {
      FGPU_TRY(both<T>(ga, fp, from, sh, fx, s));
    } else {
      FGPU_TRY((run_symmetric<T, true>(ga, n, fp, part, s)));
      FGPU_TRY(step<T>(from, gp, sh, fx, s));
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

int fgpu_orthogonalize_tile(int64_t rows, int64_t cols, int product) {
  if (check_common(rows, cols, FGPU_DTYPE_F32) != FGPU_OK || rows == 0 || cols == 0 || product < 0 || product > 2) return -1;
  const Shape sh((int)rows, (int)cols);
  auto whole = [](const Cut& q, int m, int n) { return q.tile == kFewTile && few_half(m, n) ? 16 : q.tile; };
  if (product && takes_both(sh.rows, sh.cols)) return 0;
  if (product == 2) return whole(cut_product(sh.rows, sh.cols, sh.small, sh.tall ? 0 : 1), sh.rows, sh.cols);
  const SymmetricCut c = product ? cut_symmetric(sh.small, sh.small, false) : cut_symmetric(sh.small, sh.large, sh.tall);
  if (!c.joined) return whole(c.whole, sh.small, sh.small);
  return c.part.tile + FGPU_TILE_TRIANGLE + (c.part.splits > 1 ? FGPU_TILE_PARTS : 0);
}

fgpu_status fgpu_orthogonalize(const void* d_x, int64_t rows, int64_t cols, int dtype, int steps, float a, float b, float c,
                               float eps, void* d_y, void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, cols, dtype));
  FGPU_CHECK(steps >= 1 && steps <= FGPU_ORTHO_MAX_STEPS, FGPU_ERR_ARG, "orthogonalize: 1 to 64 steps");
  FGPU_CHECK(std::isfinite(a) && std::isfinite(b) && std::isfinite(c), FGPU_ERR_ARG,
             "orthogonalize: coefficients must be finite");
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

// gated.hpp -- the epilogue of a gated layer's tiled products: h = act(g) u from accumulators that hold both.
#pragma once

#include "head.hpp"

namespace fgpu {

// A lane holds eight columns of g in one pair of fragments and of u in the next: of 64 rows of the B tile, 32 hidden columns.
// Waves of the largest tile cover two such groups, 64 columns, whose stores then are whole lines (store_lines).
using GatedTile256 = GemmTile<256, 256, 4, 2>;
using GatedTile128 = Tile128;
using GatedTile64 = GemmTile<64, 64, 4, 1>;

// What 8-bit integer products are multiplied by: a row's scale, a column's.  T float accumulators: nothing.
struct Scales {
  const float* row = nullptr;
  const float* col = nullptr;
};
// Eight columns of a row from two fragments' accumulators, scaled where they are integers, with the bias.
template <class A>
__device__ __forceinline__ f32x8 eight(const A& lo, const A& hi, float row, const f32x8& col, const f32x8& bias) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (std::is_same_v<A, i32x4>) v.set(e, fmaf((float)(e < 4 ? lo[e] : hi[e - 4]) * col[e], row, bias[e]));
    else v.set(e, (e < 4 ? lo[e] : hi[e - 4]) + bias[e]);
  }
  return v;
}

// 64 columns of 16 rows of 16 bits each, of which a lane holds eight from 8 (lane / 16) on and the eight 32 further (a and b) of
// row lane % 16, as 128 bytes of eight rows a store: lanes eight rows apart swap halves.  16 rows of 64 bytes each, half a
// line, write a good third slower (65536 x 4096 with both factors kept, k 64 472 -> 333 us, k 1024 1120 -> 1080).  rows: how
// many of the 16.
template <bool STREAM>
__device__ __forceinline__ void store_lines(uint16_t* p, int64_t ld, int lane, int rows, const u32x4& x, const u32x4& y) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
  const bool upper = (lane & 8) == 0;
  u32x4 first, second;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t other = (uint32_t)dpp_mov<0x128>((int)(upper ? y[i] : x[i]));  // row_ror:8
    first[i] = upper ? x[i] : other, second[i] = upper ? other : y[i];
  }
  const int row = lane & 7;
  u32x4u* at = reinterpret_cast<u32x4u*>(p + row * ld + 8 * (lane >> 4) + (upper ? 0 : 32));
  u32x4u* next = reinterpret_cast<u32x4u*>(p + (row + 8) * ld + 8 * (lane >> 4) + (upper ? 0 : 32));
  if constexpr (STREAM) {
    if (row < rows) __builtin_nontemporal_store((u32x4u)first, at);
    if (row + 8 < rows) __builtin_nontemporal_store((u32x4u)second, next);
  } else {
    if (row < rows) *at = first;
    if (row + 8 < rows) *next = second;
  }
}
template <bool STREAM>
__device__ __forceinline__ void store_lines(bf16* p, int64_t ld, int lane, int rows, const f32x8& a, const f32x8& b) {
  store_lines<STREAM>((uint16_t*)p, ld, lane, rows, __builtin_bit_cast(u32x4, to_bf16x8(a)),
                      __builtin_bit_cast(u32x4, to_bf16x8(b)));
}

template <class T, int ACT>
struct GatedEpi {
  Finish f;  // bias [2 n], out [m][n], pre [m][2 n], stream
  Scales s;
  int m, n;

  template <class G>
  struct Side {
    __device__ void fetch(const GatedEpi&, int, int, int) {}
  };
  template <class G, class A>
  __device__ __forceinline__ void finish(A (&acc)[G::FN][G::FM], const GemmWave<G>& w, char*, const Side<G>&) const {
    f.stream ? rows<true>(acc, w) : rows<false>(acc, w);
  }
  // STREAM: results past the caches.
  template <bool STREAM, class G, class A>
  __device__ __forceinline__ void rows(A (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    static_assert(G::FN % 4 == 0, "groups of 32 hidden columns");
    constexpr bool kInt = std::is_same_v<A, i32x4>;
    if constexpr (sizeof(T) == 2 && G::FN == 8) {
      if (w.n0 + w.wn * 64 + 64 <= n) return lines<STREAM>(acc, w);
    }
    const f32x8 zero{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
    for (int q = 0; q < G::FN / 4; ++q) {
      const int c = w.n0 + (w.wn * (G::FN / 4) + q) * 32 + 8 * (w.lane >> 4), cnt = n - c;
      if (cnt <= 0) continue;
      f32x8 bg = zero, bu = zero, sg = zero, su = zero;
      if (f.bias) bg = load8_n((const T*)f.bias + c, cnt), bu = load8_n((const T*)f.bias + n + c, cnt);
      if (kInt) sg = load8_n(s.col + c, cnt), su = load8_n(s.col + n + c, cnt);
#pragma unroll
      for (int j = 0; j < G::FM; ++j) {
        const int64_t row = w.row(j);
        if (row >= m) continue;
        const float sr = kInt ? s.row[row] : 1.0f;
        const f32x8 g = eight(acc[4 * q][j], acc[4 * q + 1][j], sr, sg, bg);
        f32x8 u = eight(acc[4 * q + 2][j], acc[4 * q + 3][j], sr, su, bu);
        if (f.pre) {
          T* pre = (T*)f.pre + row * 2 * n + c;
          store8_n<STREAM>(pre, g, cnt);
          store8_n<STREAM>(pre + n, u, cnt);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) u.set(e, act_value<T>(g[e], ACT) * u[e]);
        store8_n<STREAM>((T*)f.out + row * n + c, u, cnt);
      }
    }
  }
  // The same where a wave's 64 columns all lie inside.
  template <bool STREAM, class G, class A>
  __device__ __forceinline__ void lines(A (&acc)[G::FN][G::FM], const GemmWave<G>& w) const {
    constexpr bool kInt = std::is_same_v<A, i32x4>;
    const int c = w.n0 + w.wn * 64, lc = c + 8 * (w.lane >> 4);
    const f32x8 zero{{0, 0, 0, 0}, {0, 0, 0, 0}};
    f32x8 bg[2] = {zero, zero}, bu[2] = {zero, zero}, sg[2] = {zero, zero}, su[2] = {zero, zero};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (f.bias) bg[q] = load8((const T*)f.bias + lc + 32 * q), bu[q] = load8((const T*)f.bias + n + lc + 32 * q);
      if (kInt) sg[q] = load8(s.col + lc + 32 * q), su[q] = load8(s.col + n + lc + 32 * q);
    }
#pragma unroll
    for (int j = 0; j < G::FM; ++j) {
      const int64_t row = w.m0 + (w.wm * G::FM + j) * 16;
      const int inside = (int)min((int64_t)16, m - row);
      if (inside <= 0) break;
      const float sr = kInt && (w.lane & 15) < inside ? s.row[row + (w.lane & 15)] : 1.0f;
      f32x8 g[2], u[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        g[q] = eight(acc[4 * q][j], acc[4 * q + 1][j], sr, sg[q], bg[q]);
        u[q] = eight(acc[4 * q + 2][j], acc[4 * q + 3][j], sr, su[q], bu[q]);
      }
      if (f.pre) {
        T* pre = (T*)f.pre + row * 2 * n + c;
        store_lines<STREAM>(pre, 2 * (int64_t)n, w.lane, inside, g[0], g[1]);
        store_lines<STREAM>(pre + n, 2 * (int64_t)n, w.lane, inside, u[0], u[1]);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) u[q].set(e, act_value<T>(g[q][e], ACT) * u[q][e]);
      store_lines<STREAM>((T*)f.out + row * n + c, n, w.lane, inside, u[0], u[1]);
    }
  }
};

// Results of more than the last-level cache's 256 MB go past it (head_gemm.hip has both sides).
inline bool past_caches(int64_t bytes) { return bytes > (int64_t)256 << 20; }

// n hidden columns over k units (OfInt8: pairs), by the plan of a product of 2 n columns.
template <int PAIRS, class Num, class T, int ACT>
fgpu_status run_gated(const GemmArgs& g, int tile, const GatedEpi<T, ACT>& e, hipStream_t s) {
  const int grid = g.tiles_m * g.tiles_n;
  using E = GatedEpi<T, ACT>;
  if constexpr (PAIRS == 1) {
    if (tile == 64) gemm_kernel<GatedTile64, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile64::threads, 0, s>>>(g, e);
    if (tile == 128) gemm_kernel<GatedTile128, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile128::threads, 0, s>>>(g, e);
  }
  if (tile == 256) gemm_kernel<GatedTile256, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile256::threads, 0, s>>>(g, e);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}
template <int PAIRS, class Num, class T>
fgpu_status run_gated(const GemmOperand& a, const GemmOperand& b, int64_t up, int m, int n, int k, const Plan& q, Finish f,
                      const Scales& sc, hipStream_t s) {
  const GemmArgs g{a, b, m, n, k, q.tiles_m, q.tiles_n, 1, ceil_div(k, kGemmBK) * kGemmBK, up};
  f.stream = past_caches((int64_t)m * n * (f.pre ? 3 : 1) * (int64_t)sizeof(T));
  switch (f.act) {
    case FGPU_ACT_NONE: return run_gated<PAIRS, Num>(g, q.tile, GatedEpi<T, FGPU_ACT_NONE>{f, sc, m, n}, s);
    case FGPU_ACT_RELU: return run_gated<PAIRS, Num>(g, q.tile, GatedEpi<T, FGPU_ACT_RELU>{f, sc, m, n}, s);
    case FGPU_ACT_GELU: return run_gated<PAIRS, Num>(g, q.tile, GatedEpi<T, FGPU_ACT_GELU>{f, sc, m, n}, s);
    default: return run_gated<PAIRS, Num>(g, q.tile, GatedEpi<T, FGPU_ACT_SILU>{f, sc, m, n}, s);
  }
}

}  // namespace fgpu

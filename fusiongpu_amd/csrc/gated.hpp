// gated.hpp -- the epilogue of a gated layer's tiled products: h = act(g) u from accumulators that hold both.
#pragma once

#include "head.hpp"

namespace fgpu {

// Waves cover 64 rows of the B tile, 32 hidden columns and what they go with, so a lane holds eight columns of g in one pair
// of fragments and of u in the next.
using GatedTile256 = Tile256;
using GatedTile128 = Tile128;
using GatedTile64 = GemmTile<64, 64, 4, 1>;

// What 8-bit integer products are multiplied by: a row's scale, a column's.  T float accumulators: nothing.
struct Scales {
  const float* row = nullptr;
  const float* col = nullptr;
};
// Eight columns of a row from two fragments' accumulators, scaled where they are integers.
template <class A>
__device__ __forceinline__ f32x8 eight(const A& lo, const A& hi, float row, const f32x8& col) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (std::is_same_v<A, i32x4>) v.set(e, (float)(e < 4 ? lo[e] : hi[e - 4]) * row * col[e]);
    else v.set(e, e < 4 ? lo[e] : hi[e - 4]);
  }
  return v;
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
        f32x8 g = eight(acc[4 * q][j], acc[4 * q + 1][j], sr, sg), u = eight(acc[4 * q + 2][j], acc[4 * q + 3][j], sr, su);
        g.lo += bg.lo, g.hi += bg.hi, u.lo += bu.lo, u.hi += bu.hi;
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
};

// Results of more than the last-level cache's 256 MB go past it (head_gemm.hip has both sides).
inline bool past_caches(int64_t bytes) { return bytes > (int64_t)256 << 20; }

// n hidden columns over k units (OfInt8: pairs), by the plan of a product of 2 n columns.
template <int PAIRS, class Num, class T, int ACT>
fgpu_status run_gated(const GemmArgs& g, int tile, const GatedEpi<T, ACT>& e, hipStream_t s) {
  const int grid = g.tiles_m * g.tiles_n;
  using E = GatedEpi<T, ACT>;
  if (tile == 256) {
    gemm_kernel<GatedTile256, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile256::threads, 0, s>>>(g, e);
  } else if (tile == 64) {
    gemm_kernel<GatedTile64, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile64::threads, 0, s>>>(g, e);
  } else if constexpr (PAIRS == 1) {
    gemm_kernel<GatedTile128, true, true, PAIRS, E, Num, kGated><<<grid, GatedTile128::threads, 0, s>>>(g, e);
  }
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

// head_direct.hip -- products of few tiles: fragments straight from the caller's arrays, k split over a workgroup's waves.
//
// Where a product has too few 64 x 64 tiles to fill the GPU, what counts is how soon the first bytes arrive and how many
// launches follow one another, not the rate of the matrix units.  Here eight waves share a 32 x 32 (or 16 x 16) tile, each
// with an eighth of k: a wave loads its fragments from global memory as they lie (any stride and alignment, no packed
// copy; float32 is split into its bf16 triple in registers, dz is formed from dy and the kept pre-activation as it is
// read), the partial tiles meet in LDS, and the epilogue is the product's own: one launch a product, or one for both
// gradients and a column sum.
//
// Bound by latency: one row x 1024 x 1024 in bf16 takes 4.6 us on the GPU, of which its 2 MB of weights are 0.4 at the
// rate of a copy and a launch 2: 64 workgroups, four k steps a wave, which it loads two at a time, so it waits for two rounds
// of loads and for the join; 128 x 768 x 2048 6.7 us (tiled 7.3 with the caches warm); float32 400 x 256 x 256 6.9 us
// (tiled, with its two copies, 12).  Beyond a few rounds of tiles the fragments' loads from the caches bound it (each
// element is read once a 32-wide tile) and the tiled products take over: head_linear.hip has the rule and both sides.
#include <algorithm>

#include "head.hpp"

namespace fgpu {
namespace {

constexpr int kDirectWaves = 8;
constexpr int kDirectThreads = kDirectWaves * kWave;
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));

// Eight consecutive elements as they lie in memory.
template <class T>
struct Run8 {
  static constexpr int words = 8 * sizeof(T) / 16;
  u32x4 w[words];
  // The first n (none for n <= 0), then zeros; avail: elements of the array from p on.
  __device__ __forceinline__ void load(const T* p, int n, int64_t avail) {
#pragma unroll
    for (int i = 0; i < words; ++i) w[i] = u32x4{0, 0, 0, 0};
    if (n <= 0) return;
    if (avail >= 8) {
#pragma unroll
      for (int i = 0; i < words; ++i) w[i] = reinterpret_cast<const u32x4u*>(p)[i];
      if (n >= 8) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (sizeof(T) == 4) w[e / 4][e % 4] = e < n ? w[e / 4][e % 4] : 0;
        else w[0][e / 2] = e < n ? w[0][e / 2] : e % 2 ? w[0][e / 2] & 0xFFFFu : 0;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= n) continue;
      if constexpr (sizeof(T) == 4) w[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(p)[e];
      else w[0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (e % 2 * 16);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[e / 4][e % 4]);
    return __uint_as_float(e % 2 ? w[0][e / 2] & 0xFFFF0000u : w[0][e / 2] << 16);
  }
  __device__ __forceinline__ void set(int e, float v) {  // float32 only
    w[e / 4][e % 4] = __float_as_uint(v);
  }
};

template <class T>
__device__ __forceinline__ Frag<T> to_frag(const Run8<T>& r) {
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    f.p[0] = __builtin_bit_cast(bf16x8, r.w[0]);
  } else {
    f32x8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.set(e, r.get(e));
    split8(v, f.p[0], f.p[1], f.p[2]);
  }
  return f;
}
// How a wave reads one operand's F fragments (16 F rows x 32 k).
template <class T, int F, bool KC, bool DZ>
struct DirectRead {
  static constexpr int kLds = KC ? 0 : Frag<T>::planes * 32 * F * 16 * 2;  // bytes a wave
  static constexpr int runs = F;  // of eight a lane (strided: 32 rows x 16 F columns over 64 lanes)
  Run8<T> r[runs], z[DZ ? runs : 1];

  __device__ __forceinline__ void load(const DirectOperand& o, int r0, int nr, int k0, int nk, int lane) {
#pragma unroll
    for (int i = 0; i < runs; ++i) {
      int64_t at;
      int n;
      if constexpr (KC) {
        const int row = r0 + 16 * i + (lane & 15), k = k0 + 8 * (lane >> 4);
        at = (int64_t)row * o.ld + k;
        n = row < nr ? nk - k : 0;
      } else {
        constexpr int a_row = 2 * F;  // runs a row
        const int t = lane + kWave * i, k = k0 + t / a_row, col = r0 + t % a_row * 8;
        at = (int64_t)k * o.ld + col;
        n = k < nk ? nr - col : 0;
      }
      r[i].load((const T*)o.p + at, n, o.count - at);
      if (DZ) z[i].load((const T*)o.pre + at, n, o.count - at);
    }
  }
  // The fragments, dz formed where DZ.  extra (bf16 dz, if `sums`): what its rounding to bf16 left, again in bf16, and what
  // was left of that: the three hold the float32 value, which the column sums take.
  __device__ __forceinline__ void frags(Frag<T> (&f)[F], bf16x8 (&extra)[2][F], int act, bool sums, char* lds, int lane) {
    Frag<T> g[runs];
    f32x8 left[runs];  // of dz
#pragma unroll
    for (int i = 0; i < runs; ++i) {
      if constexpr (DZ) {
        if constexpr (sizeof(T) == 4) {  // as float32 planes; in bf16 rounded, for the reason in head_prep.hip
#pragma unroll
          for (int e = 0; e < 8; ++e) r[i].set(e, r[i].get(e) * act_slope<T>(z[i].get(e), act));
          g[i] = to_frag(r[i]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = r[i].get(e) * act_slope<T>(z[i].get(e), act);
            g[i].p[0][e] = (bf16)v;
            left[i].set(e, v - (float)(bf16)v);
          }
        }
      } else {
        g[i] = to_frag(r[i]);
      }
    }
    if constexpr (KC) {
#pragma unroll
      for (int i = 0; i < F; ++i) f[i] = g[i];
    } else {
      put_and_turn<Frag<T>::planes>(lds, lane, [&](int i, int p) { return g[i].p[p]; },
                                    [&](int i, int p, const bf16x8& v) { f[i].p[p] = v; });
      if constexpr (DZ && sizeof(T) == 2) {
        if (sums) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            put_and_turn<1>(lds, lane, [&](int i, int) { return to_bf16x8(left[i]); },
                            [&](int i, int, const bf16x8& v) { extra[q][i] = v; });
            if (q) break;
#pragma unroll
            for (int i = 0; i < runs; ++i)
#pragma unroll
              for (int e = 0; e < 8; ++e) left[i].set(e, left[i][e] - (float)(bf16)left[i][e]);
          }
        }
      }
    }
  }
  // Rows of k in, fragments out, through the wave's own LDS and its transposing load.
  template <int P, class In, class Out>
  __device__ __forceinline__ void put_and_turn(char* lds, int lane, In in, Out out) {
    typedef __attribute__((address_space(3))) s16x4 lds_half;
    constexpr int row_bytes = F * 32, a_row = 2 * F;
    wave_lds_order();
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < runs; ++i) {
        const int t = lane + kWave * i;
        *reinterpret_cast<bf16x8*>(lds + p * 32 * row_bytes + t / a_row * row_bytes + t % a_row * 16) = in(i, p);
      }
    wave_lds_order();
    const int i16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < F; ++i) {
        char* at = lds + p * 32 * row_bytes + (8 * g + (i16 >> 2)) * row_bytes + i * 32 + (i16 & 3) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds_char*)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds_char*)(at + 4 * row_bytes));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        out(i, p, __builtin_bit_cast(bf16x8, v));
      }
    wave_lds_order();
  }
};

template <class T, int FM, int FN>
constexpr int direct_lds(bool akc, bool bkc) {
  const int stage = kDirectWaves * ((akc ? 0 : Frag<T>::planes * 32 * FM * 32) + (bkc ? 0 : Frag<T>::planes * 32 * FN * 32));
  const int join = kDirectWaves * (FM * FN + FM) * 1024;
  return stage > join ? stage : join;
}

// One tile of one product: `tile` counts column tiles first.
template <class T, int FM, int FN, bool AKC, bool BKC, bool DZ>
__device__ __forceinline__ void direct_tile(const DirectJob& j, int tile, char* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tiles_n = (j.n + 16 * FN - 1) / (16 * FN);
  const int m0 = tile / tiles_n * 16 * FM, n0 = tile % tiles_n * 16 * FN;
  const int steps = (j.k + 31) / 32, per = (steps + kDirectWaves - 1) / kDirectWaves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  using RA = DirectRead<T, FM, AKC, DZ>;
  using RB = DirectRead<T, FN, BKC, false>;
  char* la = lds + wave * (RA::kLds + RB::kLds);
  const bool sums = j.column_sum && n0 == 0;
  f32x4 acc[FN][FM], col[FM];
#pragma unroll
  for (int b = 0; b < FM; ++b) {
    col[b] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int a = 0; a < FN; ++a) acc[a][b] = f32x4{0, 0, 0, 0};
  }
  const bf16 one1 = (bf16)1.0f;
  const bf16x8 one = {one1, one1, one1, one1, one1, one1, one1, one1};
  auto work = [&](RA& a, RB& b) {
    Frag<T> fa[FM], fb[FN];
    bf16x8 ea[2][FM], eb[2][FN];
    a.frags(fa, ea, j.act, sums, la, lane);
    b.frags(fb, eb, 0, false, la + RA::kLds, lane);
#pragma unroll
    for (int x = 0; x < FM; ++x)
#pragma unroll
      for (int y = 0; y < FN; ++y) acc[y][x] = mma(fb[y], fa[x], acc[y][x]);
    if (!AKC && sums) {
#pragma unroll
      for (int x = 0; x < FM; ++x) {
        if constexpr (sizeof(T) == 4) {
          col[x] = mma(one, fa[x].p[2], col[x]);
          col[x] = mma(one, fa[x].p[1], col[x]);
        } else if constexpr (DZ) {
          col[x] = mma(one, ea[1][x], col[x]);
          col[x] = mma(one, ea[0][x], col[x]);
        }
        col[x] = mma(one, fa[x].p[0], col[x]);
      }
    }
  };
  // Two steps' loads in flight before the first one's products.
  for (int s = s0; s < s1; s += 2) {
    RA a0, a1;
    RB b0, b1;
    a0.load(j.a, m0, j.m, s * 32, j.k, lane);
    b0.load(j.b, n0, j.n, s * 32, j.k, lane);
    const bool two = s + 1 < s1;
    if (two) {
      a1.load(j.a, m0, j.m, s * 32 + 32, j.k, lane);
      b1.load(j.b, n0, j.n, s * 32 + 32, j.k, lane);
    }
    work(a0, b0);
    if (two) work(a1, b1);
  }
  f32x4* join = reinterpret_cast<f32x4*>(lds);  // [wave][fragment][lane], the sums' fragments last
  constexpr int kFrags = FM * FN + FM;
  __syncthreads();
#pragma unroll
  for (int y = 0; y < FN; ++y)
#pragma unroll
    for (int x = 0; x < FM; ++x) join[(wave * kFrags + y * FM + x) * 64 + lane] = acc[y][x];
  if (!AKC && sums) {
#pragma unroll
    for (int x = 0; x < FM; ++x) join[(wave * kFrags + FM * FN + x) * 64 + lane] = col[x];
  }
  __syncthreads();
  for (int i = tid; i < FM * FN * 64; i += kDirectThreads) {
    const int f = i / 64, l = i & 63;
    f32x4 v = join[f * 64 + l];
#pragma unroll
    for (int w = 1; w < kDirectWaves; ++w) v += join[(w * kFrags + f) * 64 + l];
    const int m = m0 + f % FM * 16 + (l & 15), n = n0 + f / FM * 16 + (l >> 4) * 4;
    if (j.f.out && m < j.m && n < j.n) finish4<T>(j.f, v, (int64_t)m * j.n + n, n, j.n - n);
  }
  if (!AKC && sums && tid < 16 * FM) {
    const int f = FM * FN + tid / 16, m = m0 + tid;
    float v = 0;
#pragma unroll
    for (int w = 0; w < kDirectWaves; ++w) v += join[(w * kFrags + f) * 64 + (tid & 15)][0];
    if (m < j.m) ((T*)j.column_sum)[m] = (T)v;
  }
}

template <class T, int FM, int FN>
__global__ __launch_bounds__(kDirectThreads) void direct_forward_kernel(DirectJob j) {
  __shared__ __attribute__((aligned(1024))) char lds[direct_lds<T, FM, FN>(true, true)];
  direct_tile<T, FM, FN, true, true, false>(j, blockIdx.x, lds);
}

// The tiles of `x` (k contiguous x strided: an input's gradient), then those of `w` (both strided: a weight's, with the
// column sums of its first operand).
template <class T, bool DZ>
__global__ __launch_bounds__(kDirectThreads) void direct_backward_kernel(DirectJob x, int x_tiles, DirectJob w) {
  __shared__ __attribute__((aligned(1024))) char lds[direct_lds<T, 2, 2>(false, false)];
  const int b = blockIdx.x;
  if (b < x_tiles)
    direct_tile<T, 2, 2, true, false, DZ>(x, b, lds);
  else
    direct_tile<T, 2, 2, false, false, DZ>(w, b - x_tiles, lds);
}

int tiles_of(const DirectJob& j, int fm, int fn) { return ceil_div(j.m, 16 * fm) * ceil_div(j.n, 16 * fn); }

}  // namespace

fgpu_status launch_direct_forward(const DirectJob& j, bool f32, hipStream_t s) {
  const bool thin = j.m <= 16;
  const int grid = tiles_of(j, thin ? 1 : 2, thin ? 1 : 2);
  if (f32)
    thin ? direct_forward_kernel<float, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_forward_kernel<float, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  else
    thin ? direct_forward_kernel<bf16, 1, 1><<<grid, kDirectThreads, 0, s>>>(j)
         : direct_forward_kernel<bf16, 2, 2><<<grid, kDirectThreads, 0, s>>>(j);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

fgpu_status launch_direct_backward(const DirectJob* x, const DirectJob* w, bool f32, hipStream_t s) {
  const DirectJob none{};
  const int xt = x ? tiles_of(*x, 2, 2) : 0, wt = w ? tiles_of(*w, 2, 2) : 0;
  if (xt + wt == 0) return FGPU_OK;
  const bool dz = (x && x->a.pre) || (w && w->a.pre);
  const auto k = f32 ? (dz ? direct_backward_kernel<float, true> : direct_backward_kernel<float, false>)
                     : (dz ? direct_backward_kernel<bf16, true> : direct_backward_kernel<bf16, false>);
  k<<<xt + wt, kDirectThreads, 0, s>>>(x ? *x : none, xt, w ? *w : none);
  FGPU_HIP(hipGetLastError());
  return FGPU_OK;
}

// Microseconds, fitted over 1 to 16384 rows and 64 to 2048 dims: a start, the k steps (32) of a wave one after the other,
// and all tiles' steps at what 256 CUs take for one each.
namespace {
int wave_steps(int64_t k) { return ceil_div(ceil_div(k, 32), kDirectWaves); }
double tile_steps(int64_t m, int64_t n, int64_t k) { return (double)ceil_div(m, 32) * ceil_div(n, 32) * wave_steps(k) / 256; }
}  // namespace
double direct_forward_estimate_us(const Product& p) {
  if (p.m <= 16) return p.f32 ? 7.5 : 4.5;
  // Rows that are not whole 16-byte groups load at half the rate or less.
  const double ragged = p.k % 8 == 0 ? 1 : p.f32 ? 1.2 : 2.4;
  return 3 + std::max<double>(wave_steps(p.k), tile_steps(p.m, p.n, p.k)) * (p.f32 ? 2.2 : 0.95) * ragged;
}
double direct_backward_estimate_us(int rows, int in_dim, int out_dim, bool f32) {
  const int longest = std::max(wave_steps(out_dim), wave_steps(rows));
  const double all = tile_steps(rows, in_dim, out_dim) + tile_steps(out_dim, in_dim, rows);
  const double ragged = in_dim % 8 || out_dim % 8 ? 1.3 : 1;
  return f32 ? 2 + (1.8 * longest + 2.2 * all) * ragged : 2.5 + (1.0 * longest + 0.6 * all) * ragged;
}

}  // namespace fgpu

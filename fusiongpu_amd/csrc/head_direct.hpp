// head_direct.hpp -- what the kernels of few tiles share (head_direct.hip, head_gated.hip): fragments straight from the
// caller's arrays, k split over a workgroup's waves, partial tiles joined in LDS.
#pragma once

#include "head.hpp"

namespace fgpu {

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
// How a wave reads one operand's F fragments (16 F rows x 32 k).  GATED: a fragment's first eight rows are rows of the
// operand, the others the ones `up` rows further on.
template <class T, int F, bool KC, bool DZ, bool GATED = false>
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
        const int row = GATED ? r0 + 8 * i + (lane & 7) : r0 + 16 * i + (lane & 15), k = k0 + 8 * (lane >> 4);
        at = (int64_t)(GATED && (lane & 8) ? row + o.up : row) * o.ld + k;
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
template <class T, int FM, int FN, bool AKC, bool BKC, bool DZ, bool GATED = false>
__device__ __forceinline__ void direct_tile(const DirectJob& j, int tile, char* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int kCols = GATED ? 8 * FN : 16 * FN;
  const int tiles_n = (j.n + kCols - 1) / kCols;
  const int m0 = tile / tiles_n * 16 * FM, n0 = tile % tiles_n * kCols;
  const int steps = (j.k + 31) / 32, per = (steps + kDirectWaves - 1) / kDirectWaves;
  const int s0 = wave * per, s1 = min(steps, s0 + per);
  using RA = DirectRead<T, FM, AKC, DZ>;
  using RB = DirectRead<T, FN, BKC, false, GATED>;
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
    if (GATED && l >= 32) continue;  // the products that the first lanes' go with
    f32x4 v = join[f * 64 + l];
#pragma unroll
    for (int w = 1; w < kDirectWaves; ++w) v += join[(w * kFrags + f) * 64 + l];
    if constexpr (GATED) {
      f32x4 u = join[f * 64 + l + 32];
#pragma unroll
      for (int w = 1; w < kDirectWaves; ++w) u += join[(w * kFrags + f) * 64 + l + 32];
      const int m = m0 + f % FM * 16 + (l & 15), n = n0 + f / FM * 8 + (l >> 4) * 4;
      if (m < j.m && n < j.n) finish4_gated<T>(j.f, v, u, m, j.n, n, j.n - n);
      continue;
    }
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

}  // namespace fgpu

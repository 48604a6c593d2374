// mfma_gemm.hpp -- the matrix-product core of the query head's operators (head_linear.hip, head_gated.hip, head_int8.hip,
// head_ortho.hip, head_loss.hip).
//
// D[m][n] = sum_k A(m, k) B(n, k) on MFMA, bf16 with float32 accumulators unless said otherwise (OfHalf, OfInt8).  Each
// operand is read either with k contiguous (rows of k) or with k strided (rows of m or n, one row a k), so the forward
// product x W^T and both gradients dz W and dz^T x come from one kernel without a transposed copy.  float32 operands are
// held as three bf16 planes (split2 below) and the k loop walks the six plane pairs that are more than 2^-22 of the whole.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace fgpu {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

using bf16 = __bf16;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16 v) { return (float)v; }

// Four consecutive elements as float32, at any address an element may have (global memory takes unaligned vectors).
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4u __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ f32x4 load4(const float* p) { return *reinterpret_cast<const f32x4u*>(p); }
__device__ __forceinline__ f32x4 load4(const bf16* p) {
  return __builtin_convertvector(*reinterpret_cast<const bf16x4u*>(p), f32x4);
}
__device__ __forceinline__ void store4(float* p, f32x4 v) { *reinterpret_cast<f32x4u*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, f32x4 v) {
  *reinterpret_cast<bf16x4u*>(p) = __builtin_convertvector(v, bf16x4);
}
struct f32x8 {
  f32x4 lo, hi;
  __device__ float operator[](int i) const { return i < 4 ? lo[i] : hi[i - 4]; }
  __device__ void set(int i, float v) {
    if (i < 4) lo[i] = v;
    else hi[i - 4] = v;
  }
};
typedef __bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));
__device__ __forceinline__ f32x8 load8(const float* p) { return {load4(p), load4(p + 4)}; }
__device__ __forceinline__ f32x8 to_f32x8(const bf16x8& v) {
  const bf16x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
  return {__builtin_convertvector(lo, f32x4), __builtin_convertvector(hi, f32x4)};
}
__device__ __forceinline__ f32x8 load8(const bf16* p) {
  const bf16x8 v = *reinterpret_cast<const bf16x8u*>(p);
  return to_f32x8(v);
}
__device__ __forceinline__ f32x8 operator-(const f32x8& a, const f32x8& b) { return {a.lo - b.lo, a.hi - b.hi}; }
__device__ __forceinline__ void store8(float* p, const f32x8& v) {
  store4(p, v.lo);
  store4(p + 4, v.hi);
}
__device__ __forceinline__ bf16x8 to_bf16x8(const f32x8& v) {
  const bf16x4 lo = __builtin_convertvector(v.lo, bf16x4), hi = __builtin_convertvector(v.hi, bf16x4);
  return bf16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}
__device__ __forceinline__ void store8(bf16* p, const f32x8& v) { *reinterpret_cast<bf16x8u*>(p) = to_bf16x8(v); }
// The same past the caches.
__device__ __forceinline__ void stream8(float* p, const f32x8& v) {
  __builtin_nontemporal_store(v.lo, reinterpret_cast<f32x4u*>(p));
  __builtin_nontemporal_store(v.hi, reinterpret_cast<f32x4u*>(p + 4));
}
__device__ __forceinline__ void stream8(bf16* p, const f32x8& v) {
  __builtin_nontemporal_store(to_bf16x8(v), reinterpret_cast<bf16x8u*>(p));
}
// The first `n` (1 to 4) of them; the others read as zero and are not written.
template <class T>
__device__ __forceinline__ f32x4 load4_n(const T* p, int n) {
  if (n >= 4) return load4(p);
  f32x4 v = {0, 0, 0, 0};
  for (int i = 0; i < n; ++i) v[i] = to_f32(p[i]);
  return v;
}
template <class T>
__device__ __forceinline__ void store4_n(T* p, f32x4 v, int n) {
  if (n >= 4) {
    store4(p, v);
    return;
  }
  for (int i = 0; i < n; ++i) p[i] = (T)v[i];
}

// Eight consecutive values from p on, the first cnt of them.
template <class T>
__device__ __forceinline__ f32x8 load8_n(const T* p, int cnt) {
  if (cnt >= 8) return load8(p);
  f32x8 v{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < cnt) v.set(e, to_f32(p[e]));
  return v;
}
template <bool STREAM, class T>
__device__ __forceinline__ void store8_n(T* p, const f32x8& v, int cnt) {
  if (cnt >= 8) {
    if constexpr (STREAM) stream8(p, v);
    else store8(p, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < cnt) p[e] = (T)v[e];
}

// x = h + m + l exactly (24 significant bits in three bf16 of 8) for |x| from 2^-110 on; below, l drops under bf16's
// smallest numbers.  The first is cut off rather than rounded, so that no finite x, and no product of two whose own product
// is finite, becomes infinite; the others are rounded.  So |m| < 2^-7 and |l| <= 2^-16 of x's power of two, and the
// products left out, m l + l m, are below 2^-22 of x y (2^-26 on average).  Rounding the first too makes them 2^-24, but
// products within 2^-8 of the type's end overflow then, one-term products' mean error goes only from 3.9e-8 to 3.4e-8 (a
// sum of 64 5.2e-8 to 4.7e-8, in the library's float32 product 1.4e-7), and small calls take 3 % longer.  Of a value that
// is not finite, m and l are NaN.  Two values at a time, the first in the low halves.
__device__ __forceinline__ void split2(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
  const uint32_t xh = __float_as_uint(x) & 0xFFFF0000u, yh = __float_as_uint(y) & 0xFFFF0000u;
  h = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);  // the high halves
  const f32x2 r = {x - __uint_as_float(xh), y - __uint_as_float(yh)};
  m = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
  const f32x2 q = {r[0] - __uint_as_float(m << 16), r[1] - __uint_as_float(m & 0xFFFF0000u)};
  l = __builtin_bit_cast(uint32_t, __builtin_convertvector(q, bf16x2));
}
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split8(const f32x8& v, bf16x8& h, bf16x8& m, bf16x8& l) {
  u32x4 a, b, c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t x, y, z;
    split2(v[2 * i], v[2 * i + 1], x, y, z);
    a[i] = x, b[i] = y, c[i] = z;
  }
  h = __builtin_bit_cast(bf16x8, a), m = __builtin_bit_cast(bf16x8, b), l = __builtin_bit_cast(bf16x8, c);
}
__device__ __forceinline__ void split4(const f32x4& v, bf16x4& h, bf16x4& m, bf16x4& l) {
  u32x2 a, b, c;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t x, y, z;
    split2(v[2 * i], v[2 * i + 1], x, y, z);
    a[i] = x, b[i] = y, c[i] = z;
  }
  h = __builtin_bit_cast(bf16x4, a), m = __builtin_bit_cast(bf16x4, b), l = __builtin_bit_cast(bf16x4, c);
}

// One operand of a product.  k_contig: element (r, k) at p[r ld + k]; k strided: at p[k ld + r].  p is 16-byte aligned
// and ld a multiple of 8, plane (elements) the distance of the split planes.
struct GemmOperand {
  const uint16_t* p;
  int64_t ld;
  int64_t plane;
};

// What a product's tiles are: all of D; (gated) columns of both factors in each; (triangle) of a symmetric D the ones on and
// below the diagonal.
enum GemmForm { kPlain, kGated, kTriangle };

struct GemmArgs {
  GemmOperand a, b;
  int m, n, k;
  int tiles_m, tiles_n;
  int splits;       // workgroups a tile, each on its own part of k
  int k_per_split;  // a multiple of kGemmBK
  int64_t up = 0;   // gated products: elements from a row of B to the one that its product goes with
};

// What the elements are: operands always move as 16-byte vectors of 16-bit units, eight of a row in a lane, and only the
// matrix instruction tells them apart.
struct OfBf16 {
  using Acc = f32x4;
  static __device__ __forceinline__ Acc mma(const bf16x8& n, const bf16x8& m, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(n, m, c, 0, 0, 0);
  }
};
struct OfHalf {
  using Acc = f32x4;
  static __device__ __forceinline__ Acc mma(const bf16x8& n, const bf16x8& m, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, n), __builtin_bit_cast(f16x8, m), c, 0, 0, 0);
  }
};
// Two 8-bit integers a unit: k counts pairs.  2^16 products of -128 and -128 are 2^30, which an accumulator holds;
// 2^17 would be 2^31.
struct OfInt8 {
  using Acc = i32x4;
  static __device__ __forceinline__ Acc mma(const bf16x8& n, const bf16x8& m, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, n), __builtin_bit_cast(i32x4, m), c, 0, 0, 0);
  }
};

// A lane's eight k of one row as MFMA operands: one bf16 vector, or the three planes of float32.
template <class T>
struct Frag {
  static constexpr int planes = sizeof(T) == 4 ? 3 : 1;
  bf16x8 p[planes];
};
template <class T>
__device__ __forceinline__ Frag<T> to_planes(const f32x8& v) {
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    f.p[0] = to_bf16x8(v);
  } else {
    split8(v, f.p[0], f.p[1], f.p[2]);
  }
  return f;
}
__device__ __forceinline__ f32x4 mma(const bf16x8& n, const bf16x8& m, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(n, m, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Frag<bf16>& n, const Frag<bf16>& m, f32x4 c) { return mma(n.p[0], m.p[0], c); }
__device__ __forceinline__ f32x4 mma(const Frag<float>& n, const Frag<float>& m, f32x4 c) {
  c = mma(n.p[2], m.p[0], c);
  c = mma(n.p[0], m.p[2], c);
  c = mma(n.p[1], m.p[1], c);
  c = mma(n.p[1], m.p[0], c);
  c = mma(n.p[0], m.p[1], c);
  return mma(n.p[0], m.p[0], c);
}

constexpr int kGemmBK = 64;

// Plane pairs (a, b) in the order they are accumulated, the smallest products first: of three planes six, of two three.
template <int PAIRS = 6>
__device__ __forceinline__ int pair_a(int p) { return PAIRS == 3 ? p == 0 : (0x201100 >> (4 * (5 - p))) & 0xF; }
template <int PAIRS = 6>
__device__ __forceinline__ int pair_b(int p) { return PAIRS == 3 ? p == 1 : (0x021010 >> (4 * (5 - p))) & 0xF; }

// Tiles: BM x BN a workgroup of WM x WN waves, each wave (BM / WM) x (BN / WN) in 16 x 16 MFMA tiles.
template <int BM_, int BN_, int WM_, int WN_>
struct GemmTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int waves = WM * WN, threads = waves * kWave;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int stage_bytes = (BM + BN) * kGemmBK * 2;
};
using Tile256 = GemmTile<256, 256, 2, 4>;
using Tile128 = GemmTile<128, 128, 2, 2>;
using Tile64 = GemmTile<64, 64, 2, 2>;
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;

// A barrier behind which every wave's loads to LDS have landed.  The wait is written out: before a barrier at the head of
// a loop the compiler leaves it away for loads that the loop's end issued.
__device__ __forceinline__ void landed_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), the other counters at their limits
  __syncthreads();
}
// The same for all loads but a wave's last N, which stay in flight (loads are counted in the order they were issued), and
// behind which its own LDS reads have ended.
template <int N>
__device__ __forceinline__ void landed_barrier_but() {
  static_assert(N < 16, "the counter's low bits");
  asm volatile("" ::: "memory");  // no access passes
  __builtin_amdgcn_s_waitcnt(0x0070 | N);  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The part of an operand's LDS tile that one lane fills (16 bytes a load straight to LDS), and the addresses its
// fragments are read from.  R: rows of m or n in the tile, NT: threads.
//
// k contiguous: R rows of 128 bytes (64 k), the row's eight 16-byte chunks permuted by chunk ^ (row & 7), so the 16
// rows of a fragment read spread over the banks.  k strided: 64 rows of R elements, read with the transposing LDS load,
// in which 16 lanes read four rows of 32 bytes; chunk pairs are permuted by the row's low bits so that those rows, and
// the ones eight further that the next 16 lanes read, lie in different banks.
// Rows of a B fragment are taken in the order b_row (below): their low bits differ elsewhere.
template <bool KC, bool ISB, int CHUNKS>
__device__ __forceinline__ int tile_swizzle(int row) {
  if constexpr (KC && CHUNKS == 4) return (row >> (ISB ? 3 : 2)) & 3;  // rows of 64 bytes: four of them span the banks
  if constexpr (KC && ISB) return (row & 3) | (((row >> 3) & 1) << 2);
  if constexpr (KC) return row & 7;
  return (ISB ? 4 * (row & 3) : 2 * (row & 3)) & (CHUNKS - 1);
}
// Row i of fragment f of the B operand is n = 32 (f / 2) + 8 (i / 4) + 4 (f % 2) + i % 4: a lane's two accumulators of a
// fragment pair (rows 4 (lane / 16) + r of each) are then eight consecutive columns, one 16-byte bf16 store.
__device__ __forceinline__ int b_row(int f, int i) { return 32 * (f >> 1) + 8 * (i >> 2) + 4 * (f & 1) + (i & 3); }

template <int R, int NT, bool KC, bool ISB, int BK = kGemmBK>
struct TileLoad {
  static constexpr int row_bytes = KC ? BK * 2 : R * 2;
  static constexpr int rows = KC ? R : BK;
  static constexpr int rows_a_load = NT * 16 / row_bytes;
  static constexpr int loads = rows / rows_a_load;
  static constexpr int chunks = row_bytes / 16;
  static_assert(KC || rows_a_load % 16 == 0, "the permutation must not depend on the load");
  static_assert(rows % rows_a_load == 0, "whole loads");

  uint32_t voff;   // byte offset of the lane's chunk in load 0, from the tile's first element
  uint32_t vstep;  // byte distance of a lane's chunks in successive loads (uniform)
  int kc;          // KC: first k of the lane's chunk

  __device__ void init(int64_t ld, int tid) {
    const int row = tid / chunks, slot = tid % chunks;
    const int chunk = slot ^ tile_swizzle<KC, ISB, chunks>(row);
    voff = (uint32_t)((int64_t)row * ld * 2) + chunk * 16;
    vstep = (uint32_t)((int64_t)rows_a_load * ld * 2);
    kc = chunk * 8;
  }
  // Issues the loads of k0 .. k0 + BK - 1 into the tile at `lds`.  r0: the tile's first row (m or n) of nr.  Reads beyond the
  // operand give zeros: the buffer ends with its last group of eight, and a chunk past the end of k is sent beyond it.
  // Not `live`: all zeros, nothing read.
  __device__ __forceinline__ void issue(const GemmOperand& o, int plane, int r0, int nr, int k0, int nk, lds_char* lds,
                                        int wave, bool live = true) const {
    const uint16_t* base = o.p + plane * o.plane;
    int64_t last;  // elements from base to the end of the last one wanted
    if constexpr (KC) {
      base += (int64_t)r0 * o.ld + k0;
      last = (int64_t)(min(nr - r0, R) - 1) * o.ld + min(((nk + 7) & ~7) - k0, BK);
    } else {
      base += (int64_t)k0 * o.ld + r0;
      last = (int64_t)(min(nk - k0, BK) - 1) * o.ld + min(((nr + 7) & ~7) - r0, R);
    }
    auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, live ? (int)(last * 2) : 0, 0x00027000);
    const uint32_t off = (KC && kc >= nk - k0) ? 0x80000000u : voff;
#pragma unroll
    for (int i = 0; i < loads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + i * (NT * 16) + wave * (kWave * 16)), 16,
                                               off + i * vstep, 0, 0, 0);
  }
};

// The same for the B operand of a gated product, k contiguous: of each 64 rows of the tile the first half are rows of B, the
// second half the ones `up` elements further on that their products go with.  A wave's lanes fill rows of one half.
template <int R, int NT>
struct GatedTileLoad : TileLoad<R, NT, true, true> {
  using Base = TileLoad<R, NT, true, true>;
  static constexpr int wave_rows = kWave * 16 / Base::row_bytes;
  __device__ void init(int64_t ld, int tid) {
    Base::init(ld, tid);
    this->voff -= (uint32_t)((int64_t)(tid / kWave * wave_rows) * ld * 2);  // from the wave's first row
  }
  __device__ __forceinline__ void issue(const GemmOperand& o, int64_t up, int plane, int r0, int nr, int k0, int nk,
                                        lds_char* lds, int wave) const {
    const uint16_t* base = o.p + plane * o.plane + (int64_t)r0 * o.ld + k0;
    const int64_t last = (int64_t)(min(nr - r0, R / 2) - 1) * o.ld + min(((nk + 7) & ~7) - k0, kGemmBK);
    const uint32_t off = this->kc >= nk - k0 ? 0x80000000u : this->voff;
#pragma unroll
    for (int i = 0; i < Base::loads; ++i) {
      const int row = i * Base::rows_a_load + wave * wave_rows;  // of the tile, the wave's first
      auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base + (row & 32 ? up : 0)), 0,
                                                    (int)(last * 2), 0x00027000);
      const uint32_t at = (uint32_t)((row >> 6) * 32 + (row & 31)) * (uint32_t)(o.ld * 2);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + i * (NT * 16) + wave * (kWave * 16)), 16, off + at, 0,
                                               0, 0);
    }
  }
};

// A lane's fragments of 16 rows x 32 k (k half kk of the 64) from the tile at `lds`.
template <int R, bool KC, bool ISB, int BK = kGemmBK>
struct TileRead {
  uint32_t base;  // k contiguous: address of the lane's row and chunk in fragment 0; strided: the in-row part
  uint32_t rowp;  // strided: the row's part
  __device__ void init(int lane, int first_row) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int row = ISB ? b_row(0, i) : i;
      base = (first_row + row) * BK * 2 + ((g ^ tile_swizzle<KC, ISB, BK / 8>(row)) * 16);
      rowp = 0;
    } else {
      const int s = tile_swizzle<KC, ISB, R / 8>(i >> 2);
      rowp = (g * 8 + (i >> 2)) * R * 2;
      const int in = ISB ? (i & 3) * 16 : ((i & 3) >> 1) * 16 + (i & 1) * 8;
      base = (first_row * 2) ^ (s * 16) ^ in;
    }
  }
  __device__ __forceinline__ bf16x8 get(const lds_char* lds, int f, int kk) const {
    typedef __attribute__((address_space(3))) const bf16x8 lds_frag;
    typedef __attribute__((address_space(3))) s16x4 lds_half;
    if constexpr (KC) {
      // In B, fragment 1 of a pair starts four rows on, which the permutation does not see.
      const int rows = ISB ? 32 * (f >> 1) + 4 * (f & 1) : 16 * f;
      return *(lds_frag*)(lds + ((base ^ (kk * 64)) + rows * BK * 2));
    } else {
      // The permutation stays inside 128 bytes of A's rows and 256 of B's: what lies above is added as an immediate.
      const uint32_t in = ISB ? (base ^ ((f >> 1) * 64 & 255)) + (f & 1) * 8 + ((f >> 1) * 64 & ~255)
                              : (base ^ (f * 32 & 127)) + (f * 32 & ~127);
      const uint32_t a = rowp + in + kk * 32 * R * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds + a));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(lds + a + 4 * R * 2));
      s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(bf16x8, v);
    }
  }
};

// Workgroup -> (tile_m, tile_n, split).  Consecutive workgroups go to the eight XCDs in turn; each XCD gets a contiguous
// run of tiles, walked in groups of eight tile rows, so its L2 serves the operand rows that neighbouring tiles share.
__device__ __forceinline__ void gemm_tile_of(const GemmArgs& g, int wg, int total, int& tm, int& tn, int& sp) {
  constexpr int kXcd = 8, kGroup = 8;
  const int per = total / kXcd, rest = total % kXcd, x = wg % kXcd;
  int t = x * per + min(x, rest) + wg / kXcd;
  const int tiles = g.tiles_m * g.tiles_n;
  sp = t / tiles;  // a split's tiles follow one another: they share its part of the operands
  t -= sp * tiles;
  const int group = kGroup * g.tiles_n, first = t / group * kGroup;
  const int gm = min(g.tiles_m - first, kGroup), in = t % group;
  tm = first + in % gm;
  tn = in / gm;
}

// The same over the t (t + 1) / 2 tiles on and below the diagonal, row by row.
__host__ __device__ __forceinline__ int triangle_tiles(int t) { return t * (t + 1) / 2; }
__device__ __forceinline__ void triangle_at(int t, int& tm, int& tn) {
  tm = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
  if (triangle_tiles(tm + 1) <= t) ++tm;
  if (triangle_tiles(tm) > t) --tm;
  tn = t - triangle_tiles(tm);
}
__device__ __forceinline__ void gemm_triangle_of(const GemmArgs& g, int wg, int total, int& tm, int& tn, int& sp) {
  constexpr int kXcd = 8;
  const int per = total / kXcd, rest = total % kXcd, x = wg % kXcd;
  const int t = x * per + min(x, rest) + wg / kXcd, tiles = triangle_tiles(g.tiles_m);
  sp = t / tiles;
  triangle_at(t - sp * tiles, tm, tn);
}

// Where a wave's part of a tile lies, for its epilogue.
template <class T>
struct GemmWave {
  int m0, n0;      // the tile's first row and column
  int tm, tn, sp;  // the tile, and the split
  int wm, wn, lane;
  char* lds;       // the wave's own part of a tile buffer, lds_bytes long
  static constexpr int lds_bytes = T::stage_bytes / T::waves;
  __device__ int row(int j) const { return m0 + (wm * T::FM + j) * 16 + (lane & 15); }
  __device__ int first_col() const { return n0 + wn * T::FN * 16; }
  __device__ int col(int p) const { return first_col() + 32 * p + 8 * (lane >> 4); }
};
// acc[f][j]: a lane holds columns col(p) .. col(p) + 7 of row(j) in acc[2 p][j] and acc[2 p + 1][j].

template <class T, bool BKC, int FORM>
using GemmLoadB = std::conditional_t<FORM == kGated, GatedTileLoad<T::BN, T::threads>, TileLoad<T::BN, T::threads, BKC, true>>;

// One workgroup a tile.  Of a k step's 64, the fragments of one half are read while the other half's products run, so the
// LDS's latency passes behind the matrix instructions; the step's only barrier lies between its halves, when every wave
// holds the last fragments of this buffer and the next one's loads, issued a whole step before, have to have landed.
//
// s0 and s1 are two variables of the kernel: the compiler then knows that the buffer being read is not the one being
// filled and waits for loads only at the barriers.
//
// The smallest tiles hold all three planes of float32 operands for 32 k at a time and form the six products from them:
// a barrier for 24 matrix instructions a wave instead of eight, and half the loads (a 64-wide step of k 1.2 us instead of
// 2.1 while a workgroup has its CU to itself).  Of two planes every tile holds both: the three products read each plane's
// fragments once instead of three times in two (8192 x 1024 x 1024 on 128 x 128 44 -> 41 us, on 256 x 256 61 -> 57).
constexpr int kPlanesBK = 32;
template <class T, int PAIRS>
constexpr bool gemm_planes() { return PAIRS == 3 || (PAIRS > 1 && T::BM == 64); }
constexpr int planes_of(int pairs) { return pairs == 6 ? 3 : pairs == 3 ? 2 : 1; }
template <class T, int PAIRS>
constexpr int gemm_stage() {
  return gemm_planes<T, PAIRS>() ? planes_of(PAIRS) * (T::BM + T::BN) * kPlanesBK * 2 : T::stage_bytes;
}

// k contiguous in both operands: a third buffer, so that two stages' loads are in flight (1000 x 385 x 771 forward 22.8 ->
// 19.4 us, 4096 x 1024 x 1024 79 -> 76; with strided operands, whose fragments take twice the LDS loads, a third of the CU's
// workgroups less costs as much as it gives: 16384 x 768 x 128 backward 86 -> 91).
template <class T, int PAIRS, bool KC>
constexpr int gemm_third() { return gemm_planes<T, PAIRS>() && KC && T::BM == 64 ? gemm_stage<T, PAIRS>() : 16; }

template <class T, bool AKC, bool BKC, int PAIRS, class Num, class Acc>
__device__ __forceinline__ void planes_products(const GemmArgs& g, Acc& acc, int m0, int n0, int kbeg, int kend, int wm, int wn,
                                                char (&s0)[gemm_stage<T, PAIRS>()], char (&s1)[gemm_stage<T, PAIRS>()],
                                                char (&s2)[gemm_third<T, PAIRS, AKC && BKC>()]) {
  constexpr int P = planes_of(PAIRS);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  TileLoad<T::BM, T::threads, AKC, false, kPlanesBK> la;
  TileLoad<T::BN, T::threads, BKC, true, kPlanesBK> lb;
  la.init(g.a.ld, tid);
  lb.init(g.b.ld, tid);
  TileRead<T::BM, AKC, false, kPlanesBK> ra;
  TileRead<T::BN, BKC, true, kPlanesBK> rb;
  ra.init(lane, wm * (T::BM / T::WM));
  rb.init(lane, wn * (T::BN / T::WN));
  constexpr int pa = T::BM * kPlanesBK * 2, pb = T::BN * kPlanesBK * 2;  // bytes a plane
  if (kbeg >= kend) return;
  const int klast = kbeg + (kend - kbeg - 1) / kPlanesBK * kPlanesBK;
  // Past the end the loads read nothing: a step is the same everywhere, and the compiler sees which loads are older than
  // the wait (a step that loads only sometimes would make it wait for all of them).
  auto issue = [&](char* s, int k) {
    const bool live = k < kend;
    k = min(k, klast);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      la.issue(g.a, p, m0, g.m, k, g.k, (lds_char*)s + p * pa, wave, live);
      lb.issue(g.b, p, n0, g.n, k, g.k, (lds_char*)s + P * pa + p * pb, wave, live);
    }
  };
  auto work = [&](char* s) {
    bf16x8 a[T::FM][P], b[T::FN][P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < T::FN; ++i) b[i][p] = rb.get((const lds_char*)s + P * pa + p * pb, i, 0);
#pragma unroll
      for (int j = 0; j < T::FM; ++j) a[j][p] = ra.get((const lds_char*)s + p * pa, j, 0);
    }
#pragma unroll
    for (int j = 0; j < T::FM; ++j)
#pragma unroll
      for (int i = 0; i < T::FN; ++i)
#pragma unroll
        for (int q = 0; q < PAIRS; ++q)
          acc[i][j] = Num::mma(b[i][pair_b<PAIRS>(q)], a[j][pair_a<PAIRS>(q)], acc[i][j]);
  };
  constexpr int B = kPlanesBK, in_flight = P * (decltype(la)::loads + decltype(lb)::loads);  // of one stage
  if constexpr (!(AKC && BKC) || T::BM > 64) {
    issue(s0, kbeg);
    int k = kbeg;
    for (; k + B < kend; k += 2 * B) {
      landed_barrier();
      issue(s1, k + B);
      work(s0);
      landed_barrier();
      if (k + 2 * B < kend) issue(s0, k + 2 * B);
      work(s1);
    }
    if (k < kend) {
      landed_barrier();
      work(s0);
    }
  } else {
    // The stage at k lies in `cur`, the next one's loads are in flight, and nobody reads `free` any more behind the barrier.
    auto step = [&](char* cur, char* free, int k) {
      landed_barrier_but<in_flight>();
      issue(free, k + 2 * B);
      work(cur);
    };
    issue(s0, kbeg);
    issue(s1, kbeg + B);
    int k = kbeg;
    for (; k + 2 * B < kend; k += 3 * B) {
      step(s0, s2, k);
      step(s1, s0, k + B);
      step(s2, s1, k + 2 * B);
    }
    if (k < kend) {
      step(s0, s2, k);
      if (k + B < kend) step(s1, s0, k + B);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the epilogue writes where loads may still be under way
  }
}

template <class T, bool AKC, bool BKC, int PAIRS, class Num, int FORM, class Epi>
__device__ __forceinline__ void gemm_tile(const GemmArgs& g, const Epi& epi, int wg, int wgs, char (&s0)[gemm_stage<T, PAIRS>()],
                                          char (&s1)[gemm_stage<T, PAIRS>()], char (&s2)[gemm_third<T, PAIRS, AKC && BKC>()]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  int tm, tn, sp;
  if constexpr (FORM == kTriangle) gemm_triangle_of(g, wg, wgs, tm, tn, sp);
  else gemm_tile_of(g, wg, wgs, tm, tn, sp);
  const int m0 = tm * T::BM, n0 = tn * (FORM == kGated ? T::BN / 2 : T::BN);
  const int kbeg = sp * g.k_per_split, kend = min(g.k, kbeg + g.k_per_split);
  typename Num::Acc acc[T::FN][T::FM];
#pragma unroll
  for (int i = 0; i < T::FN; ++i)
#pragma unroll
    for (int j = 0; j < T::FM; ++j) acc[i][j] = typename Num::Acc{0, 0, 0, 0};
  typename Epi::template Side<T> side;
  if constexpr (gemm_planes<T, PAIRS>()) {
    static_assert(FORM != kGated, "both factors' columns: through GemmLoadB");
    side.fetch(epi, m0, n0, tid);
    planes_products<T, AKC, BKC, PAIRS, Num>(g, acc, m0, n0, kbeg, kend, wm, wn, s0, s1, s2);
  } else {
    const int steps = max(0, (kend - kbeg + kGemmBK - 1) / kGemmBK) * PAIRS;

    TileLoad<T::BM, T::threads, AKC, false> la;
    GemmLoadB<T, BKC, FORM> lb;
    la.init(g.a.ld, tid);
    lb.init(g.b.ld, tid);
    TileRead<T::BM, AKC, false> ra;
    TileRead<T::BN, BKC, true> rb;
    ra.init(lane, wm * (T::BM / T::WM));
    rb.init(lane, wn * (T::BN / T::WN));
    constexpr int boff = T::BM * kGemmBK * 2;

    int pk = kbeg, pp = 0;  // the next stage to load
    // The pairs of one k step follow one another, so a plane's tile is read again while it is in the L2.
    auto issue = [&](char* s) {
      const int qa = PAIRS == 1 ? 0 : pair_a<PAIRS>(pp), qb = PAIRS == 1 ? 0 : pair_b<PAIRS>(pp);
      la.issue(g.a, qa, m0, g.m, pk, g.k, (lds_char*)s, wave);
      if constexpr (FORM == kGated) lb.issue(g.b, g.up, qb, n0, g.n, pk, g.k, (lds_char*)s + boff, wave);
      else lb.issue(g.b, qb, n0, g.n, pk, g.k, (lds_char*)s + boff, wave);
      if (PAIRS == 1 || ++pp == PAIRS) {
        pp = 0;
        pk += kGemmBK;
      }
    };
    struct Half {
      bf16x8 a[T::FM], b[T::FN];
    };
    auto read = [&](Half& h, char* s, int kk) {
#pragma unroll
      for (int i = 0; i < T::FN; ++i) h.b[i] = rb.get((const lds_char*)s + boff, i, kk);
#pragma unroll
      for (int j = 0; j < T::FM; ++j) h.a[j] = ra.get((const lds_char*)s, j, kk);
    };
    auto multiply = [&](const Half& h) {
#pragma unroll
      for (int j = 0; j < T::FM; ++j)
#pragma unroll
        for (int i = 0; i < T::FN; ++i)
          acc[i][j] = Num::mma(h.b[i], h.a[j], acc[i][j]);
    };
    Half h0, h1;
    // One step: the buffer `cur` holds it, `next` the following one; `more`: the one after that exists.
    auto step = [&](char* cur, char* next, bool more) {
      read(h1, cur, 1);
      multiply(h0);
      landed_barrier();
      if (more) issue(cur);
      read(h0, next, 0);
      multiply(h1);
    };
    int left = steps;
    if (left > 0) {
      issue(s0);
      side.fetch(epi, m0, n0, tid);  // what the epilogue needs from memory comes in behind the products
      landed_barrier();
      if (left > 1) issue(s1);
      read(h0, s0, 0);
      for (; left >= 2; left -= 2) {
        step(s0, s1, left > 2);
        step(s1, s0, left > 3);
      }
      if (left) step(s0, s1, false);
    } else {
      side.fetch(epi, m0, n0, tid);
    }
  }
  __syncthreads();
  const GemmWave<T> w{m0, n0, tm, tn, sp, wm, wn, lane, s1 + wave * (T::stage_bytes / T::waves)};
  epi.template finish<T>(acc, w, s1, side);
}

// Registers for two waves a SIMD: one workgroup of 256 x 256 a CU, two of 128 x 128.
template <class T, bool AKC, bool BKC, int PAIRS, class Epi, class Num = OfBf16, int FORM = kPlain>
__global__ __launch_bounds__(T::threads, 2) void gemm_kernel(GemmArgs g, Epi epi) {
  __shared__ __attribute__((aligned(1024))) char s0[gemm_stage<T, PAIRS>()];
  __shared__ __attribute__((aligned(1024))) char s1[gemm_stage<T, PAIRS>()];
  __shared__ __attribute__((aligned(1024))) char s2[gemm_third<T, PAIRS, AKC && BKC>()];
  gemm_tile<T, AKC, BKC, PAIRS, Num, FORM>(g, epi, blockIdx.x, gridDim.x, s0, s1, s2);
}

// Both gradients of a small layer in one launch: the first x_wgs workgroups form x (A with k contiguous, B strided), the
// others w (both strided).
template <class T, int PAIRS, class Epi>
__global__ __launch_bounds__(T::threads, 2) void gemm_pair_kernel(GemmArgs x, Epi ex, int x_wgs, GemmArgs w, Epi ew) {
  __shared__ __attribute__((aligned(1024))) char s0[gemm_stage<T, PAIRS>()];
  __shared__ __attribute__((aligned(1024))) char s1[gemm_stage<T, PAIRS>()];
  __shared__ __attribute__((aligned(1024))) char s2[gemm_third<T, PAIRS, false>()];
  const int b = blockIdx.x;
  if (b < x_wgs)
    gemm_tile<T, true, false, PAIRS, OfBf16, kPlain>(x, ex, b, x_wgs, s0, s1, s2);
  else
    gemm_tile<T, false, false, PAIRS, OfBf16, kPlain>(w, ew, b - x_wgs, gridDim.x - x_wgs, s0, s1, s2);
}

}  // namespace fgpu

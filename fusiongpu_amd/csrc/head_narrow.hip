// head_narrow.hip -- the contrastive loss of up to 128 dims, where a row's vector and its gradient fit the registers.
//
// A wave holds 32 rows, or 16 (their vectors as MFMA operands, and in the backward pass their gradients as accumulators);
// tiles of 64 or 128 vectors of the other side pass through LDS.  The scores of a tile come out of the first product with eight
// consecutive columns a lane, which is just how the second product wants its k: the score gradient goes from the
// accumulators through the exponential back into the matrix unit without leaving the registers, and the 2 (float32: 6)
// bytes an element that a stored gradient would be written and read with, more than the product's own time at these
// widths, are saved.  Rows are the queries for the statistics and dq, the candidates for dc and dbias.
//
// In bfloat16 the score gradients enter the second product rounded, but where a target is among a wave's 32 x 16, its own,
// about as large as its row's others together, would put its rounding on the whole result: there what the rounding left
// enters too, as a second operand (few products: a row has one target).  In norm the gradients are then as far from the
// exact ones as their own rounding puts them, 0.0017, instead of 0.0020 to 0.0026, for 2 % of the time (8192 x 65536 x 128,
// both gradients, 713 -> 725 us).
//
// Bound by the matrix units and, beside them, by the LDS (every wave reads the whole tile, once a product) and the
// exponentials.  1000 x 100000 x 128 in float32: statistics 140 us (1.1 PFLOP/s in bf16 products), dq 277 us (1.1, the
// score product formed again); 8192 x 65536 x 128 in bf16: forward 226 us, both gradients 0.70 ms (0.79 PFLOP/s).
#include <algorithm>

#include "loss_scores.hpp"

namespace fgpu {
namespace {

constexpr int kNWaves = 8, kNThreads = kNWaves * kWave;
// Streamed vectors a tile: more work between two barriers where the planes leave room.  `small`: the shape for few rows and
// columns, whose half tiles of half the rows reach four times the CUs (bf16, 128 dims, wide / small: forward 1024 x 1024
// 15 / 9.7 us, 4096 x 4096 20.0 / 19.6, 1024 x 65536 44 / 48; backward 1024 x 1024 23 / 20, 4096 x 4096 51 / 56, 1024 x
// 65536 125 / 151).  bf16 alone: float32's wide shape has the smaller tiles already.
constexpr int narrow_tile(bool f32, bool small) { return f32 || small ? 64 : 128; }
constexpr int kNRowBytes = 256;       // of a tile's row in LDS: 128 dims
enum { kStats = 0, kDq = 1, kDc = 2 };

// Fragments of 16 rows a wave holds: two, but one where the gradient and the three planes of float32 rows of more than 64
// dims would not fit the registers of two waves a SIMD (four waves of two fragments, one a SIMD, take 315 us instead of
// 290 at 1000 x 100000 x 128).
constexpr int narrow_frags(bool f32, bool small, int mode, int kb) { return small || (f32 && mode != kStats && kb > 2) ? 1 : 2; }
constexpr int narrow_block_rows(bool f32, bool small, int mode, int kb) {
  return 16 * kNWaves * narrow_frags(f32, small, mode, kb);
}
int dim_blocks(int dim) { return dim <= 64 ? 2 : dim <= 96 ? 3 : 4; }

struct NarrowArgs {
  GemmOperand r, s;  // the rows' side and the streamed one
  int nr, ns, dim;
  int row_blocks, splits, tiles_per_split;
  LossArgs a;
  const LossRow* rows;  // backward
  f32x2* stats;         // kStats: [split][nr]
  float* target2;
  float* part;          // backward: [split][nr][dim4], or NULL: the result itself
  Finish f;             // for one split
  float* dbias;         // kDc: [split][nr], or NULL
};

// Sixteen 16-byte chunks a row, permuted by the row's bits 0, 1, 3 and 4, which differ over the rows that one read of
// either product takes: 16 rows of the score product's fragments (b_row's order), four rows of the transposing load.
__device__ __forceinline__ int narrow_swizzle(int row) {
  return ((row & 1) << 1) | ((row & 2) << 1) | (row & 8) | ((row >> 4) & 1);
}

// What the streamed side adds to the scores: {bias2, id} of a candidate or a query's LossRow.
template <int TILE>
struct StreamSide {
  float v0[TILE], v1[TILE];
  int t[TILE], id[TILE];
};
struct CandidateSide {  // as ColumnSide reads it
  const float* bias2;
  const int* col_id;
};

template <class T, bool SMALL>
constexpr int narrow_stage() { return Frag<T>::planes * narrow_tile(sizeof(T) == 4, SMALL) * kNRowBytes; }
template <class T, bool SMALL>
using Streamed = StreamSide<narrow_tile(sizeof(T) == 4, SMALL)>;

template <class T, int KB, int MODE, bool SMALL>
__device__ __forceinline__ void narrow_rows(const NarrowArgs& g, int wg, int wgs, char (&s0)[narrow_stage<T, SMALL>()],
                                            char (&s1)[narrow_stage<T, SMALL>()], Streamed<T, SMALL>& d0,
                                            Streamed<T, SMALL>& d1) {
  constexpr int kNTile = narrow_tile(sizeof(T) == 4, SMALL);
  constexpr int P = Frag<T>::planes, D = 2 * KB;  // D: 16-wide fragments of the gradient
  constexpr int F = narrow_frags(P == 3, SMALL, MODE, KB);
  typedef __attribute__((address_space(3))) const bf16x8 lds_frag;
  typedef __attribute__((address_space(3))) s16x4 lds_half;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, g4 = lane >> 4;
  int tm, tn, sp;
  GemmArgs map{};
  map.tiles_m = g.row_blocks, map.tiles_n = 1, map.splits = g.splits;
  gemm_tile_of(map, wg, wgs, tm, tn, sp);
  const int r0 = (tm * kNWaves + wave) * 16 * F;
  const int t0 = sp * g.tiles_per_split, t1 = min((g.ns + kNTile - 1) / kNTile, t0 + g.tiles_per_split);

  // the streamed tile's loads
  const int lrow = tid >> 4, lchunk = (tid & 15) ^ narrow_swizzle(lrow);
  const uint32_t voff = lchunk * 8 < g.dim ? (uint32_t)(lrow * g.s.ld * 2) + lchunk * 16 : 0x80000000u;
  const uint32_t vstep = (uint32_t)(32 * g.s.ld * 2);
  auto issue = [&](int t, char* s) {
    const int rows = min(g.ns - t * kNTile, kNTile);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint16_t* base = g.s.p + p * g.s.plane + (int64_t)t * kNTile * g.s.ld;
      auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0,
                                                    (int)(((rows - 1) * g.s.ld + ((g.dim + 7) & ~7)) * 2), 0x00027000);
#pragma unroll
      for (int i = 0; i < kNTile / 32; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc, (lds_void*)((lds_char*)s + p * (kNTile * kNRowBytes) + i * (32 * kNRowBytes) + wave * 1024), 16,
            voff + i * vstep, 0, 0, 0);
    }
  };
  // a vector a thread of the first wave: fetched with the tile's loads, laid out when the tile before is done
  LossRow side{};
  auto fetch = [&](int t) {
    if (tid >= kNTile) return;
    const int n = t * kNTile + tid;
    if constexpr (MODE == kDc) {
      side = LossRow{INFINITY, 0.0f, -1, 0};
      if (n < g.ns) side = g.rows[n];
    } else {
      side.lse2 = -INFINITY, side.id = 0;
      if (n < g.ns) {
        const float b = g.a.bias ? g.a.bias[n] : 0.0f;
        side.lse2 = b <= FGPU_MASK_BIAS ? -INFINITY : b * kLog2e;
        if (g.a.ids) side.id = g.a.ids[n];
      }
    }
  };
  auto put = [&](StreamSide<kNTile>& d) {
    if (tid >= kNTile) return;
    d.v0[tid] = side.lse2, d.id[tid] = side.id;
    if constexpr (MODE == kDc) d.v1[tid] = side.weight, d.t[tid] = side.target;
  };
  if (t0 < t1) {
    issue(t0, s0);
    fetch(t0);
    put(d0);
  }

  // the rows' side
  Frag<T> rf[KB][F];
  int row_t[F], row_id[F];
  float row_v[F], row_w[F];  // kDq: lse and weight; kDc: bias
#pragma unroll
  for (int j = 0; j < F; ++j) {
    const int row = r0 + 16 * j + i16;
    const bool in = row < g.nr;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int at = 32 * k + 8 * g4;
        bf16x8 v = {};
        if (in && at < g.dim) v = *reinterpret_cast<const bf16x8*>(g.r.p + p * g.r.plane + (int64_t)row * g.r.ld + at);
        rf[k][j].p[p] = v;
      }
    row_t[j] = -1, row_id[j] = 0, row_v[j] = INFINITY, row_w[j] = 0;
    if (!in) continue;
    if constexpr (MODE == kStats) {
      const int t = g.a.target[row];
      if ((uint32_t)t < (uint32_t)g.a.nc) {
        row_t[j] = t;
        if (g.a.ids) row_id[j] = g.a.ids[t];
      }
    } else if constexpr (MODE == kDq) {
      const LossRow r = g.rows[row];
      row_t[j] = r.target, row_id[j] = r.id, row_v[j] = r.lse2, row_w[j] = r.weight;
    } else {
      const float b = g.a.bias ? g.a.bias[row] : 0.0f;
      row_v[j] = b <= FGPU_MASK_BIAS ? -INFINITY : b * kLog2e;
      if (g.a.ids) row_id[j] = g.a.ids[row];
    }
  }

  float top[F], sum[F];  // kStats: of the lane's columns; kDc: sum[] is dbias
  f32x4 grad[MODE == kStats ? 1 : D][F];
#pragma unroll
  for (int j = 0; j < F; ++j) {
    top[j] = -INFINITY, sum[j] = 0;
#pragma unroll
    for (int f = 0; f < (MODE == kStats ? 1 : D); ++f) grad[f][j] = f32x4{0, 0, 0, 0};
  }

  const int brow = b_row(0, i16);
  const uint32_t kc_row = brow * kNRowBytes, kc_in = (g4 ^ narrow_swizzle(brow)) * 16;
  const int trow = 8 * g4 + (i16 >> 2);
  const uint32_t tr_row = trow * kNRowBytes + (i16 & 1) * 8, tr_in = (((i16 & 3) >> 1) ^ narrow_swizzle(trow)) * 16;
  auto work = [&](int t, char* s, const StreamSide<kNTile>& d) {
    const lds_char* l = (const lds_char*)s;
    // One at a time, the statistics' registers do for two workgroups a CU.
    constexpr int kTogether = MODE == kStats ? 1 : 2;
#pragma unroll kTogether
    for (int p = 0; p < kNTile / 32; ++p) {  // 32 of the tile's vectors
      f32x4 x[2][F];
#pragma unroll
      for (int j = 0; j < F; ++j) x[0][j] = x[1][j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Frag<T> f;
#pragma unroll
          for (int q = 0; q < P; ++q)
            f.p[q] = *(lds_frag*)(l + kc_row + (kc_in ^ (k * 64)) + (32 * p + 4 * h) * kNRowBytes + q * (kNTile * kNRowBytes));
#pragma unroll
          for (int j = 0; j < F; ++j) x[h][j] = mma(f, rf[k][j], x[h][j]);
        }
      const int c8 = 32 * p + 8 * g4, n = t * kNTile + c8;
      Frag<T> gf[F];
      // The tile's vectors with their dims 16 f .. 16 f + 15 as rows.
      auto turned = [&](int f, int q) {
        const lds_char* at = l + tr_row + (tr_in ^ (f * 32)) + 32 * p * kNRowBytes + q * (kNTile * kNRowBytes);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)at);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_half*)(at + 4 * kNRowBytes));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
      };
      // Score gradients as the second product's operand; bf16, `some` (the same in all lanes): also what rounding leaves.
      auto operand = [&](int j, const f32x8& v, bool some) {
        gf[j] = to_planes<T>(v);
        if constexpr (P == 1) {
          if (some) {
            const bf16x8 left = to_bf16x8(v - to_f32x8(gf[j].p[0]));
#pragma unroll
            for (int f = 0; f < D; ++f) grad[f][j] = mma(turned(f, 0), left, grad[f][j]);
          }
        }
      };
      if constexpr (MODE != kDc) {
        ColumnSide cs;
        cs.load(CandidateSide{d.v0, d.id}, c8);
#pragma unroll
        for (int j = 0; j < F; ++j) {
          f32x8 v{x[0][j], x[1][j]};
          uint32_t at;
          const bool here = scores8(g.a, v, cs, RowSide{row_t[j], row_id[j]}, n, at);
          if constexpr (MODE == kStats) {
            if (here) {
              float y = 0;
#pragma unroll
              for (int e = 0; e < 8; ++e) y = at == e ? v[e] : y;
              g.target2[r0 + 16 * j + i16] = y;
            }
            float m = top[j];
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);  // a NaN score makes the sum NaN
            const float base = m == -INFINITY ? 0.0f : m;
            float more = sum[j] * fast_exp2(top[j] - base);
#pragma unroll
            for (int e = 0; e < 8; ++e) more += fast_exp2(v[e] - base);
            top[j] = m, sum[j] = more;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.set(e, fast_exp2(v[e] - row_v[j]));
            if (here) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v.set(e, at == e ? v[e] - 1.0f : v[e]);
            }
            operand(j, v, P == 1 && __any(here));  // the row's weight waits for the sum
          }
        }
      } else {
        float lse[8], w[8];
        int qt[8], qid[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) lse[e] = d.v0[c8 + e], w[e] = d.v1[c8 + e], qt[e] = d.t[c8 + e], qid[e] = d.id[c8 + e];
#pragma unroll
        for (int j = 0; j < F; ++j) {
          const int cand = r0 + 16 * j + i16;
          f32x8 v{x[0][j], x[1][j]};
          bool rare = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v.set(e, fast_exp2(fmaf(g.a.scale2, v[e], row_v[j]) - lse[e]));
            rare |= qt[e] == cand;
            if (g.a.ids) rare |= qid[e] == row_id[j];
          }
          const bool some = __any(rare);
          if (some) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              if (g.a.ids && qid[e] == row_id[j] && qt[e] != cand && qt[e] >= 0) v.set(e, 0.0f);
              if (qt[e] == cand) v.set(e, v[e] - 1.0f);
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v.set(e, v[e] * w[e]);
            sum[j] += v[e];
          }
          operand(j, v, some);
        }
      }
      if constexpr (MODE != kStats) {
#pragma unroll
        for (int f = 0; f < D; ++f) {
          Frag<T> c;
#pragma unroll
          for (int q = 0; q < P; ++q) c.p[q] = turned(f, q);
#pragma unroll
          for (int j = 0; j < F; ++j) grad[f][j] = mma(c, gf[j], grad[f][j]);
        }
      }
    }
  };
  const bool active = r0 < g.nr;  // a wave without rows keeps to the barriers
  for (int t = t0; t < t1; t += 2) {
    landed_barrier();  // tile t is in s0 and d0; nobody reads s1 and d1 any more
    if (t + 1 < t1) issue(t + 1, s1), fetch(t + 1);
    if (active) work(t, s0, d0);
    if (t + 1 >= t1) break;
    put(d1);
    landed_barrier();
    if (t + 2 < t1) issue(t + 2, s0), fetch(t + 2);
    if (active) work(t + 1, s1, d1);
    if (t + 2 < t1) put(d0);
  }
  if (!active) return;

#pragma unroll
  for (int j = 0; j < F; ++j) {
    const int row = r0 + 16 * j + i16;
    if constexpr (MODE == kStats) {
      float m = fmaxf(top[j], __int_as_float(xchg<16>(__float_as_int(top[j]))));
      m = fmaxf(m, __int_as_float(xchg<32>(__float_as_int(m))));
      float y = sum[j] * fast_exp2(top[j] - (m == -INFINITY ? 0.0f : m));
      y += __int_as_float(xchg<16>(__float_as_int(y)));
      y += __int_as_float(xchg<32>(__float_as_int(y)));
      if (g4 == 0 && row < g.nr) g.stats[(int64_t)sp * g.nr + row] = f32x2{m, y};
    } else {
      if constexpr (MODE == kDc) {
        float y = sum[j] + __int_as_float(xchg<16>(__float_as_int(sum[j])));
        y += __int_as_float(xchg<32>(__float_as_int(y)));
        if (g.dbias && g4 == 0 && row < g.nr) g.dbias[(int64_t)sp * g.nr + row] = y;
      }
      const int d4 = (g.dim + 3) & ~3;
#pragma unroll
      for (int f = 0; f < D; ++f) {
        const int at = 16 * f + 4 * g4;
        if (row >= g.nr || at >= g.dim) continue;
        if constexpr (MODE == kDq) grad[f][j] *= row_w[j];
        if (g.part) *reinterpret_cast<f32x4*>(g.part + ((int64_t)sp * g.nr + row) * d4 + at) = grad[f][j];
        else if (g.f.out) finish4<T>(g.f, grad[f][j], (int64_t)row * g.dim + at, at, g.dim - at);
      }
    }
  }
}

#define FGPU_NARROW_LDS                                                        \
  __shared__ __attribute__((aligned(1024))) char s0[narrow_stage<T, SMALL>()]; \
  __shared__ __attribute__((aligned(1024))) char s1[narrow_stage<T, SMALL>()]; \
  __shared__ Streamed<T, SMALL> d0, d1

// bf16: registers for two workgroups a CU.
template <class T, int KB, bool SMALL>
__global__ __launch_bounds__(kNThreads, sizeof(T) == 2 ? 4 : 2) void narrow_stats_kernel(NarrowArgs g) {
  FGPU_NARROW_LDS;
  narrow_rows<T, KB, kStats, SMALL>(g, blockIdx.x, gridDim.x, s0, s1, d0, d1);
}
// The first q_wgs workgroups form dq, the others dc and dbias.
template <class T, int KB, bool SMALL>
__global__ __launch_bounds__(kNThreads, 2) void narrow_backward_kernel(NarrowArgs q, int q_wgs, NarrowArgs c) {
  FGPU_NARROW_LDS;
  const int b = blockIdx.x;
  if (b < q_wgs)
    narrow_rows<T, KB, kDq, SMALL>(q, b, q_wgs, s0, s1, d0, d1);
  else
    narrow_rows<T, KB, kDc, SMALL>(c, b - q_wgs, gridDim.x - q_wgs, s0, s1, d0, d1);
}
#undef FGPU_NARROW_LDS

struct NarrowPlan {
  bool small;
  int tile, block_rows, splits;
  double us;
};
// Splits of the streamed side: enough workgroups for `cus` CUs in even rounds, each tile at `tile_us`, the parts of a split
// gradient written and read once more (3 TB/s; 1.5 where little is to be joined).  The small shape's two gradients share one
// round between them.
NarrowPlan plan_at(int nr, int ns, bool f32, bool small, int mode, int kb, int cus, double tile_us, double part_bytes, int most) {
  NarrowPlan best{small, narrow_tile(f32, small), narrow_block_rows(f32, small, mode, kb), 0, 0};
  const int blocks = ceil_div(nr, best.block_rows), tiles = ceil_div(ns, best.tile);
  for (int s = 1; s <= std::min(tiles, most); ++s) {
    const int64_t wgs = (int64_t)blocks * s;
    int rounds = ceil_div(wgs, cus);
    if (small && mode != kStats && wgs > cus / 2) rounds = std::max(2, rounds);
    const double join = s > 1 ? s * part_bytes / (small ? 1.5e6 : 3e6) : 0;
    const double us = rounds * (ceil_div(tiles, s) * tile_us + (small ? 2.5 : 4)) + join;
    if (s == 1 || us < best.us) best.splits = s, best.us = us;
  }
  return best;
}
void set_splits(NarrowArgs& g, const NarrowPlan& p) {
  g.row_blocks = ceil_div(g.nr, p.block_rows);
  g.tiles_per_split = ceil_div(ceil_div(g.ns, p.tile), p.splits);
  g.splits = ceil_div(ceil_div(g.ns, p.tile), g.tiles_per_split);
}
NarrowPlan stats_plan(int nq, int nc, bool f32) {
  if (f32) return plan_at(nq, nc, true, false, kStats, 0, 256, 2.5, 8.0 * nq, 512);
  const NarrowPlan a = plan_at(nq, nc, false, false, kStats, 0, 512, 3.0, 8.0 * nq, 512);
  const NarrowPlan b = plan_at(nq, nc, false, true, kStats, 0, 512, 1.2, 8.0 * nq, 512);
  return b.us < a.us ? b : a;
}
// Of both gradients, whichever is asked for: their shape is one, and what is not asked for does not change the other's bits.
void gradient_plans(int nq, int nc, int dim, bool f32, int most, NarrowPlan& q, NarrowPlan& c) {
  const int kb = dim_blocks(dim);
  const double row_bytes = 4.0 * ((dim + 3) & ~3);
  for (bool small : {false, true}) {
    if (small && f32) break;
    const double tile_us = f32 ? 5.0 : small ? 1.65 : 5.1;
    const NarrowPlan a = plan_at(nq, nc, f32, small, kDq, kb, 256, tile_us, nq * row_bytes, most);
    const NarrowPlan b = plan_at(nc, nq, f32, small, kDc, kb, 256, tile_us, nc * row_bytes, most);
    if (!small || a.us + b.us < q.us + c.us) q = a, c = b;
  }
}

template <class F>
fgpu_status by_blocks(int dim, F&& f) {
  const int kb = dim_blocks(dim);
  if (kb == 2) return f(std::integral_constant<int, 2>{});
  if (kb == 3) return f(std::integral_constant<int, 3>{});
  return f(std::integral_constant<int, 4>{});
}

}  // namespace

int narrow_stats_splits(int nq, int nc, bool f32) {
  NarrowArgs g{};
  g.nr = nq, g.ns = nc;
  set_splits(g, stats_plan(nq, nc, f32));
  return g.splits;
}

fgpu_status launch_narrow_stats(const LossArgs& a, const GemmOperand& q, const GemmOperand& c, int dim, bool f32, int splits,
                                f32x2* part, float* target2, hipStream_t s) {
  NarrowPlan plan = stats_plan(a.nq, a.nc, f32);
  plan.splits = splits;
  NarrowArgs g{};
  g.r = q, g.s = c, g.nr = a.nq, g.ns = a.nc, g.dim = dim, g.a = a, g.stats = part, g.target2 = target2;
  set_splits(g, plan);
  return by_blocks(dim, [&](auto kb) -> fgpu_status {
    constexpr int KB = decltype(kb)::value;
    const int grid = g.row_blocks * g.splits;
    if (f32) narrow_stats_kernel<float, KB, false><<<grid, kNThreads, 0, s>>>(g);
    else if (plan.small) narrow_stats_kernel<bf16, KB, true><<<grid, kNThreads, 0, s>>>(g);
    else narrow_stats_kernel<bf16, KB, false><<<grid, kNThreads, 0, s>>>(g);
    FGPU_HIP(hipGetLastError());
    return FGPU_OK;
  });
}

size_t narrow_backward_bytes(int nq, int nc, int dim, bool f32, int most_splits) {
  const size_t d4 = (dim + 3) & ~3;
  NarrowPlan pq, pc;
  gradient_plans(nq, nc, dim, f32, most_splits, pq, pc);
  const int sq = pq.splits, sc = pc.splits;
  return (sq > 1 ? carve_bytes<float>((size_t)sq * nq * d4) : 0) +
         (sc > 1 ? carve_bytes<float>((size_t)sc * nc * d4) + carve_bytes<float>((size_t)sc * nc) : 0);
}

fgpu_status launch_narrow_backward(const NarrowBackward& b, int most_splits, void* ws, hipStream_t s) {
  const int nq = b.a.nq, nc = b.a.nc;
  const size_t d4 = (b.dim + 3) & ~3;
  NarrowPlan pq, pc;
  gradient_plans(nq, nc, b.dim, b.f32, most_splits, pq, pc);
  char* at = static_cast<char*>(ws);
  auto take = [&](size_t floats) {
    float* p = reinterpret_cast<float*>(at);
    at += carve_bytes<float>(floats);
    return p;
  };
  NarrowArgs q{}, c{};
  SplitJob jq, jc;
  ColumnSum sums;
  bool sum_up = false;
  q.r = b.q, q.s = b.c, q.nr = nq, q.ns = nc, q.dim = c.dim = b.dim, q.a = c.a = b.a, q.rows = c.rows = b.rows;
  c.r = b.c, c.s = b.q, c.nr = nc, c.ns = nq;
  q.f.out = b.dq, c.f.out = b.dc, q.f.alpha = c.f.alpha = b.scale;
  if (b.dq) {
    set_splits(q, pq);
    if (pq.splits > 1) {
      q.part = take((size_t)pq.splits * nq * d4);
      jq.part = q.part, jq.m = nq, jq.n = b.dim, jq.splits = q.splits, jq.f = q.f;
    }
  }
  if (b.dc || b.dbias) {
    set_splits(c, pc);
    c.dbias = b.dbias;
    if (pc.splits > 1) {
      c.part = take((size_t)pc.splits * nc * d4);
      if (b.dc) jc.part = c.part, jc.m = nc, jc.n = b.dim, jc.splits = c.splits, jc.f = c.f;
      if (b.dbias) {
        c.dbias = take((size_t)pc.splits * nc);
        sums.part = c.dbias, sums.parts = c.splits, sums.stride = sums.cols = nc, sums.out = b.dbias;
        sum_up = true;
      }
    }
  }
  const int nwq = q.row_blocks * q.splits, nwc = c.row_blocks * c.splits;
  if (nwq + nwc == 0) return FGPU_OK;
  FGPU_TRY(by_blocks(b.dim, [&](auto kb) -> fgpu_status {
    constexpr int KB = decltype(kb)::value;
    if (b.f32) narrow_backward_kernel<float, KB, false><<<nwq + nwc, kNThreads, 0, s>>>(q, nwq, c);
    else if (pq.small) narrow_backward_kernel<bf16, KB, true><<<nwq + nwc, kNThreads, 0, s>>>(q, nwq, c);
    else narrow_backward_kernel<bf16, KB, false><<<nwq + nwc, kNThreads, 0, s>>>(q, nwq, c);
    FGPU_HIP(hipGetLastError());
    return FGPU_OK;
  }));
  return launch_join(jq, jc, sum_up ? &sums : nullptr, b.f32, s);
}

}  // namespace fgpu

// loss_scores.hpp -- the scores of the contrastive loss from a product's elements, as head_loss.hip and head_narrow.hip take
// them.
#pragma once

#include "head.hpp"

namespace fgpu {

// A lane's eight columns.
struct ColumnSide {
  float bias2[8];  // -inf: masked, or beyond the candidates
  int id[8];
  bool masked;  // some lane of the wave has such a column
  template <class L>
  __device__ __forceinline__ void load(const L& l, int c) {
    bool some = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bias2[e] = l.bias2[c + e], id[e] = l.col_id[c + e];
      some |= bias2[e] == -INFINITY;
    }
    masked = __any(some);
  }
};
struct RowSide {
  int t, id;
};
// The scores of those columns at one row, from the product's elements: s = scale2 x + bias2, -inf where the column is
// masked or holds another copy of the row's document.  Masked columns, copies and the target itself are few: they stand
// behind tests that a wave passes as one (comparing ids costs an instruction an element, selecting would cost four more).
// Returns whether the row's target is among the columns (`at`: which one).
__device__ __forceinline__ bool scores8(const LossArgs& a, f32x8& v, const ColumnSide& c, const RowSide& w, int n, uint32_t& at) {
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = fmaf(a.scale2, v[e], c.bias2[e]);
  if (c.masked) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = c.bias2[e] == -INFINITY ? -INFINITY : s[e];  // whatever its vector holds
  }
  at = (uint32_t)(w.t - n);
  const bool here = w.t >= 0 && at < 8;
  if (a.ids) {
    bool same = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) same |= c.id[e] == w.id;
    if (__any(same)) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (w.t >= 0 && c.id[e] == w.id && !(here && at == e)) s[e] = -INFINITY;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v.set(e, s[e]);
  return here;
}

}  // namespace fgpu

// head_gated.hip -- the gated layer h = act(x Wg^T + bg) (x Wu^T + bu) and its gradients.
//
// Both projections are one product against the stacked weight [Wg; Wu]: a tile's B operand takes 32 rows of Wg and then the
// 32 of Wu that belong to the same hidden columns (GatedTileLoad), so a lane's accumulators hold g and u of the same
// columns and act(g) u is formed before anything is stored.
#include <algorithm>

#include "gated.hpp"

namespace fgpu {
namespace {

constexpr int kMaxHidden = FGPU_HEAD_MAX_DIM / 2;

fgpu_status check_common(int64_t rows, int in_dim, int hidden, int dtype, int act) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "gated linear: unknown dtype");
  FGPU_CHECK(act >= FGPU_ACT_NONE && act <= FGPU_ACT_SILU, FGPU_ERR_ARG, "gated linear: unknown activation");
  FGPU_CHECK(rows >= 0 && in_dim >= 1 && hidden >= 1, FGPU_ERR_ARG, "gated linear: rows >= 0, in_dim and hidden >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && in_dim <= FGPU_HEAD_MAX_DIM && hidden <= kMaxHidden, FGPU_ERR_UNSUPPORTED,
             "gated linear: more than 2^30 rows, 2^16 input dims or 2^15 hidden ones");
  return FGPU_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Between the kernel of few tiles and the tiled ones, by the estimates that the linear layer of 2 hidden columns goes by.
bool forward_direct(const Product& p, const Plan& q) {
  double tiled = q.us;
  if (needs_pack(p.k, p.f32)) tiled += 5.7 + ((double)p.m + p.n) * p.k * (p.f32 ? 10 : 4) / 4e6;
  return !q.tile || direct_forward_estimate_us(p) < tiled;
}

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

int fgpu_gated_linear_tile(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return -1;
  const Product p{(int)rows, 2 * hidden, in_dim, dtype == FGPU_DTYPE_F32};
  const Plan q = plan_product(p, false);
  return forward_direct(p, q) ? 0 : q.tile;
}

size_t fgpu_gated_linear_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const Product p{(int)rows, 2 * hidden, in_dim, f32};
  if (!needs_pack(in_dim, f32) || forward_direct(p, plan_product(p, false))) return 0;
  return packed_bytes(rows, in_dim, f32) + packed_bytes(2 * hidden, in_dim, f32);
}

fgpu_status fgpu_gated_linear(const void* d_x, const void* d_w, const void* d_bias, int64_t rows, int in_dim, int hidden,
                              int dtype, int act, void* d_h, void* d_pre, void* d_workspace, size_t workspace_bytes,
                              void* stream) {
  FGPU_TRY(check_common(rows, in_dim, hidden, dtype, act));
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_w && d_h, FGPU_ERR_ARG, "gated linear: null x, weight or output");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "gated linear: x, weight and workspace must be 16-byte aligned");
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  const Product p{(int)rows, 2 * hidden, in_dim, f32};
  const Plan q = plan_product(p, false);
  Finish f;
  f.bias = d_bias, f.out = d_h, f.pre = d_pre, f.act = act;
  if (forward_direct(p, q)) {
    DirectJob j{{d_x, in_dim, rows * in_dim, nullptr}, {d_w, in_dim, (int64_t)2 * hidden * in_dim, nullptr}, p.m, hidden, in_dim,
                0, f, nullptr};
    j.b.up = hidden;
    return launch_direct_gated(j, f32, s);
  }
  Carve ws(d_workspace, workspace_bytes);
  GemmOperand a = as_is(d_x, in_dim), b = as_is(d_w, in_dim);
  Prep prep;
  if (needs_pack(in_dim, f32)) {
    a = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    b = packed(ws.take<char>(packed_bytes(2 * hidden, in_dim, f32)), 2 * hidden, in_dim);
    prep.copy[0] = {d_x, rows, in_dim, a};
    prep.copy[1] = {d_w, 2 * hidden, in_dim, b};
  }
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "gated linear: workspace smaller than fgpu_gated_linear_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  if (f32) return run_gated<6, OfBf16, float>(a, b, hidden * b.ld, p.m, hidden, in_dim, q, f, {}, s);
  return run_gated<1, OfBf16, bf16>(a, b, hidden * b.ld, p.m, hidden, in_dim, q, f, {}, s);
}

size_t fgpu_gated_linear_backward_workspace_bytes(int64_t rows, int in_dim, int hidden, int dtype) {
  if (check_common(rows, in_dim, hidden, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const int out = 2 * hidden;
  const Product p[2] = {{(int)rows, in_dim, out, f32}, {out, in_dim, (int)rows, f32}};
  size_t b = packed_bytes(rows, out, f32) + carve_bytes<float>((size_t)dz_chunks((int)rows, hidden) * out);
  if (needs_pack(in_dim, f32)) b += packed_bytes(rows, in_dim, f32) + packed_bytes(out, in_dim, f32);
  return b + products_workspace_bytes(p, 2);
}

fgpu_status fgpu_gated_linear_backward(const void* d_dh, const void* d_x, const void* d_w, const void* d_pre, int64_t rows,
                                       int in_dim, int hidden, int dtype, int act, void* d_dx, void* d_dw, void* d_db,
                                       void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, in_dim, hidden, dtype, act));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const int m = (int)rows, out = 2 * hidden;
  hipStream_t s = as_stream(stream);
  FGPU_CHECK(rows == 0 || (d_dh && d_pre), FGPU_ERR_ARG, "gated linear backward: null dh or kept halves");
  FGPU_CHECK(rows == 0 || ((!d_dx || d_w) && (!d_dw || d_x)), FGPU_ERR_ARG,
             "gated linear backward: dx needs the weight, dw needs x");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "gated linear backward: x, weight and workspace must be 16-byte aligned");
  if (rows == 0) {
    if (d_dw) FGPU_TRY(launch_zeros((int64_t)out * in_dim, f32, d_dw, s));
    if (d_db) FGPU_TRY(launch_zeros(out, f32, d_db, s));
    return FGPU_OK;
  }
  if (!d_dx && !d_dw && !d_db) return FGPU_OK;
  const Product px{m, in_dim, out, f32}, pw{out, in_dim, m, f32};
  const bool products = d_dx || d_dw, pk = needs_pack(in_dim, f32);
  Carve ws(d_workspace, workspace_bytes);
  Prep prep;
  GemmOperand z{}, w = as_is(d_w, in_dim), x = as_is(d_x, in_dim);
  if (products) z = packed(ws.take<char>(packed_bytes(rows, out, f32)), rows, out);
  ColumnSum sums;
  if (d_db) {
    sums.parts = dz_chunks(m, hidden), sums.stride = sums.cols = out, sums.out = d_db, sums.f32 = f32;
    sums.part = ws.take<float>((size_t)sums.parts * out);
  }
  prep.dz = {d_dh, d_pre, act, m, hidden, dz_chunks(m, hidden), z, const_cast<float*>(sums.part), true};
  if (pk && d_dx) {
    w = packed(ws.take<char>(packed_bytes(out, in_dim, f32)), out, in_dim);
    prep.copy[0] = {d_w, out, in_dim, w};
  }
  if (pk && d_dw) {
    x = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    prep.copy[1] = {d_x, rows, in_dim, x};
  }
  Finish fx, fw;
  fx.out = d_dx, fw.out = d_dw;
  const ProductJob jobs[2] = {{px, z, w, true, false, fx, d_dx != nullptr}, {pw, z, x, false, false, fw, d_dw != nullptr}};
  const Product ps[2] = {px, pw};
  void* parts = ws.take<char>(products_workspace_bytes(ps, 2));
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE,
             "gated linear backward: workspace smaller than fgpu_gated_linear_backward_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  if (!products) return launch_column_sums(sums, nullptr, s);
  return launch_products(jobs, 2, d_db ? &sums : nullptr, parts, s);
}

}  // extern "C"

// head_linear.hip -- the linear layer y = act(x W^T + b) + r and its gradients.
#include <algorithm>

#include "head.hpp"

namespace fgpu {
namespace {

fgpu_status check_common(int64_t rows, int in_dim, int out_dim, int dtype, int act) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "linear: unknown dtype");
  FGPU_CHECK(act >= FGPU_ACT_NONE && act <= FGPU_ACT_SILU, FGPU_ERR_ARG, "linear: unknown activation");
  FGPU_CHECK(rows >= 0 && in_dim >= 1 && out_dim >= 1, FGPU_ERR_ARG, "linear: rows >= 0, in_dim and out_dim >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && in_dim <= FGPU_HEAD_MAX_DIM && out_dim <= FGPU_HEAD_MAX_DIM,
             FGPU_ERR_UNSUPPORTED, "linear: more than 2^30 rows or 2^16 dims");
  return FGPU_OK;
}
DirectOperand direct(const void* p, int64_t rows, int64_t cols, const void* pre = nullptr) { return {p, cols, rows * cols, pre}; }

// Whether the products of few tiles take the direct kernels (head_direct.hip): by the estimates of both, fitted to
// measurements; a launch is priced at 2.7 us, what a caller pays for it in a row of small calls.  Measured from call
// to call in a captured row of them, without an activation (us, tiled / direct): forward bf16 1 x 1024 x 1024 (rows, in,
// out) 7.4 / 5.3, 128 x 1024 x 1024 9.4 / 8.0, 512 x 1024 x 1024 8.5 / 12; float32 128 x 768 x 2048 22 / 11, 512 x 1024 x
// 1024 27 / 21, 1024^3 33 / 38; backward bf16 400 x 256 x 256 11.5 / 6.1, 256 x 1024 x 1024 15 / 11, 512 x 1024 x 1024
// 15.7 / 16.0, 1024^3 19 / 25; float32 400 x 256 x 256 18 / 8.8, 777 x 333 x 555 26 / 21, 512 x 1024 x 1024 36 / 46.
constexpr double kLaunch = 2.7;
bool forward_direct(const Product& p) {
  double tiled = products_estimate_us(&p, 1);
  if (needs_pack(p.k, p.f32)) tiled += kLaunch + 3 + ((double)p.m + p.n) * p.k * (p.f32 ? 10 : 4) / 4e6;
  return direct_forward_estimate_us(p) < tiled;
}
bool backward_direct(const Product& px, const Product& pw) {
  const Product p[2] = {px, pw};
  const double bytes = px.f32 ? (double)px.m * px.k * 14 + (double)px.m * px.n * 10 : (double)px.m * px.k * 6;
  const double tiled = products_estimate_us(p, 2) + 2 * kLaunch + 6 + bytes / 4e6;
  return direct_backward_estimate_us(px.m, px.n, px.k, px.f32) < tiled;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

int fgpu_linear_tile(int64_t rows, int in_dim, int out_dim, int dtype, int product) {
  if (check_common(rows, in_dim, out_dim, dtype, 0) != FGPU_OK || rows == 0 || product < 0 || product > 2) return -1;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const Product p[3] = {{(int)rows, out_dim, in_dim, f32}, {(int)rows, in_dim, out_dim, f32}, {out_dim, in_dim, (int)rows, f32}};
  if (product == 0) return forward_direct(p[0]) ? 0 : products_tile(p, 1, 0);
  return backward_direct(p[1], p[2]) ? 0 : products_tile(p + 1, 2, product - 1);
}

size_t fgpu_linear_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype) {
  if (check_common(rows, in_dim, out_dim, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const Product p{(int)rows, out_dim, in_dim, f32};
  if (forward_direct(p)) return 0;
  size_t b = products_workspace_bytes(&p, 1);
  if (needs_pack(in_dim, f32)) b += packed_bytes(rows, in_dim, f32) + packed_bytes(out_dim, in_dim, f32);
  return b;
}

fgpu_status fgpu_linear(const void* d_x, const void* d_w, const void* d_bias, const void* d_residual, int64_t rows,
                        int in_dim, int out_dim, int dtype, int act, void* d_y, void* d_pre, void* d_workspace,
                        size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, in_dim, out_dim, dtype, act));
  if (rows == 0) return FGPU_OK;
  FGPU_CHECK(d_x && d_w && d_y, FGPU_ERR_ARG, "linear: null x, weight or output");
  FGPU_CHECK(aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "linear: x, weight and workspace must be 16-byte aligned");
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const Product p{(int)rows, out_dim, in_dim, f32};
  hipStream_t s = as_stream(stream);
  Finish f;
  f.bias = d_bias, f.residual = d_residual, f.out = d_y, f.pre = d_pre, f.act = act;
  if (forward_direct(p))
    return launch_direct_forward({direct(d_x, rows, in_dim), direct(d_w, out_dim, in_dim), p.m, p.n, p.k, 0, f, nullptr}, f32, s);
  Carve ws(d_workspace, workspace_bytes);
  GemmOperand a = as_is(d_x, in_dim), b = as_is(d_w, in_dim);
  Prep prep;
  if (needs_pack(in_dim, f32)) {
    a = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    b = packed(ws.take<char>(packed_bytes(out_dim, in_dim, f32)), out_dim, in_dim);
    prep.copy[0] = {d_x, rows, in_dim, a};
    prep.copy[1] = {d_w, out_dim, in_dim, b};
  }
  void* parts = ws.take<char>(products_workspace_bytes(&p, 1));
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "linear: workspace smaller than fgpu_linear_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  const ProductJob j{p, a, b, true, true, f};
  return launch_products(&j, 1, nullptr, parts, s);
}

size_t fgpu_linear_backward_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype) {
  if (check_common(rows, in_dim, out_dim, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  const Product p[2] = {{(int)rows, in_dim, out_dim, f32}, {out_dim, in_dim, (int)rows, f32}};
  if (backward_direct(p[0], p[1])) return 0;
  size_t b = packed_bytes(rows, out_dim, f32) + carve_bytes<float>((size_t)dz_chunks((int)rows, out_dim) * out_dim);
  if (needs_pack(in_dim, f32)) b += packed_bytes(rows, in_dim, f32) + packed_bytes(out_dim, in_dim, f32);
  return b + products_workspace_bytes(p, 2);
}

fgpu_status fgpu_linear_backward(const void* d_dy, const void* d_x, const void* d_w, const void* d_pre, int64_t rows,
                                 int in_dim, int out_dim, int dtype, int act, void* d_dx, void* d_dw, void* d_db,
                                 void* d_workspace, size_t workspace_bytes, void* stream) {
  FGPU_TRY(check_common(rows, in_dim, out_dim, dtype, act));
  const bool f32 = dtype == FGPU_DTYPE_F32;
  hipStream_t s = as_stream(stream);
  FGPU_CHECK(rows == 0 || d_dy, FGPU_ERR_ARG, "linear backward: null dy");
  FGPU_CHECK(rows == 0 || ((!d_dx || d_w) && (!d_dw || d_x) && (act == FGPU_ACT_NONE || d_pre)), FGPU_ERR_ARG,
             "linear backward: dx needs the weight, dw needs x, an activation needs the kept pre-activation");
  FGPU_CHECK(aligned16(d_dy) && aligned16(d_x) && aligned16(d_w) && aligned16(d_workspace), FGPU_ERR_ARG,
             "linear backward: dy, x, weight and workspace must be 16-byte aligned");
  if (rows == 0) {
    if (d_dw) FGPU_TRY(launch_zeros((int64_t)out_dim * in_dim, f32, d_dw, s));
    if (d_db) FGPU_TRY(launch_zeros(out_dim, f32, d_db, s));
    return FGPU_OK;
  }
  const int m = (int)rows;
  const Product px{m, in_dim, out_dim, f32}, pw{out_dim, in_dim, m, f32};
  Finish fx, fw;
  fx.out = d_dx, fw.out = d_dw;
  if (backward_direct(px, pw)) {
    const DirectOperand z = direct(d_dy, rows, out_dim, act != FGPU_ACT_NONE ? d_pre : nullptr);
    const DirectJob jx{z, direct(d_w, out_dim, in_dim), px.m, px.n, px.k, act, fx, nullptr};
    DirectJob jw{z, direct(d_x, rows, in_dim), pw.m, pw.n, pw.k, act, fw, d_db};
    if (!d_dw) jw.b = direct(d_dy, rows, out_dim), jw.n = 1;  // the sums alone: one column tile, its product unused
    return launch_direct_backward(d_dx ? &jx : nullptr, d_dw || d_db ? &jw : nullptr, f32, s);
  }
  const bool make_dz = act != FGPU_ACT_NONE || needs_pack(out_dim, f32), pk = needs_pack(in_dim, f32);
  Carve ws(d_workspace, workspace_bytes);
  Prep prep;
  GemmOperand z = as_is(d_dy, out_dim), w = as_is(d_w, in_dim), x = as_is(d_x, in_dim);
  if (make_dz && (d_dx || d_dw)) z = packed(ws.take<char>(packed_bytes(rows, out_dim, f32)), rows, out_dim);
  const bool store_dz = make_dz && (d_dx || d_dw);
  ColumnSum sums;
  if (d_db) {
    sums.parts = dz_chunks(m, out_dim), sums.stride = sums.cols = out_dim, sums.out = d_db, sums.f32 = f32;
    sums.part = ws.take<float>((size_t)sums.parts * out_dim);
  }
  if (store_dz || d_db) {
    prep.dz = {d_dy, d_pre, act, m, out_dim, dz_chunks(m, out_dim), store_dz ? z : GemmOperand{}, const_cast<float*>(sums.part)};
  }
  if (pk && d_dx) {
    w = packed(ws.take<char>(packed_bytes(out_dim, in_dim, f32)), out_dim, in_dim);
    prep.copy[0] = {d_w, out_dim, in_dim, w};
  }
  if (pk && d_dw) {
    x = packed(ws.take<char>(packed_bytes(rows, in_dim, f32)), rows, in_dim);
    prep.copy[1] = {d_x, rows, in_dim, x};
  }
  const ProductJob jobs[2] = {{px, z, w, true, false, fx, d_dx != nullptr}, {pw, z, x, false, false, fw, d_dw != nullptr}};
  const Product ps[2] = {px, pw};
  void* parts = ws.take<char>(products_workspace_bytes(ps, 2));
  FGPU_CHECK(ws.held(), FGPU_ERR_WORKSPACE, "linear backward: workspace smaller than fgpu_linear_backward_workspace_bytes");
  FGPU_TRY(launch_prep(prep, f32, s));
  if (!d_dx && !d_dw) return d_db ? launch_column_sums(sums, nullptr, s) : FGPU_OK;
  return launch_products(jobs, 2, d_db ? &sums : nullptr, parts, s);
}

}  // extern "C"

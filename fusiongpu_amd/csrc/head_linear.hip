// head_linear.hip -- the linear layer y = act(x W^T + b) + r and its gradients.
#include <algorithm>

#include "head.hpp"

namespace fgpu {
namespace {

constexpr int kDzCols = 256;  // columns a workgroup of dz_kernel owns: 64 lanes x 4

// dz = dy act'(pre), stored as an operand (bf16, or three planes), and the column sums of dz over the workgroup's rows.
// `dst.p` NULL: the sums alone (dy itself is the operand).
template <class T>
__global__ __launch_bounds__(256) void dz_kernel(const T* dy, const T* pre, int act, int rows, int cols,
                                                 int rows_a_chunk, uint16_t* dst, int64_t ldp, int64_t plane,
                                                 float* part) {
  __shared__ f32x4 sum[4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = blockIdx.x * kDzCols + lane * 4, cnt = min(cols - c, 4);
  const int r0 = blockIdx.y * rows_a_chunk, r1 = min(rows, r0 + rows_a_chunk);
  f32x4 acc = {0, 0, 0, 0};
  if (c < (dst ? ldp : cols)) {
    for (int r = r0 + w; r < r1; r += 4) {
      f32x4 v = {0, 0, 0, 0};
      if (cnt > 0) {
        v = load4_n(dy + (int64_t)r * cols + c, cnt);
        if (act != FGPU_ACT_NONE) {
          const f32x4 z = load4_n(pre + (int64_t)r * cols + c, cnt);
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] *= act_slope(z[k], act);
        }
      }
      acc += v;
      if (dst) {
        uint16_t* d = dst + (int64_t)r * ldp + c;
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<bf16x4*>(d) = __builtin_convertvector(v, bf16x4);
        } else {
          bf16x4 h, m, l;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            bf16 a, b, e;
            split_f32(v[k], a, b, e);
            h[k] = a, m[k] = b, l[k] = e;
          }
          *reinterpret_cast<bf16x4*>(d) = h;
          *reinterpret_cast<bf16x4*>(d + plane) = m;
          *reinterpret_cast<bf16x4*>(d + 2 * plane) = l;
        }
      }
    }
  }
  if (!part) return;
  sum[w][lane] = acc;
  __syncthreads();
  if (w == 0 && cnt > 0) {
    for (int k = 1; k < 4; ++k) acc += sum[k][lane];
    for (int k = 0; k < min(cnt, 4); ++k) part[(int64_t)blockIdx.y * cols + c + k] = acc[k];
  }
}

int dz_chunks(int rows, int cols) {
  const int per = std::max(16, ceil_div((int64_t)rows * ceil_div(cols, kDzCols), 2048) );
  return ceil_div(rows, (per + 3) / 4 * 4);
}

fgpu_status check_common(int64_t rows, int in_dim, int out_dim, int dtype, int act) {
  FGPU_CHECK(dtype == FGPU_DTYPE_F32 || dtype == FGPU_DTYPE_BF16, FGPU_ERR_ARG, "linear: unknown dtype");
  FGPU_CHECK(act >= FGPU_ACT_NONE && act <= FGPU_ACT_SILU, FGPU_ERR_ARG, "linear: unknown activation");
  FGPU_CHECK(rows >= 0 && in_dim >= 1 && out_dim >= 1, FGPU_ERR_ARG, "linear: rows >= 0, in_dim and out_dim >= 1");
  FGPU_CHECK(rows <= FGPU_HEAD_MAX_ROWS && in_dim <= FGPU_HEAD_MAX_DIM && out_dim <= FGPU_HEAD_MAX_DIM,
             FGPU_ERR_UNSUPPORTED, "linear: more than 2^30 rows or 2^16 dims");
  return FGPU_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace fgpu

using namespace fgpu;

extern "C" {

size_t fgpu_linear_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype) {
  if (check_common(rows, in_dim, out_dim, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  size_t b = product_workspace_bytes({(int)rows, out_dim, in_dim, f32});
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
  Carve ws(d_workspace, workspace_bytes);
  GemmOperand a = as_is(d_x, in_dim), b = as_is(d_w, in_dim);
  void *pa = nullptr, *pb = nullptr;
  if (needs_pack(in_dim, f32)) {
    pa = ws.take<char>(packed_bytes(rows, in_dim, f32));
    pb = ws.take<char>(packed_bytes(out_dim, in_dim, f32));
  }
  void* part = ws.take<char>(product_workspace_bytes(p));
  FGPU_CHECK(ws.ok(), FGPU_ERR_WORKSPACE, "linear: workspace smaller than fgpu_linear_workspace_bytes");
  hipStream_t s = as_stream(stream);
  if (pa) {
    a = packed(pa, rows, in_dim);
    b = packed(pb, out_dim, in_dim);
    FGPU_TRY(launch_pack(d_x, rows, in_dim, f32, a, nullptr, nullptr, 0, s));
    FGPU_TRY(launch_pack(d_w, out_dim, in_dim, f32, b, nullptr, nullptr, 0, s));
  }
  Finish f;
  f.bias = d_bias, f.residual = d_residual, f.out = d_y, f.pre = d_pre, f.act = act;
  return launch_product(p, a, true, b, true, f, part, s);
}

size_t fgpu_linear_backward_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype) {
  if (check_common(rows, in_dim, out_dim, dtype, 0) != FGPU_OK || rows == 0) return 0;
  const bool f32 = dtype == FGPU_DTYPE_F32;
  size_t b = packed_bytes(rows, out_dim, f32) + carve_bytes<float>((size_t)dz_chunks((int)rows, out_dim) * out_dim);
  if (needs_pack(in_dim, f32)) b += packed_bytes(rows, in_dim, f32) + packed_bytes(out_dim, in_dim, f32);
  return b + std::max(product_workspace_bytes({(int)rows, in_dim, out_dim, f32}),
                      product_workspace_bytes({out_dim, in_dim, (int)rows, f32}));
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
  if (rows == 0) {  // sums over no rows
    if (d_dw) FGPU_TRY(launch_column_finish(nullptr, 0, 0, (int64_t)out_dim * in_dim, f32, d_dw, s));
    if (d_db) FGPU_TRY(launch_column_finish(nullptr, 0, 0, out_dim, f32, d_db, s));
    return FGPU_OK;
  }
  const int m = (int)rows;
  const Product px{m, in_dim, out_dim, f32}, pw{out_dim, in_dim, m, f32};
  Carve ws(d_workspace, workspace_bytes);
  const int chunks = dz_chunks(m, out_dim);
  const bool make_dz = act != FGPU_ACT_NONE || needs_pack(out_dim, f32), pk = needs_pack(in_dim, f32);
  char* dz = make_dz ? ws.take<char>(packed_bytes(rows, out_dim, f32)) : nullptr;
  float* part = ws.take<float>((size_t)chunks * out_dim);
  char* xp = pk && d_dw ? ws.take<char>(packed_bytes(rows, in_dim, f32)) : nullptr;
  char* wp = pk && d_dx ? ws.take<char>(packed_bytes(out_dim, in_dim, f32)) : nullptr;
  char* gw = ws.take<char>(std::max(d_dx ? product_workspace_bytes(px) : 0, d_dw ? product_workspace_bytes(pw) : 0));
  FGPU_CHECK(ws.ok(), FGPU_ERR_WORKSPACE, "linear backward: workspace smaller than fgpu_linear_backward_workspace_bytes");
  GemmOperand z = make_dz ? packed(dz, rows, out_dim) : as_is(d_dy, out_dim);
  if (make_dz || d_db) {
    const int per = ceil_div(m, chunks);
    const dim3 grid(ceil_div(packed_ld(out_dim), kDzCols), chunks);
    uint16_t* dst = make_dz ? const_cast<uint16_t*>(z.p) : nullptr;
    float* pt = d_db ? part : nullptr;
    if (f32)
      dz_kernel<float><<<grid, 256, 0, s>>>((const float*)d_dy, (const float*)d_pre, act, m, out_dim, per, dst, z.ld, z.plane, pt);
    else
      dz_kernel<bf16><<<grid, 256, 0, s>>>((const bf16*)d_dy, (const bf16*)d_pre, act, m, out_dim, per, dst, z.ld, z.plane, pt);
    FGPU_HIP(hipGetLastError());
    if (d_db) FGPU_TRY(launch_column_finish(part, chunks, out_dim, out_dim, f32, d_db, s));
  }
  if (d_dx) {
    GemmOperand w = as_is(d_w, in_dim);
    if (wp) {
      w = packed(wp, out_dim, in_dim);
      FGPU_TRY(launch_pack(d_w, out_dim, in_dim, f32, w, nullptr, nullptr, 0, s));
    }
    Finish f;
    f.out = d_dx;
    FGPU_TRY(launch_product(px, z, true, w, false, f, gw, s));
  }
  if (d_dw) {
    GemmOperand x = as_is(d_x, in_dim);
    if (xp) {
      x = packed(xp, rows, in_dim);
      FGPU_TRY(launch_pack(d_x, rows, in_dim, f32, x, nullptr, nullptr, 0, s));
    }
    Finish f;
    f.out = d_dw;
    FGPU_TRY(launch_product(pw, z, false, x, false, f, gw, s));
  }
  return FGPU_OK;
}

}  // extern "C"

// head.hpp -- what the query head's operators share: products with a fused epilogue, packed operands, column sums.
#pragma once

#include "mfma_gemm.hpp"

namespace fgpu {

// ---- activations -------------------------------------------------------------
// gelu(z) = z Phi(z).  Phi's tail T(|z|) = 1 - Phi(|z|) is the rational form 7.1.26 of Abramowitz and Stegun's handbook,
// erfc(x) = t (a1 + t (a2 + ...)) exp(-x^2) with t = 1 / (1 + p x), whose error stays below 1.5e-7 (under a float32 ulp
// of Phi near 1); it needs the exp(-z^2 / 2) that the derivative needs too.
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * 0.70710678118654752f;
  e = fast_exp2(x * x * -kLog2e);  // exp(-z^2 / 2)
  const float t = fast_rcp(fmaf(0.3275911f, x, 1.0f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * e;
  return z < 0 ? tail : 1.0f - tail;
}
__device__ __forceinline__ float sigmoid(float z) { return fast_rcp(1.0f + fast_exp2(-kLog2e * z)); }

__device__ __forceinline__ float act_value(float z, int act) {
  if (act == FGPU_ACT_RELU) return z < 0 ? 0.0f : z;
  if (act == FGPU_ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  if (act == FGPU_ACT_SILU) return z * sigmoid(z);
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == FGPU_ACT_RELU) return z > 0 ? 1.0f : 0.0f;
  if (act == FGPU_ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    return fmaf(z * 0.39894228040143268f, e, c);
  }
  if (act == FGPU_ACT_SILU) {
    const float s = sigmoid(z);
    return s * fmaf(z, 1.0f - s, 1.0f);
  }
  return 1.0f;
}

// ---- sums across lanes -----------------------------------------------------------
// Sum over aligned groups of N lanes (16, 32 or 64), the same bits in all of them.  Four exchanges inside a row of 16
// lanes (pairs, quads, then the mirrored half and the mirrored row, whose sums are already alike), two swaps beyond.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  v += __int_as_float(dpp_mov<0xB1>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x4E>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x141>(__float_as_int(v)));
  v += __int_as_float(dpp_mov<0x140>(__float_as_int(v)));
  if constexpr (N >= 32) v += __int_as_float(xchg<16>(__float_as_int(v)));
  if constexpr (N >= 64) v += __int_as_float(xchg<32>(__float_as_int(v)));
  return v;
}

// ---- products (head_gemm.hip) -------------------------------------------------
// What becomes of D: out = act(alpha D + bias) + residual, with the value before act in `pre`; out and residual [m][n].
struct Finish {
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* out = nullptr;
  void* pre = nullptr;
  float alpha = 1.0f;
  int act = FGPU_ACT_NONE;
  // Products added up over several calls (Product::chunked): D += add before the rest, and `sum` takes D in place of the
  // result; both [m][n rounded up to 4] float32.
  const float* add = nullptr;
  float* sum = nullptr;
};

// A product of m x n over k, of bf16 operands and results, or (f32) of split planes and float32 results.
struct Product {
  int m, n, k;
  bool f32;
  bool chunked = false;
};
size_t product_workspace_bytes(const Product& p);
// `ws`: product_workspace_bytes.
fgpu_status launch_product(const Product& p, const GemmOperand& a, bool a_kc, const GemmOperand& b, bool b_kc,
                           const Finish& f, void* ws, hipStream_t s);

// An array as an operand: itself where its rows can be read as they are (bf16, cols % 8 == 0), otherwise a copy with
// rows of packed_ld(cols) elements, float32 as three planes.
inline int64_t packed_ld(int64_t cols) { return (cols + 7) / 8 * 8; }
inline bool needs_pack(int64_t cols, bool f32) { return f32 || cols % 8 != 0; }
inline size_t packed_bytes(int64_t rows, int64_t cols, bool f32) {
  return carve_bytes<uint16_t>((size_t)rows * packed_ld(cols) * (f32 ? 3 : 1));
}
inline GemmOperand as_is(const void* p, int64_t cols) { return {static_cast<const uint16_t*>(p), cols, 0}; }
inline GemmOperand packed(void* p, int64_t rows, int64_t cols) {
  return {static_cast<uint16_t*>(p), packed_ld(cols), rows * packed_ld(cols)};
}
// Copies src [rows][cols] to `dst`.  zero_bias (NULL: no row): rows whose bias masks them become zero; zero_target: rows
// whose target lies outside [0, nc) do.
fgpu_status launch_pack(const void* src, int64_t rows, int64_t cols, bool f32, const GemmOperand& dst,
                        const float* zero_bias, const int32_t* zero_target, int nc, hipStream_t s);

// ---- column sums ---------------------------------------------------------------
// out[c] = sum over the parts of part[p * stride + c], c < cols, rounded to the result's type; parts are added in a
// fixed order.
fgpu_status launch_column_finish(const float* part, int parts, int64_t stride, int64_t cols, bool f32_out, void* out,
                                 hipStream_t s);

// Two such sums in one launch: the second one's parts lie `cols` after the first one's; either result may be NULL.
fgpu_status launch_column_finish2(const float* part, int parts, int64_t stride, int64_t cols, bool f32_out, void* out0,
                                  void* out1, hipStream_t s);

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

}  // namespace fgpu

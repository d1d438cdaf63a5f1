// The tensor-core product behind the dense operators (tc_gemm.cu): what a launch is told, and its host entry.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "common.cuh"

namespace gphl {

// A matrix in device memory as the product reads it: `rows` x `cols`, cols contiguous, `ld` elements from row to row.
struct Matrix {
  const void *p;
  int64_t rows, cols, ld;
};

enum Activation { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };

// out[i, j] = sum_k A[i, k] B[j, k] for i < m, j < n, in fp32.
//   a[0..1], b[0..1]   an operand that is stored with k contiguous ("K-major": rows are i or j), or with i / j contiguous (a_mn / b_mn:
//                      rows are k; 16-bit types only)
//   dual               NONE: a[0], b[0].  CONCAT: k runs over (a[0], b[0]) and then (a[1], b[1]).  BATCH: two products into out[0], out[1].
//                      GATED: g = A b[0]^T, u = A b[1]^T, out[0] = act(g) * u
//                      GATED_GRAD: the same g and u, out[0] = dh u act'(g), out[1] = dh act(g) (16-bit types)
//   typed              rows are grouped by type: rows [ptr[t], ptr[t+1]) use rows [t n, (t+1) n) of b
// e4m3 operands (fp8) are K-major and carry scales: A one per (row, block of 128 k), B one per (block of 128 j, block of 128 k).
enum Dual { DUAL_NONE, DUAL_CONCAT, DUAL_BATCH, DUAL_GATED, DUAL_GATED_GRAD };
struct GemmCall {
  int in_type = GPHL_BF16;              // GPHL_BF16 / GPHL_F16; ignored when fp8
  bool fp8 = false, a_mn = false, b_mn = false;
  Dual dual = DUAL_NONE;
  int64_t m = 0, n = 0, k = 0;          // k: of one pair of operands
  Matrix a[2] = {}, b[2] = {};
  const int32_t *ptr = nullptr;
  int64_t types = 1;
  const float *a_scale = nullptr, *b_scale[2] = {};
  int64_t a_scale_row = 0, a_scale_block = 0;      // strides of a_scale
  int act = ACT_SILU;
  void *out[2] = {};
  int64_t ld_out = 0;
  int out_type = GPHL_BF16;
  float *g = nullptr, *u = nullptr;     // GATED: also stored, m x n with row stride ld_gu
  int64_t ld_gu = 0;
  const void *dh = nullptr;             // GATED_GRAD: m x n, contiguous, of in_type
  uint8_t *q = nullptr;                 // GATED: out as e4m3 codes (row stride ld_out) and scales (block * q_scale_stride + row)
  float *q_scale = nullptr;
  int64_t q_scale_stride = 0;
  void *workspace = nullptr;            // gemm_workspace_bytes() of the same call
};

int64_t gemm_workspace_bytes(const GemmCall &c);
int gemm(const GemmCall &c, const char *what, cudaStream_t stream);
// few_rows.cu: e4m3 products of few rows, without tiles.
int few_rows_parts(const GemmCall &c);
int few_rows(const GemmCall &c, float *part, int64_t ld_part, int64_t part_u, const char *what, cudaStream_t stream);
int gemm_wait_timeouts(int *count);
int gemm_reset_wait_timeouts();

#ifdef __CUDACC__
// One instruction each (2 units in the last place): division and exponential would cost several.  Results below 2^-126 are 0: silu is from g = -87 down.
// exp(-g) as exp2(-LOG2E g) also has the rounding of that product: 2^-23 |g| relative, 3e-6 at g = -50.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_fast(float g) { return rcp_fast(1.f + exp2_fast(-LOG2E * g)); }
// Phi(g), and e = exp(-g^2 / 2) by the way.  The tail is Phi(-x) = e P(t) with t = 1 / (1 + 0.3 x): P is a polynomial without a constant term
// whose relative error over 0 <= x <= 14 was made as small as possible (1.5e-7 exactly evaluated, 4.8e-7 in fp32), so that Phi keeps its leading
// digits down to where e leaves fp32 (g = -13.2).  Farther out e's own argument bounds it: g^2 / 2 is off by 1.5 * 2^-24 of itself (g = -8: 3e-6).
__device__ __forceinline__ float normal_cdf(float g, float &e) {
  const float t = rcp_fast(fmaf(0.3f, fabsf(g), 1.f));
  e = exp2_fast(-0.5f * LOG2E * g * g);
  float p = fmaf(t, 0.035674773f, -0.15720308f);
  p = fmaf(t, p, 0.2063535f), p = fmaf(t, p, -0.05368364f), p = fmaf(t, p, 0.12856163f);
  p = fmaf(t, p, 0.09991349f), p = fmaf(t, p, 0.12075396f), p = fmaf(t, p, 0.1196293f);
  const float tail = t * p * e;
  return g < 0.f ? tail : 1.f - tail;
}
template <int ACT> __device__ __forceinline__ float activate(float g) {
  if constexpr (ACT == ACT_SILU) return g * sigmoid_fast(g);
  if constexpr (ACT == ACT_GELU) {
    float e;
    return g * normal_cdf(g, e);
  }
  return g <= 0.f ? 0.f : g;                       // a NaN stays one, -inf gives 0
}
// dg = dh u act'(g), du = dh act(g)
template <int ACT> __device__ __forceinline__ void gate_grads(float dh, float &g, float &u) {
  float h, d;                                      // act(g) and act'(g)
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid_fast(g);
    h = g * s, d = fmaf(h, 1.f - s, s);
  } else if constexpr (ACT == ACT_GELU) {
    float e;
    const float c = normal_cdf(g, e);
    h = g * c, d = c + g * 0.39894228040143268f * e;
  } else {
    h = activate<ACT_RELU>(g), d = g > 0.f ? 1.f : 0.f;
  }
  g = dh * u * d, u = dh * h;
}
// Two neighbouring elements at once: h = act(g) u, and the pair dg, du into g, u.  silu and gelu in packed arithmetic (one instruction for both
// elements but for exponential and reciprocal; gelu, 300,000 x 256 -> 1024 in bf16: 430 to 450 us forward, 482 an element at a time).
__device__ __forceinline__ uint64_t both(float v) { return pack2(v, v); }
__device__ __forceinline__ uint64_t sigmoid2(uint64_t g) {
  float a, b;
  unpack2(fmul2(g, both(-LOG2E)), a, b);
  unpack2(fadd2(pack2(exp2_fast(a), exp2_fast(b)), both(1.f)), a, b);
  return pack2(rcp_fast(a), rcp_fast(b));
}
__device__ __forceinline__ uint64_t normal_cdf2(uint64_t g, uint64_t &e) {
  float a, b, g0, g1, t0, t1;
  unpack2(ffma2(both(0.3f), g & 0x7fffffff7fffffffull, both(1.f)), a, b);
  const uint64_t t = pack2(rcp_fast(a), rcp_fast(b));
  unpack2(fmul2(fmul2(both(-0.5f * LOG2E), g), g), a, b);
  e = pack2(exp2_fast(a), exp2_fast(b));
  uint64_t p = ffma2(t, both(0.035674773f), both(-0.15720308f));
  p = ffma2(t, p, both(0.2063535f)), p = ffma2(t, p, both(-0.05368364f)), p = ffma2(t, p, both(0.12856163f));
  p = ffma2(t, p, both(0.09991349f)), p = ffma2(t, p, both(0.12075396f)), p = ffma2(t, p, both(0.1196293f));
  const uint64_t tail = fmul2(fmul2(t, p), e);
  unpack2(tail, t0, t1);
  unpack2(fsub2(both(1.f), tail), a, b);
  unpack2(g, g0, g1);
  return pack2(g0 < 0.f ? t0 : a, g1 < 0.f ? t1 : b);
}
template <int ACT> __device__ __forceinline__ void gate2(float &g0, float &g1, float u0, float u1) {
  if constexpr (ACT == ACT_SILU) {
    const uint64_t g = pack2(g0, g1);
    unpack2(fmul2(fmul2(g, sigmoid2(g)), pack2(u0, u1)), g0, g1);
  } else if constexpr (ACT == ACT_GELU) {
    uint64_t e;
    const uint64_t g = pack2(g0, g1);
    unpack2(fmul2(fmul2(g, normal_cdf2(g, e)), pack2(u0, u1)), g0, g1);
  } else {
    g0 = activate<ACT>(g0) * u0, g1 = activate<ACT>(g1) * u1;
  }
}
template <int ACT> __device__ __forceinline__ void gate_grads2(float dh0, float dh1, float &g0, float &g1, float &u0, float &u1) {
  if constexpr (ACT == ACT_SILU) {
    const uint64_t dh = pack2(dh0, dh1), g = pack2(g0, g1), s = sigmoid2(g), h = fmul2(g, s);
    const uint64_t d = ffma2(h, fsub2(both(1.f), s), s);
    unpack2(fmul2(fmul2(dh, pack2(u0, u1)), d), g0, g1);
    unpack2(fmul2(dh, h), u0, u1);
  } else if constexpr (ACT == ACT_GELU) {
    uint64_t e;
    const uint64_t dh = pack2(dh0, dh1), g = pack2(g0, g1), c = normal_cdf2(g, e), h = fmul2(g, c);
    const uint64_t d = ffma2(fmul2(both(0.39894228040143268f), g), e, c);
    unpack2(fmul2(fmul2(dh, pack2(u0, u1)), d), g0, g1);
    unpack2(fmul2(dh, h), u0, u1);
  } else {
    gate_grads<ACT>(dh0, g0, u0);
    gate_grads<ACT>(dh1, g1, u1);
  }
}
// Calls f with the activation as a constant: the choice is made once for many elements (a branch an element, unrolled, also overran the
// instruction cache: 300,000 x 256 -> 1024 in 1.11 ms).
template <typename F> __device__ __forceinline__ void with_activation(int act, F f) {
  if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
  else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>());
  else f(std::integral_constant<int, ACT_RELU>());
}
#endif

}  // namespace gphl

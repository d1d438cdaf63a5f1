// Gated feed-forward h = act(x Wg) * (x Wu) and its backward pass, on the product of tc_gemm.cu.
//
// Forward: one launch (two where k is split); a tile multiplies the same rows by columns of both weights, so that g and u of an element meet in one
// thread.  Backward: dg and du, then dx = [dg du] [Wg Wu]^T as one product
// over both pairs, and dWg, dWu as one launch of two.  dg and du come from g and u in fp32 (16-bit copies would add their
// rounding): either stored by the forward pass and read by an elementwise kernel, or made again by the forward's product with dh in its
// epilogue, which costs 4 m k f operations and saves 16 bytes an element.
//
// dg and du are rounded to 16 bits, as a gradient between two layers is: operands of 32 bits would halve the tensor core's rate and double the bytes of
// the step's largest tensors.  dx and dW are then off by 2.3e-3 (bf16) and 2.9e-4 (fp16) in the norm, with their own rounding alone by 1.7e-3 and 2.1e-4.
// In fp16 they also take its range: dh u act'(g) beyond 65504 is infinite, as where such a gradient is stored between two operators.
#include <algorithm>

#include "rows.cuh"
#include "tc_gemm.cuh"

namespace gphl {

// A thread per 8 columns of a row; dg and du have rows of ld (a multiple of 8), g and u of ld_gu (a multiple of 4).
template <typename T>
__global__ void __launch_bounds__(256) gate_grads_kernel(const T *__restrict__ dh, const float *__restrict__ g, const float *__restrict__ u, int64_t ld_gu,
                                                         int64_t m, int64_t f, int act, bool vec, T *__restrict__ dg, T *__restrict__ du, int64_t ld) {
  const int64_t units = ld / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / units, c = (i - row * units) * 8;
  if (row >= m) return;
  float a[8], gg[8], uu[8];
  const bool whole = c + 8 <= f;
  const T *src = dh + row * f + c;
  if (vec && whole) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(src);
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = to_float(reinterpret_cast<const T *>(&raw)[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = c + j < f ? to_float(src[j]) : 0.f;
  }
  const float *pg = g + row * ld_gu + c, *pu = u + row * ld_gu + c;
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    const bool in = c + j < f;                         // rows of g and u are padded to 4
    const float4 x = in ? *reinterpret_cast<const float4 *>(pg + j) : make_float4(0, 0, 0, 0);
    const float4 y = in ? *reinterpret_cast<const float4 *>(pu + j) : make_float4(0, 0, 0, 0);
    gg[j] = x.x, gg[j + 1] = x.y, gg[j + 2] = x.z, gg[j + 3] = x.w;
    uu[j] = y.x, uu[j + 1] = y.y, uu[j + 2] = y.z, uu[j + 3] = y.w;
  }
  uint4 og, ou;
  with_activation(act, [&](auto k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) gate_grads<decltype(k)::value>(a[j], gg[j], uu[j]);
  });
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    reinterpret_cast<T *>(&og)[j] = from_float<T>(gg[j]);
    reinterpret_cast<T *>(&ou)[j] = from_float<T>(uu[j]);
  }
  *reinterpret_cast<uint4 *>(dg + row * ld + c) = og;
  *reinterpret_cast<uint4 *>(du + row * ld + c) = ou;
}

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

static int gated_sizes(int32_t act, int64_t m, int64_t k, int64_t f) {
  GPHL_REQUIRE(m >= 0 && k >= 0 && f >= 0, "negative size");
  GPHL_REQUIRE(act >= GPHL_ACT_SILU && act <= GPHL_ACT_RELU, "gated: unknown activation %d", act);
  GPHL_REQUIRE(m < INT32_MAX - 256 && k <= (1 << 24) && f <= (1 << 24), "size out of range");
  return GPHL_OK;
}

static GemmCall forward_call(int dtype, int act, int64_t m, int64_t k, int64_t f) {
  GemmCall c;
  c.in_type = c.out_type = dtype, c.dual = DUAL_GATED, c.m = m, c.n = f, c.k = k, c.act = act, c.ld_out = f;
  return c;
}
static GemmCall grads_call(int dtype, int act, int64_t m, int64_t k, int64_t f) {
  GemmCall c = forward_call(dtype, act, m, k, f);
  c.dual = DUAL_GATED_GRAD, c.ld_out = up(f, 8);
  return c;
}
static GemmCall dx_call(int dtype, int64_t m, int64_t k, int64_t f) {
  GemmCall c;
  c.in_type = c.out_type = dtype, c.dual = DUAL_CONCAT, c.m = m, c.n = k, c.k = f, c.ld_out = k;
  return c;
}
// dW as the weights lie: (k, f) = x^T dg, or (f, k) = dg^T x
static GemmCall dw_call(int dtype, int64_t m, int64_t k, int64_t f, bool transposed) {
  GemmCall c;
  c.in_type = c.out_type = dtype, c.dual = DUAL_BATCH, c.a_mn = c.b_mn = true;
  c.m = transposed ? f : k, c.n = transposed ? k : f, c.k = m, c.ld_out = c.n;
  return c;
}

}  // namespace gphl

using namespace gphl;

extern "C" int64_t gphl_gated_workspace_bytes(int64_t m, int64_t k, int64_t f) { return gemm_workspace_bytes(forward_call(GPHL_BF16, 0, m, k, f)); }

extern "C" int gphl_gated(int32_t dtype, int32_t act, int64_t m, int64_t k, int64_t f, const void *x, int64_t ldx, const void *wg, const void *wu,
                          int64_t ldw, int32_t w_transposed, void *h, float *g, float *u, int64_t ld_gu, void *workspace, void *stream_) {
  int rc = gated_sizes(act, m, k, f);
  if (rc != GPHL_OK) return rc;
  GPHL_REQUIRE(dtype == GPHL_BF16 || dtype == GPHL_F16, "gated: bf16 or fp16 only");
  if (m == 0 || f == 0) return GPHL_OK;
  GPHL_REQUIRE(k > 0, "gated: the inner dimension is empty");
  GPHL_REQUIRE(x && wg && wu && h && !g == !u, "null pointer argument");
  GPHL_REQUIRE(ldx >= k && ldw >= (w_transposed ? k : f), "gated: rows are shorter than they hold");
  GPHL_REQUIRE(!g || (ld_gu >= f && ld_gu % 4 == 0 && aligned16(g) && aligned16(u)), "gated: rows of g and u must start on 16-byte boundaries");
  GemmCall c = forward_call(dtype, act, m, k, f);
  c.a[0] = {x, m, k, ldx};
  c.b_mn = !w_transposed;
  for (int i = 0; i < 2; ++i) c.b[i] = w_transposed ? Matrix{i ? wu : wg, f, k, ldw} : Matrix{i ? wu : wg, k, f, ldw};
  c.out[0] = h, c.g = g, c.u = u, c.ld_gu = ld_gu, c.workspace = workspace;
  return gemm(c, "gated", static_cast<cudaStream_t>(stream_));
}

// Workspace: dg and du, then the largest of the products' own.
extern "C" int64_t gphl_gated_grad_workspace_bytes(int64_t m, int64_t k, int64_t f) {
  if (m <= 0 || k <= 0 || f <= 0) return 0;
  const int64_t grads = 2 * up(m * up(f, 8) * 2, 256);
  return grads + std::max({gemm_workspace_bytes(grads_call(GPHL_BF16, 0, m, k, f)), gemm_workspace_bytes(dx_call(GPHL_BF16, m, k, f)),
                           gemm_workspace_bytes(dw_call(GPHL_BF16, m, k, f, false)), gemm_workspace_bytes(dw_call(GPHL_BF16, m, k, f, true))});
}

extern "C" int gphl_gated_grad(int32_t dtype, int32_t act, int64_t m, int64_t k, int64_t f, const void *dh, const float *g, const float *u, int64_t ld_gu,
                               const void *x, int64_t ldx, const void *wg, const void *wu, int64_t ldw, int32_t w_transposed, void *dx, void *dwg,
                               void *dwu, void *workspace, void *stream_) {
  int rc = gated_sizes(act, m, k, f);
  if (rc != GPHL_OK) return rc;
  GPHL_REQUIRE(dtype == GPHL_BF16 || dtype == GPHL_F16, "gated_grad: bf16 or fp16 only");
  GPHL_REQUIRE(!dwg == !dwu, "gated_grad: the weights' gradients are wanted together");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (m == 0 || k == 0 || f == 0) {                    // sums of nothing
    if (dx && m > 0 && k > 0) GPHL_CUDA(cudaMemsetAsync(dx, 0, (size_t)(m * k * 2), stream));
    if (dwg && k > 0 && f > 0) {
      GPHL_CUDA(cudaMemsetAsync(dwg, 0, (size_t)(k * f * 2), stream));
      GPHL_CUDA(cudaMemsetAsync(dwu, 0, (size_t)(k * f * 2), stream));
    }
    return GPHL_OK;
  }
  GPHL_REQUIRE(dh && !g == !u && workspace && ((!dx && g) || (wg && wu)) && ((!dwg && g) || x), "null pointer argument");
  GPHL_REQUIRE(ldx >= k && ldw >= (w_transposed ? k : f), "gated_grad: rows are shorter than they hold");
  GPHL_REQUIRE(!g || (ld_gu >= f && ld_gu % 4 == 0 && aligned16(g) && aligned16(u)), "gated_grad: rows of g and u must start on 16-byte boundaries");
  GPHL_REQUIRE(aligned16(workspace), "gated_grad: the workspace must start on a 16-byte boundary");
  const int64_t ld = up(f, 8), bytes = up(m * ld * 2, 256);
  char *dg = static_cast<char *>(workspace), *du = dg + bytes, *rest = du + bytes;
  const Matrix rows{x, m, k, ldx};
  Matrix w[2];
  for (int i = 0; i < 2; ++i) w[i] = w_transposed ? Matrix{i ? wu : wg, f, k, ldw} : Matrix{i ? wu : wg, k, f, ldw};
  if (g) {
    const int64_t threads = m * (ld / 8);
    GPHL_REQUIRE(threads < (int64_t)INT32_MAX * 256, "size out of range");
    const bool vec = f % 8 == 0 && aligned16(dh);
    const unsigned grid = (unsigned)((threads + 255) / 256);
    if (dtype == GPHL_BF16)
      gate_grads_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16 *>(dh), g, u, ld_gu, m, f, act, vec,
                                                                 reinterpret_cast<__nv_bfloat16 *>(dg), reinterpret_cast<__nv_bfloat16 *>(du), ld);
    else
      gate_grads_kernel<__half><<<grid, 256, 0, stream>>>(static_cast<const __half *>(dh), g, u, ld_gu, m, f, act, vec, reinterpret_cast<__half *>(dg),
                                                          reinterpret_cast<__half *>(du), ld);
    rc = launched("gate_grads_kernel");
  } else {
    GemmCall c = grads_call(dtype, act, m, k, f);
    c.a[0] = rows, c.b[0] = w[0], c.b[1] = w[1], c.b_mn = !w_transposed;
    c.dh = dh, c.out[0] = dg, c.out[1] = du, c.workspace = rest;
    rc = gemm(c, "gated_grad", stream);
  }
  if (rc != GPHL_OK) return rc;
  const Matrix grads[2] = {{dg, m, f, ld}, {du, m, f, ld}};
  if (dx) {
    GemmCall c = dx_call(dtype, m, k, f);
    c.b_mn = w_transposed;
    for (int i = 0; i < 2; ++i) c.a[i] = grads[i], c.b[i] = w[i];
    c.out[0] = dx, c.workspace = rest;
    rc = gemm(c, "gated_grad", stream);
    if (rc != GPHL_OK) return rc;
  }
  if (dwg) {
    GemmCall c = dw_call(dtype, m, k, f, w_transposed);
    for (int i = 0; i < 2; ++i) c.a[i] = w_transposed ? grads[i] : rows, c.b[i] = w_transposed ? rows : grads[i];
    c.out[0] = dwg, c.out[1] = dwu, c.workspace = rest;
    rc = gemm(c, "gated_grad", stream);
  }
  return rc;
}

static GemmCall fp8_call(int act, int64_t m, int64_t k, int64_t f, uint8_t *q) {
  GemmCall c;
  c.fp8 = true, c.dual = DUAL_GATED, c.m = m, c.n = f, c.k = k, c.act = act, c.q = q;
  return c;
}

extern "C" int64_t gphl_gated_fp8_workspace_bytes(int64_t m, int64_t k, int64_t f, int32_t codes_out) {
  uint8_t any = 0;
  return gemm_workspace_bytes(fp8_call(0, m, k, f, codes_out ? &any : nullptr));
}

extern "C" int gphl_gated_fp8(int32_t act, int64_t m, int64_t k, int64_t f, const void *x, int64_t x_stride, const float *x_scales,
                              int64_t scale_row_stride, int64_t scale_block_stride, const void *wg, const float *wg_scales, const void *wu,
                              const float *wu_scales, int64_t w_stride, int32_t out_dtype, void *h, void *q, int64_t q_stride, float *scales,
                              int64_t scale_stride, void *workspace, void *stream_) {
  int rc = gated_sizes(act, m, k, f);
  if (rc != GPHL_OK) return rc;
  GPHL_REQUIRE(out_dtype >= GPHL_F32 && out_dtype <= GPHL_F16, "gated_fp8: unknown type %d", out_dtype);
  if (m == 0 || f == 0) return GPHL_OK;
  GPHL_REQUIRE(k > 0, "gated_fp8: the inner dimension is empty");
  GPHL_REQUIRE(x && x_scales && wg && wg_scales && wu && wu_scales && (h || q) && (!q || scales), "null pointer argument");
  GPHL_REQUIRE(x_stride >= k && w_stride >= k, "gated_fp8: code rows are shorter than k");
  GPHL_REQUIRE(!q || (q_stride == up(f, 16) && aligned16(q) && scale_stride >= m), "gated_fp8: code rows must be 16-byte aligned and padded to 16 bytes");
  GemmCall c = fp8_call(act, m, k, f, static_cast<uint8_t *>(q));
  c.a[0] = {x, m, k, x_stride}, c.b[0] = {wg, f, k, w_stride}, c.b[1] = {wu, f, k, w_stride};
  c.a_scale = x_scales, c.a_scale_row = scale_row_stride, c.a_scale_block = scale_block_stride;
  c.b_scale[0] = wg_scales, c.b_scale[1] = wu_scales;
  c.out[0] = h, c.out_type = out_dtype, c.ld_out = q ? q_stride : f;
  c.q_scale = scales, c.q_scale_stride = scale_stride, c.workspace = workspace;
  return gemm(c, "gated_fp8", static_cast<cudaStream_t>(stream_));
}

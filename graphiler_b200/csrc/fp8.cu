// e4m3 rows and weights with a scale per block of 128, and the typed product of the two.
//
// The quantisers read every value once: a few steps of a row a warp, a block per 128 x 128 tile for weights, which turns the
// tile round in shared memory (segment_mm's weights have n contiguous, the product reads k contiguous).  Scales are powers of two, so that
// scaling rounds nothing and a code is the rounding of the value itself.
#include <algorithm>

#include "rows.cuh"
#include "tc_gemm.cuh"

namespace gphl {

// NV steps of a row a warp (32 / LPR rows), all loads first.
template <typename T, typename R, int NV>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T *__restrict__ x, int64_t m, int32_t n, uint8_t *__restrict__ q, int32_t n_pad,
                                                            float *__restrict__ scales, int64_t scale_stride) {
  constexpr int RPW = 32 / R::LPR;
  const int lane = threadIdx.x & (R::LPR - 1), groups = (n + R::STEP * NV - 1) / (R::STEP * NV);
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), first = item / groups;
  const int step0 = (int)(item - first * groups) * NV;
  const int64_t at = first * RPW + (threadIdx.x & 31) / R::LPR, row = min(at, m - 1);      // rows past the last store nothing
  typename R::Raw v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = R::raw(x + row * n, step0 + i, lane, n);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float y[R::E];
    R::widen(v[i], y);
    if (i == 0 || (step0 + i) * R::STEP < n_pad) store_codes<R>(y, q + row * n_pad, scales + row, scale_stride, step0 + i, lane, n, n_pad, at < m);
  }
}

constexpr int TILE_LD = 132;                          // bytes from n to n in shared memory: 4 more than a row, so that stores spread over the banks

template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const T *__restrict__ w, int64_t k, int64_t n, uint8_t *__restrict__ q, int64_t k_stride,
                                                              float *__restrict__ scales) {
  __shared__ uint32_t tile[128 * TILE_LD / 4];
  __shared__ float s_max[8];
  const int64_t kb = blockIdx.x, nb = blockIdx.y, t = blockIdx.z, k0 = kb * 128, n0 = nb * 128;
  const int col = threadIdx.x & 127, part = threadIdx.x >> 7;      // this thread: column n0 + col, four rows of k at a time
  const T *src = w + t * k * n + n0 + col;
  const bool ok = n0 + col < n;
  float v[64], big = 0.f;
#pragma unroll
  for (int i = 0; i < 64; ++i) {
    const int64_t r = k0 + (i >> 2) * 8 + part * 4 + (i & 3);
    v[i] = ok && r < k ? to_float(src[r * n]) : 0.f;
    big = fmaxf(big, finite_abs(v[i]));
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) big = fmaxf(big, __shfl_xor_sync(FULL, big, d));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = big;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) big = fmaxf(big, s_max[i]);
  const int e = fp8_exponent(big);
  const float inv = pow2f(-e);
#pragma unroll
  for (int i = 0; i < 64; i += 4)
    tile[(col * TILE_LD + (i >> 2) * 8 + part * 4) / 4] = e4m3x2(v[i] * inv, v[i + 1] * inv) | (e4m3x2(v[i + 2] * inv, v[i + 3] * inv) << 16);
  if (threadIdx.x == 0) scales[(t * gridDim.y + nb) * gridDim.x + kb] = pow2f(e);
  __syncthreads();
  // rows of n leave as 128-byte segments; k_stride is a multiple of 16, so a word inside [k0, k_stride) is inside the row
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < 128; r += 8)
    if (n0 + r < n && k0 + lane * 4 < k_stride)
      *reinterpret_cast<uint32_t *>(q + (t * n + n0 + r) * k_stride + k0 + lane * 4) = tile[r * (TILE_LD / 4) + lane];
}

// Rows of codes start on 16-byte boundaries.  VEC: a thread per 16 neighbouring codes.  Otherwise a warp per 512 columns of a row, columns 32
// apart, so that stores to rows of any width and base are still whole lines.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t *__restrict__ q, int64_t q_stride, const float *__restrict__ scales,
                                                         int64_t row_stride, int64_t block_stride, int64_t m, int32_t n, T *__restrict__ y) {
  auto value = [](uint8_t code) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3))); };
  if constexpr (VEC) {
    const int64_t units = (n + 15) / 16, i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / units;
    const int c0 = (int)(i - row * units) * 16;        // n is a multiple of 8
    if (row >= m) return;
    const uint8_t *src = q + row * q_stride + c0;
    const float s = __ldg(scales + row * row_stride + (c0 / 128) * block_stride);
    __align__(16) uint8_t code[16];
    if (c0 + 16 <= n) *reinterpret_cast<uint4 *>(code) = *reinterpret_cast<const uint4 *>(src);
    else *reinterpret_cast<uint2 *>(code) = *reinterpret_cast<const uint2 *>(src);
    __align__(16) T out[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) out[j] = from_float<T>(c0 + j < n ? value(code[j]) * s : 0.f);
    T *dst = y + row * n + c0;
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); ++j)
      if (c0 + (j + 1) * 16 / (int)sizeof(T) <= n) reinterpret_cast<uint4 *>(dst)[j] = reinterpret_cast<const uint4 *>(out)[j];
  } else {
    const int lane = threadIdx.x & 31, steps = (n + 511) / 512;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), row = item / steps;
    const int base = (int)(item - row * steps) * 512;
    if (row >= m) return;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int c = base + lane + 32 * j;
      if (c < n) y[row * n + c] = from_float<T>(value(q[row * q_stride + c]) * __ldg(scales + row * row_stride + (c / 128) * block_stride));
    }
  }
}

// Rows of n 16-bit values to rows of n_pad: a thread per 8 values of the padded rows.
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t *__restrict__ x, int64_t m, int64_t n, uint16_t *__restrict__ y, int64_t units) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / units, c = (i - row * units) * 8;
  if (row >= m) return;
  uint16_t v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < n ? __ldg(x + row * n + c + j) : (uint16_t)0;
  *reinterpret_cast<uint4 *>(y + row * units * 8 + c) = *reinterpret_cast<const uint4 *>(v);
}

static bool known(int dtype) { return dtype >= GPHL_F32 && dtype <= GPHL_F16; }

template <typename T> static void quantize(const void *x, int64_t m, int64_t n, void *q, int64_t n_pad, float *scales, int64_t stride, cudaStream_t s) {
  const bool vec = aligned16(x) && n % (16 / (int)sizeof(T)) == 0;
  with_lanes<T>(n, vec, [&](auto r) {
    using R = decltype(r);
    auto launch = [&](auto nv) {
      constexpr int RPW = 32 / R::LPR, NV = decltype(nv)::value;
      const int64_t items = ((m + RPW - 1) / RPW) * ((n + R::STEP * NV - 1) / (R::STEP * NV));
      quantize_rows_kernel<T, R, NV><<<(unsigned)((items + 7) / 8), 256, 0, s>>>(static_cast<const T *>(x), m, (int32_t)n, static_cast<uint8_t *>(q),
                                                                                (int32_t)n_pad, scales, stride);
    };
    // several loads under way per lane where rows have them (32768 x 8192 in bf16: 148 against 253 us)
    if constexpr (R::LPR == 32) {
      if (n > 2 * R::STEP) return launch(std::integral_constant<int, 4>());
    }
    launch(std::integral_constant<int, 1>());
  });
}
template <typename T>
static void dequantize(const void *q, int64_t q_stride, const float *scales, int64_t row_stride, int64_t block_stride, int64_t m, int64_t n, void *y, cudaStream_t s) {
  if (aligned16(y) && n % 8 == 0)
    dequantize_kernel<T, true><<<(unsigned)((m * ((n + 15) / 16) + 255) / 256), 256, 0, s>>>(static_cast<const uint8_t *>(q), q_stride, scales, row_stride, block_stride,
                                                                                            m, (int32_t)n, static_cast<T *>(y));
  else
    dequantize_kernel<T, false><<<(unsigned)((m * ((n + 511) / 512) + 7) / 8), 256, 0, s>>>(static_cast<const uint8_t *>(q), q_stride, scales, row_stride, block_stride, m, (int32_t)n, static_cast<T *>(y));
}

}  // namespace gphl

using namespace gphl;

extern "C" int gphl_quantize_fp8(int32_t dtype, int64_t m, int64_t n, const void *x, void *q, int64_t q_stride, float *scales, int64_t scale_stride,
                                 void *stream_) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(known(dtype), "quantize_fp8: unknown type %d", dtype);
  GPHL_REQUIRE(m < INT32_MAX && n <= (1 << 24) && m * ((n + 127) / 128) < (int64_t)INT32_MAX * 8, "size out of range");
  if (m == 0 || n == 0) return GPHL_OK;
  GPHL_REQUIRE(x && q && scales, "null pointer argument");
  GPHL_REQUIRE(q_stride == (n + 15) / 16 * 16 && aligned16(q), "quantize_fp8: code rows must be 16-byte aligned and padded to 16 bytes");
  GPHL_REQUIRE(scale_stride >= m, "quantize_fp8: scale_stride must be at least the number of rows");
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if (dtype == GPHL_F32) quantize<float>(x, m, n, q, q_stride, scales, scale_stride, s);
  else if (dtype == GPHL_BF16) quantize<__nv_bfloat16>(x, m, n, q, q_stride, scales, scale_stride, s);
  else quantize<__half>(x, m, n, q, q_stride, scales, scale_stride, s);
  return launched("quantize_rows_kernel");
}

extern "C" int gphl_quantize_fp8_weight(int32_t dtype, int64_t n_types, int64_t k, int64_t n, const void *w, void *q, int64_t k_stride, float *scales,
                                        void *stream_) {
  GPHL_REQUIRE(n_types >= 0 && k >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(known(dtype), "quantize_fp8_weight: unknown type %d", dtype);
  GPHL_REQUIRE(n_types <= 65535 && k <= (1 << 24) && n <= 65535 * 128LL, "size out of range");
  if (n_types == 0 || k == 0 || n == 0) return GPHL_OK;
  GPHL_REQUIRE(w && q && scales, "null pointer argument");
  GPHL_REQUIRE(k_stride == (k + 15) / 16 * 16 && aligned16(q), "quantize_fp8_weight: code rows must be 16-byte aligned and padded to 16 bytes");
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  const dim3 grid((unsigned)((k + 127) / 128), (unsigned)((n + 127) / 128), (unsigned)n_types);
  uint8_t *o = static_cast<uint8_t *>(q);
  if (dtype == GPHL_F32) quantize_weight_kernel<float><<<grid, 256, 0, s>>>(static_cast<const float *>(w), k, n, o, k_stride, scales);
  else if (dtype == GPHL_BF16) quantize_weight_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(static_cast<const __nv_bfloat16 *>(w), k, n, o, k_stride, scales);
  else quantize_weight_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half *>(w), k, n, o, k_stride, scales);
  return launched("quantize_weight_kernel");
}

extern "C" int gphl_dequantize_fp8(int32_t dtype, int64_t m, int64_t n, const void *q, int64_t q_stride, const float *scales, int64_t scale_row_stride,
                                   int64_t scale_block_stride, void *y, void *stream_) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(known(dtype), "dequantize_fp8: unknown type %d", dtype);
  GPHL_REQUIRE(m < INT32_MAX && n <= (1 << 24) && m * ((n + 511) / 512) < (int64_t)INT32_MAX * 8, "size out of range");
  if (m == 0 || n == 0) return GPHL_OK;
  GPHL_REQUIRE(q && scales && y, "null pointer argument");
  GPHL_REQUIRE(q_stride >= n && q_stride % 16 == 0 && aligned16(q), "dequantize_fp8: code rows must start on 16-byte boundaries");
  cudaStream_t s = static_cast<cudaStream_t>(stream_);
  if (dtype == GPHL_F32) dequantize<float>(q, q_stride, scales, scale_row_stride, scale_block_stride, m, n, y, s);
  else if (dtype == GPHL_BF16) dequantize<__nv_bfloat16>(q, q_stride, scales, scale_row_stride, scale_block_stride, m, n, y, s);
  else dequantize<__half>(q, q_stride, scales, scale_row_stride, scale_block_stride, m, n, y, s);
  return launched("dequantize_kernel");
}

extern "C" int gphl_pad_rows_16(int64_t m, int64_t n, const void *x, void *y, void *stream_) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  if (m == 0 || n == 0) return GPHL_OK;
  const int64_t units = (n + 7) / 8;
  GPHL_REQUIRE(m * units < (int64_t)INT32_MAX * 256, "size out of range");
  GPHL_REQUIRE(x && y && aligned16(y), "null or unaligned pointer argument");
  pad_rows_kernel<<<(unsigned)((m * units + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream_)>>>(static_cast<const uint16_t *>(x), m, n,
                                                                                                     static_cast<uint16_t *>(y), units);
  return launched("pad_rows_kernel");
}

static int mm_fp8_sizes(int64_t n_types, int64_t m, int64_t k, int64_t n) {
  GPHL_REQUIRE(n_types >= 0 && m >= 0 && k >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(m < INT32_MAX - 256 && k <= (1 << 24) && n <= (1 << 24) && n_types < (1 << 20) && n_types * n < INT32_MAX - 256, "size out of range");
  return GPHL_OK;
}

extern "C" int64_t gphl_segment_mm_fp8_workspace_bytes(int64_t n_types, int32_t typed, int64_t m, int64_t k, int64_t n) {
  static const int32_t any = 0;
  GemmCall c;
  c.fp8 = true, c.m = m, c.n = n, c.k = k, c.types = n_types, c.ptr = typed ? &any : nullptr;
  return n_types > 0 ? gemm_workspace_bytes(c) : 0;
}

extern "C" int gphl_segment_mm_fp8(int64_t n_types, const int32_t *type_pointer, int64_t m, int64_t k, int64_t n, const void *x, int64_t x_stride,
                                   const float *x_scales, int64_t scale_row_stride, int64_t scale_block_stride, const void *w, int64_t w_stride,
                                   const float *w_scales, int32_t out_dtype, void *y, void *workspace, void *stream_) {
  int rc = mm_fp8_sizes(n_types, m, k, n);
  if (rc != GPHL_OK) return rc;
  GPHL_REQUIRE(known(out_dtype), "segment_mm_fp8: unknown type %d", out_dtype);
  GPHL_REQUIRE(type_pointer || n_types == 1, "segment_mm_fp8: several types need a type pointer");
  if (m == 0 || n == 0 || n_types == 0) return GPHL_OK;
  GPHL_REQUIRE(y && (k == 0 || (x && x_scales && w && w_scales)), "null pointer argument");
  GPHL_REQUIRE(x_stride >= k && w_stride >= k, "segment_mm_fp8: code rows are shorter than k");
  GemmCall c;
  c.fp8 = true, c.m = m, c.n = n, c.k = k, c.types = n_types, c.ptr = type_pointer;
  c.a[0] = {x, m, k, x_stride}, c.b[0] = {w, n_types * n, k, w_stride};
  c.a_scale = x_scales, c.a_scale_row = scale_row_stride, c.a_scale_block = scale_block_stride, c.b_scale[0] = w_scales;
  c.out[0] = y, c.ld_out = n, c.out_type = out_dtype, c.workspace = workspace;
  return gemm(c, "segment_mm_fp8", static_cast<cudaStream_t>(stream_));
}

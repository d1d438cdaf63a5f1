// Root-mean-square norm of rows, with the residual's addition:
//   r = round(x + residual)   (kept in the rows' type: what the next layer adds to is what is normalised)
//   y = r * rstd * w,   rstd = 1 / sqrt(mean(r^2) + eps)
// y in the rows' type, or as e4m3 codes with one power-of-two scale per row and block of 128 columns.  Backward, from r and rstd:
//   g = dy * w, xhat = r * rstd, dx = dr + rstd * (g - xhat * mean(g * xhat)), dw = sum over rows of dy * xhat.
//
// Memory bound.  A row is read once and stays in registers: WPR warps hold it, up to NV steps each (a step is 32 lanes x 16 bytes); the
// sum of squares is kept in fp32 by every lane (at most 32 terms) and joined in double.  Rows too wide for that are read twice.
#include <algorithm>
#include <initializer_list>

#include "rows.cuh"

namespace gphl {

struct NormArgs {
  const void *x, *res, *w;
  void *y, *r;
  uint8_t *q;               // e4m3 codes, row stride n_pad
  float *scales;            // scale of (row, block) at block * scale_stride + row
  float *rstd;
  int64_t m, scale_stride;
  int32_t n, n_pad, wpr, w_f32;
  float eps;
};

// Joins `v` over the warps of a row (all threads of the block when wpr > 1).
__device__ __forceinline__ double row_sum(double v, int wpr, int warp, int lane, double *s_part) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
  if (wpr == 1) return v;
  if (lane == 0) s_part[warp] = v;
  __syncthreads();
  v = lane < wpr ? s_part[lane] : 0.0;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
  __syncthreads();                                   // s_part may be written again
  return v;
}

// Correct rounding of v * w * rstd / scale to e4m3 where the fp32 value is too close to a border between two codes: the product in
// double, brought to fp32 by rounding to odd, which leaves the second rounding unbiased.
__device__ __noinline__ uint32_t e4m3_near_border(float v, float w, double rstd, float inv) {
  const double t = (double)v * (double)w * rstd * (double)inv;
  float f = __double2float_rz(t);
  if ((double)f != t) f = __uint_as_float(__float_as_uint(f) | 1u);
  return e4m3(f);
}

// NV > 0: the row is held in registers.  NV == 0: any width, the row is read twice.
template <typename T, bool SC, int NV, bool FP8>
__global__ void __launch_bounds__(512) rms_norm_kernel(const NormArgs a) {
  using R = Row<T, SC>;
  constexpr int E = R::E;
  __shared__ double s_part[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_block = (blockDim.x >> 5) / a.wpr;   // rows of a block: several one-warp rows, or one row
  const int64_t row = (int64_t)blockIdx.x * per_block + warp / a.wpr;
  if (row >= a.m) return;                            // whole warps, and only in blocks of one-warp rows
  const int w0 = warp % a.wpr, steps = (a.n + R::STEP - 1) / R::STEP;
  const T *x = static_cast<const T *>(a.x) + row * a.n;
  const T *res = a.res ? static_cast<const T *>(a.res) + row * a.n : nullptr;
  T *r = a.r ? static_cast<T *>(a.r) + row * a.n : nullptr;

  constexpr int KEEP = NV > 0 ? NV : 1;
  float v[KEEP][E];
  float ss = 0.f;
  double wide = 0.0;
  auto read = [&](int step, float (&t)[E]) {
    R::load(x, step, lane, a.n, t);
    if (res) {
      float u[E];
      R::load(res, step, lane, a.n, u);
#pragma unroll
      for (int j = 0; j < E; ++j) t[j] = to_float(from_float<T>(t[j] + u[j]));
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) read(step, v[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        if (r) R::store(r, step, lane, a.n, v[i]);
#pragma unroll
        for (int j = 0; j < E; ++j) ss = fmaf(v[i][j], v[i][j], ss);
      }
    }
    wide = (double)ss;
  } else {
    for (int step = w0; step < steps; step += a.wpr) {
      read(step, v[0]);
      if (r) R::store(r, step, lane, a.n, v[0]);
      ss = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) ss = fmaf(v[0][j], v[0][j], ss);
      wide += (double)ss;
    }
  }
  const double rstd_d = 1.0 / sqrt(row_sum(wide, a.wpr, warp, lane, s_part) / a.n + (double)a.eps);
  const float rstd = (float)rstd_d;
  if (a.rstd && w0 == 0 && lane == 0) a.rstd[row] = rstd;

  auto write = [&](int step, const float (&t)[E]) {
    float w[E], y[E];
    if (a.w_f32) R::load(static_cast<const float *>(a.w), step, lane, a.n, w);
    else R::load(static_cast<const T *>(a.w), step, lane, a.n, w);
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = t[j] * rstd * w[j];
    if constexpr (FP8) {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) big = fmaxf(big, finite_abs(y[j]));
      const int e = fp8_exponent(block_max<T, SC>(big));
      const float inv = pow2f(-e);
      uint32_t q[E];
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        // y carries three fp32 roundings (at most 3 x 2^-24 relative): if both ends of a wider interval have one code, it is the code
        const float s0 = y[j] * inv, s1 = y[j + 1] * inv;
        const uint32_t up = e4m3x2(s0 * (1.f + 0x1p-21f), s1 * (1.f + 0x1p-21f));
        const uint32_t dn = e4m3x2(s0 * (1.f - 0x1p-21f), s1 * (1.f - 0x1p-21f));
        q[j] = up & 0xff, q[j + 1] = up >> 8;
        if (up != dn) {
          q[j] = e4m3_near_border(t[j], w[j], rstd_d, inv);
          q[j + 1] = e4m3_near_border(t[j + 1], w[j + 1], rstd_d, inv);
        }
      }
      store_codes<T, SC>(a.q + row * a.n_pad, step, lane, a.n, a.n_pad, q);
      constexpr int LANES = 128 / E;
      const int block = R::col(step, lane, 0) / 128;
      if (lane % LANES == 0 && block * 128 < a.n) a.scales[block * a.scale_stride + row] = pow2f(e);
    } else {
      R::store(static_cast<T *>(a.y) + row * a.n, step, lane, a.n, y);
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) write(step, v[i]);
    }
  } else {
    for (int step = w0; step < steps; step += a.wpr) {
      if (r) R::load(r, step, lane, a.n, v[0]);      // this thread's own stores
      else read(step, v[0]);
      write(step, v[0]);
    }
  }
}

struct NormGradArgs {
  const void *r, *w, *dy, *dr;
  const float *rstd;
  void *dx;
  float *part;              // (gridDim.x, n) partial sums of dw
  int64_t m;
  int32_t n, wpr, w_f32;
};

// Rows are dealt to warps (or, for wpr > 1, to blocks) in turn; a lane keeps its columns, so dw gathers in its registers over all the
// rows it meets and leaves once.  The rows' sums g.xhat are joined in double.
template <typename T, bool SC, int NV>
__global__ void __launch_bounds__(512) rms_norm_grad_kernel(const NormGradArgs a) {
  using R = Row<T, SC>;
  constexpr int E = R::E;
  __shared__ double s_part[16];
  extern __shared__ float s_dw[];                    // wpr == 1: one row of n sums per warp
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_block = warps / a.wpr, w0 = warp % a.wpr, steps = (a.n + R::STEP - 1) / R::STEP;
  float dw[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) dw[i][j] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * per_block + warp / a.wpr; row < a.m; row += (int64_t)gridDim.x * per_block) {
    const T *r = static_cast<const T *>(a.r) + row * a.n, *dy = static_cast<const T *>(a.dy) + row * a.n;
    const T *dr = a.dr ? static_cast<const T *>(a.dr) + row * a.n : nullptr;
    const float rstd = __ldg(a.rstd + row);
    float xh[NV][E], g[NV][E];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        R::load(r, step, lane, a.n, xh[i]);
        R::load(dy, step, lane, a.n, g[i]);
      }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        float w[E], part = 0.f;
        if (a.w_f32) R::load(static_cast<const float *>(a.w), step, lane, a.n, w);
        else R::load(static_cast<const T *>(a.w), step, lane, a.n, w);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          xh[i][j] *= rstd;
          dw[i][j] = fmaf(g[i][j], xh[i][j], dw[i][j]);
          g[i][j] *= w[j];
          part = fmaf(g[i][j], xh[i][j], part);
        }
        sum += (double)part;
      }
    }
    const float mean = (float)(row_sum(sum, a.wpr, warp, lane, s_part) / a.n);
    T *dx = static_cast<T *>(a.dx) + row * a.n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        float o[E];
        if (dr) R::load(dr, step, lane, a.n, o);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float t = rstd * fmaf(-xh[i][j], mean, g[i][j]);
          o[j] = dr ? o[j] + t : t;
        }
        R::store(dx, step, lane, a.n, o);
      }
    }
  }
  float *part = a.part + (int64_t)blockIdx.x * a.n;
  if (a.wpr > 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = R::col(w0 + i * a.wpr, lane, j);
        if (c < a.n) part[c] = dw[i][j];
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = R::col(i, lane, j);
      if (c < a.n) s_dw[warp * a.n + c] = dw[i][j];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < warps; ++k) s += s_dw[k * a.n + c];
    part[c] = s;
  }
}

// Rows wider than the registers of 16 warps: one block per row reads its inputs twice; dw is left to rms_norm_dw_wide_kernel.
template <typename T, bool SC>
__global__ void __launch_bounds__(512) rms_norm_grad_wide_kernel(const NormGradArgs a) {
  using R = Row<T, SC>;
  constexpr int E = R::E;
  __shared__ double s_part[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, steps = (a.n + R::STEP - 1) / R::STEP;
  const int64_t row = blockIdx.x;
  const T *r = static_cast<const T *>(a.r) + row * a.n, *dy = static_cast<const T *>(a.dy) + row * a.n;
  const T *dr = a.dr ? static_cast<const T *>(a.dr) + row * a.n : nullptr;
  T *dx = static_cast<T *>(a.dx) + row * a.n;
  const float rstd = __ldg(a.rstd + row);
  float xh[E], g[E], w[E];
  auto read = [&](int step) {
    R::load(r, step, lane, a.n, xh);
    R::load(dy, step, lane, a.n, g);
    if (a.w_f32) R::load(static_cast<const float *>(a.w), step, lane, a.n, w);
    else R::load(static_cast<const T *>(a.w), step, lane, a.n, w);
#pragma unroll
    for (int j = 0; j < E; ++j) xh[j] *= rstd, g[j] *= w[j];
  };
  double sum = 0.0;
  for (int step = warp; step < steps; step += a.wpr) {
    read(step);
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) part = fmaf(g[j], xh[j], part);
    sum += (double)part;
  }
  const float mean = (float)(row_sum(sum, a.wpr, warp, lane, s_part) / a.n);
  for (int step = warp; step < steps; step += a.wpr) {
    read(step);
    float o[E];
    if (dr) R::load(dr, step, lane, a.n, o);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float t = rstd * fmaf(-xh[j], mean, g[j]);
      o[j] = dr ? o[j] + t : t;
    }
    R::store(dx, step, lane, a.n, o);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_dw_wide_kernel(const NormGradArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.n) return;
  float s = 0.f;
  for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const int64_t i = row * a.n + c;
    s = fmaf(to_float(static_cast<const T *>(a.dy)[i]), to_float(static_cast<const T *>(a.r)[i]) * __ldg(a.rstd + row), s);
  }
  a.part[(int64_t)blockIdx.y * a.n + c] = s;
}

// dw = the partial sums' sum, in a fixed order, in double.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_dw_kernel(const float *__restrict__ part, int32_t parts, int32_t n, T *__restrict__ dw) {
  __shared__ double s[8][33];
  const int lane = threadIdx.x & 31, k0 = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < n)
    for (int k = k0; k < parts; k += 8) v += (double)part[(int64_t)k * n + c];
  s[k0][lane] = v;
  __syncthreads();
  if (k0 == 0 && c < n) {
    for (int k = 1; k < 8; ++k) v += s[k][lane];
    dw[c] = from_float<T>((float)v);
  }
}

static int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

template <typename T, bool SC, int NV, bool FP8> static void norm_launch(const NormArgs &a, int warps, cudaStream_t s) {
  const int per_block = warps / a.wpr;
  rms_norm_kernel<T, SC, NV, FP8><<<(unsigned)((a.m + per_block - 1) / per_block), warps * 32, 0, s>>>(a);
}
template <typename T, bool SC, bool FP8> static void norm_dispatch(NormArgs a, int sms, cudaStream_t s) {
  using R = Row<T, SC>;
  constexpr int LOW = 8 / R::E, HIGH = 32 / R::E;    // steps a warp holds: 8 or 32 values a lane
  const int steps = (a.n + R::STEP - 1) / R::STEP;
  // Few warps a row leave most loads in flight per warp and need the fewest joins; when the rows would not fill the GPU with 8 warps an
  // SM that way, a row is spread over more warps instead (one row of 4096 columns, 16 bits: 2.3 us with 4 warps, 2.0 us with 16).
  int wpr = pow2_at_least((steps + HIGH - 1) / HIGH);
  const bool few = a.m * wpr < 8 * sms;
  if (few) wpr = std::min(16, pow2_at_least((steps + LOW - 1) / LOW));
  a.wpr = std::min(wpr, 16);
  const int warps = a.wpr == 1 ? 4 : a.wpr;
  if (steps <= a.wpr * LOW) norm_launch<T, SC, LOW, FP8>(a, warps, s);
  else if (steps <= a.wpr * HIGH) norm_launch<T, SC, HIGH, FP8>(a, warps, s);
  else norm_launch<T, SC, 0, FP8>(a, warps, s);
}
template <bool FP8> static void norm_types(const NormArgs &a, int dtype, bool vec, int sms, cudaStream_t s) {
  if (dtype == GPHL_F32) vec ? norm_dispatch<float, false, FP8>(a, sms, s) : norm_dispatch<float, true, FP8>(a, sms, s);
  else if (dtype == GPHL_BF16) vec ? norm_dispatch<__nv_bfloat16, false, FP8>(a, sms, s) : norm_dispatch<__nv_bfloat16, true, FP8>(a, sms, s);
  else vec ? norm_dispatch<__half, false, FP8>(a, sms, s) : norm_dispatch<__half, true, FP8>(a, sms, s);
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n;
}

struct GradShape {
  int wpr, warps, grid, nv;
  size_t smem;
};
// E: values of a lane's step.  At most 16 values a lane are held (registers: two row operands and the gathering dw); nv == 0: wider.
static GradShape grad_shape(int64_t m, int n, int e, int sms) {
  const int steps = (n + 32 * e - 1) / (32 * e), hold = 16 / e;
  GradShape g{};
  g.wpr = pow2_at_least((steps + hold - 1) / hold);
  if (g.wpr > 16) {
    g.wpr = 16, g.warps = 16, g.nv = 0;
    g.grid = (int)std::min<int64_t>(m, 64);          // row groups of the separate dw kernel
    return g;
  }
  g.nv = steps <= g.wpr * (hold / 2) ? hold / 2 : hold;
  g.warps = g.wpr == 1 ? 8 : g.wpr;
  const int per_block = g.warps / g.wpr;
  // 32 warps an SM: the partial rows of dw stay few
  g.grid = (int)std::min<int64_t>((m + per_block - 1) / per_block, (int64_t)sms * (32 / g.warps));
  g.smem = g.wpr == 1 ? (size_t)g.warps * n * sizeof(float) : 0;
  return g;
}
template <typename T, bool SC> static void grad_launch(NormGradArgs a, const GradShape &g, cudaStream_t s) {
  constexpr int HOLD = 16 / Row<T, SC>::E;
  a.wpr = g.wpr;
  if (g.nv == 0) {
    rms_norm_grad_wide_kernel<T, SC><<<(unsigned)a.m, 512, 0, s>>>(a);
    rms_norm_dw_wide_kernel<T><<<dim3((unsigned)((a.n + 255) / 256), (unsigned)g.grid), 256, 0, s>>>(a);
  } else if (g.nv == HOLD) {
    rms_norm_grad_kernel<T, SC, HOLD><<<g.grid, g.warps * 32, g.smem, s>>>(a);
  } else {
    rms_norm_grad_kernel<T, SC, HOLD / 2><<<g.grid, g.warps * 32, g.smem, s>>>(a);
  }
}

static int elem_size(int dtype) { return dtype == GPHL_F32 ? 4 : 2; }
static bool norm_vec(int64_t n, int dtype, std::initializer_list<const void *> ps) {
  if (n % (16 / elem_size(dtype)) != 0) return false;
  for (const void *p : ps)
    if (!aligned16(p)) return false;
  return true;
}

}  // namespace gphl

using namespace gphl;

extern "C" int gphl_rms_norm(int32_t dtype, int64_t m, int64_t n, const void *x, const void *residual, const void *w, int32_t w_dtype,
                             float eps, void *y, void *r, float *rstd, void *stream) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(dtype >= GPHL_F32 && dtype <= GPHL_F16, "rms_norm: unknown type %d", dtype);
  GPHL_REQUIRE(w_dtype == dtype || w_dtype == GPHL_F32, "rms_norm: the weight must have the rows' type or be float32");
  GPHL_REQUIRE(m < INT32_MAX && n <= (1 << 24), "size out of range");
  GPHL_REQUIRE(eps >= 0.f, "rms_norm: eps must not be negative");
  if (m == 0 || n == 0) return GPHL_OK;
  GPHL_REQUIRE(x && w && y && (r || !residual), "null pointer argument");
  NormArgs a{};
  a.x = x, a.res = residual, a.w = w, a.y = y, a.r = residual ? r : nullptr, a.rstd = rstd, a.m = m, a.n = (int32_t)n, a.eps = eps;
  a.w_f32 = w_dtype == GPHL_F32;
  norm_types<false>(a, dtype, norm_vec(n, dtype, {x, residual, w, y, r}), sm_count(), static_cast<cudaStream_t>(stream));
  return launched("rms_norm_kernel");
}

extern "C" int gphl_rms_norm_fp8(int32_t dtype, int64_t m, int64_t n, const void *x, const void *residual, const void *w, int32_t w_dtype,
                                 float eps, void *q, int64_t q_stride, float *scales, int64_t scale_stride, void *r, void *stream) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(dtype >= GPHL_F32 && dtype <= GPHL_F16, "rms_norm_fp8: unknown type %d", dtype);
  GPHL_REQUIRE(w_dtype == dtype || w_dtype == GPHL_F32, "rms_norm_fp8: the weight must have the rows' type or be float32");
  GPHL_REQUIRE(m < INT32_MAX && n <= (1 << 24), "size out of range");
  GPHL_REQUIRE(eps >= 0.f, "rms_norm_fp8: eps must not be negative");
  if (m == 0 || n == 0) return GPHL_OK;
  GPHL_REQUIRE(x && w && q && scales && (r || !residual), "null pointer argument");
  GPHL_REQUIRE(q_stride == (n + 15) / 16 * 16 && aligned16(q), "rms_norm_fp8: code rows must be 16-byte aligned and padded to 16 bytes");
  GPHL_REQUIRE(scale_stride >= m, "rms_norm_fp8: scale_stride must be at least the number of rows");
  NormArgs a{};
  a.x = x, a.res = residual, a.w = w, a.q = static_cast<uint8_t *>(q), a.scales = scales, a.scale_stride = scale_stride;
  a.r = residual ? r : nullptr, a.m = m, a.n = (int32_t)n, a.n_pad = (int32_t)q_stride, a.eps = eps, a.w_f32 = w_dtype == GPHL_F32;
  norm_types<true>(a, dtype, norm_vec(n, dtype, {x, residual, w, r}), sm_count(), static_cast<cudaStream_t>(stream));
  return launched("rms_norm_kernel");
}

extern "C" int64_t gphl_rms_norm_grad_workspace_bytes(int32_t dtype, int64_t m, int64_t n) {
  if (m <= 0 || n <= 0 || dtype < GPHL_F32 || dtype > GPHL_F16) return 0;
  // the vector or the column form may run (alignment is known at the call): the larger of the two
  const int sms = sm_count();
  const int64_t grid = std::max(grad_shape(m, (int)n, 4, sms).grid, grad_shape(m, (int)n, 16 / elem_size(dtype), sms).grid);
  return grid * n * (int64_t)sizeof(float);
}

extern "C" int gphl_rms_norm_grad(int32_t dtype, int64_t m, int64_t n, const void *r, const void *w, int32_t w_dtype, const float *rstd,
                                  const void *dy, const void *dr, void *dx, void *dw, void *workspace, void *stream_) {
  GPHL_REQUIRE(m >= 0 && n >= 0, "negative size");
  GPHL_REQUIRE(dtype >= GPHL_F32 && dtype <= GPHL_F16, "rms_norm_grad: unknown type %d", dtype);
  GPHL_REQUIRE(w_dtype == dtype || w_dtype == GPHL_F32, "rms_norm_grad: the weight must have the rows' type or be float32");
  GPHL_REQUIRE(m < INT32_MAX && n <= (1 << 24), "size out of range");
  if (n == 0) return GPHL_OK;
  GPHL_REQUIRE(dw != nullptr, "null pointer argument");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (m == 0) {
    GPHL_CUDA(cudaMemsetAsync(dw, 0, (size_t)n * (size_t)elem_size(w_dtype), stream));
    return GPHL_OK;
  }
  GPHL_REQUIRE(r && w && rstd && dy && dx && workspace, "null pointer argument");
  NormGradArgs a{};
  a.r = r, a.w = w, a.rstd = rstd, a.dy = dy, a.dr = dr, a.dx = dx, a.part = static_cast<float *>(workspace);
  a.m = m, a.n = (int32_t)n, a.w_f32 = w_dtype == GPHL_F32;
  const bool vec = norm_vec(n, dtype, {r, w, dy, dr, dx});
  const GradShape g = grad_shape(m, (int)n, vec ? 16 / elem_size(dtype) : 4, sm_count());
  if (dtype == GPHL_F32) vec ? grad_launch<float, false>(a, g, stream) : grad_launch<float, true>(a, g, stream);
  else if (dtype == GPHL_BF16) vec ? grad_launch<__nv_bfloat16, false>(a, g, stream) : grad_launch<__nv_bfloat16, true>(a, g, stream);
  else vec ? grad_launch<__half, false>(a, g, stream) : grad_launch<__half, true>(a, g, stream);
  int rc = launched("rms_norm_grad_kernel");
  if (rc != GPHL_OK) return rc;
  const unsigned blocks = (unsigned)((n + 31) / 32);
  if (w_dtype == GPHL_F32) rms_norm_dw_kernel<float><<<blocks, 256, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<float *>(dw));
  else if (w_dtype == GPHL_BF16)
    rms_norm_dw_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<__nv_bfloat16 *>(dw));
  else rms_norm_dw_kernel<__half><<<blocks, 256, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<__half *>(dw));
  return launched("rms_norm_dw_kernel");
}

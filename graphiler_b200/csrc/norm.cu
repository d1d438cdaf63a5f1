// Root-mean-square norm of rows, with the residual's addition:
//   r = round(x + residual)   (kept in the rows' type: what the next layer adds to is what is normalised)
//   y = r * rstd * w,   rstd = 1 / sqrt(mean(r^2) + eps)
// y in the rows' type, or as e4m3 codes with one power-of-two scale per row and block of 128 columns.  Backward, from r and rstd:
//   g = dy * w, xhat = r * rstd, dx = dr + rstd * (g - xhat * mean(g * xhat)), dw = sum over rows of dy * xhat.
//
// Memory bound.  A row is read once and stays in registers: WPR warps hold it, up to NV steps each (a step is 32 lanes x 16 bytes).  Sums
// of a row are fp32: at most 16 terms a lane, then a tree over lanes and warps, so an error of a few 2^-24.  (Joining them and taking the
// root in double was the bound of short rows: 600,000 x 256 in bf16 took 251 us forward and 429 us backward.)  Rows too wide for the
// registers are read twice, and a lane's terms, up to 32768 of them, are gathered with their rounding errors (Acc), so that the sum is as good.
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

// Joins `v` over the lanes of a row, or (wpr > 1) over its warps: all threads of the block.
template <int LPR> __device__ __forceinline__ float row_sum(float v, int wpr, int warp, int lane, float *s_part) {
#pragma unroll
  for (int d = LPR / 2; d >= 1; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
  if (LPR < 32 || wpr == 1) return v;
  if (lane == 0) s_part[warp] = v;
  __syncthreads();
  v = lane < wpr ? s_part[lane] : 0.f;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v += __shfl_xor_sync(FULL, v, d);
  __syncthreads();                                   // s_part may be written again
  return v;
}

// A sum with its rounding errors; one that has left fp32 has none (infinity less infinity), and stays what it is.
__device__ __forceinline__ float finite_sum(const Acc &s) { return fabsf(s.hi) <= FLT_MAX ? s.value() : s.hi; }

// NV > 0: the row is held in registers.  NV == 0: any width, the row is read twice.
template <typename T, typename R, int NV, bool FP8>
__global__ void __launch_bounds__(512) rms_norm_kernel(const NormArgs a) {
  constexpr int E = R::E, RPW = 32 / R::LPR;         // rows of a warp
  __shared__ float s_part[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (R::LPR - 1);
  const int per_block = (blockDim.x >> 5) / a.wpr * RPW;
  // rows past the last one do the last one's work over again and store nothing: all lanes of a warp take part in its shuffles
  const int64_t at = (int64_t)blockIdx.x * per_block + (warp / a.wpr) * RPW + (threadIdx.x & 31) / R::LPR, row = min(at, a.m - 1);
  const bool live = at < a.m;
  const int w0 = warp % a.wpr, steps = (a.n + R::STEP - 1) / R::STEP;
  const T *x = static_cast<const T *>(a.x) + row * a.n;
  const T *res = a.res ? static_cast<const T *>(a.res) + row * a.n : nullptr;
  T *r = a.r && live ? static_cast<T *>(a.r) + row * a.n : nullptr;

  constexpr int KEEP = NV > 0 ? NV : 1;
  float v[KEEP][E];
  float ss = 0.f;
  // a step of r, from the inputs; stored where there is a residual
  auto take = [&](typename R::Raw t, const typename R::Raw &u, int step, float (&f)[E]) {
    if (res) {
      t = R::add(t, u);
      if (r) R::store(r, step, lane, a.n, t);
    }
    R::widen(t, f);
  };
  if constexpr (NV > 0) {
    typename R::Raw xs[NV], rs[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        xs[i] = R::raw(x, step, lane, a.n);
        if (res) rs[i] = R::raw(res, step, lane, a.n);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        take(xs[i], rs[i], step, v[i]);
#pragma unroll
        for (int j = 0; j < E; ++j) ss = fmaf(v[i][j], v[i][j], ss);
      }
    }
  } else {
    Acc sum{0.f, 0.f};
    for (int step = w0; step < steps; step += a.wpr) {
      const typename R::Raw t = R::raw(x, step, lane, a.n);
      take(t, res ? R::raw(res, step, lane, a.n) : t, step, v[0]);
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) part = fmaf(v[0][j], v[0][j], part);
      sum.add(part);
    }
    ss = finite_sum(sum);
  }
  const float rstd = 1.f / sqrtf(row_sum<R::LPR>(ss, a.wpr, warp, lane, s_part) / (float)a.n + a.eps);
  if (a.rstd && w0 == 0 && lane == 0 && live) a.rstd[row] = rstd;

  auto write = [&](int step, const float (&t)[E]) {
    float w[E], y[E];
    R::weight(a.w, a.w_f32, step, lane, a.n, w);
#pragma unroll
    for (int j = 0; j < E; ++j) y[j] = t[j] * rstd * w[j];
    if constexpr (FP8) store_codes<R>(y, a.q + row * a.n_pad, a.scales + row, a.scale_stride, step, lane, a.n, a.n_pad, live);
    else if (live) R::store(static_cast<T *>(a.y) + row * a.n, step, lane, a.n, y);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) write(step, v[i]);
    }
  } else {
    for (int step = w0; step < steps; step += a.wpr) {
      const typename R::Raw t = R::raw(r ? r : x, step, lane, a.n);      // r: this thread's own stores
      R::widen(t, v[0]);
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
// rows it meets and leaves once.  The next row's r and dy are on their way while a row is finished, and a lane holds 8 values of each, so
// that 32 warps fit an SM.
template <typename T, typename R, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_grad_kernel(const NormGradArgs a) {
  constexpr int E = R::E, NV = 8 / E, RPW = 32 / R::LPR;
  __shared__ float s_part[32];
  extern __shared__ float s_dw[];                    // wpr == 1: n sums per row slot of the block
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & (R::LPR - 1), sub = (threadIdx.x & 31) / R::LPR;
  const int slots = warps / a.wpr * RPW, slot = (warp / a.wpr) * RPW + sub, w0 = warp % a.wpr, steps = (a.n + R::STEP - 1) / R::STEP;
  float dw[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) dw[i][j] = 0.f;
  typename R::Raw r[NV], dy[NV];
  float rstd = 0.f;
  // past the last row: its values again, which count for nothing
  auto fetch = [&](int64_t at) {
    const int64_t row = min(at, a.m - 1);
    rstd = __ldg(a.rstd + row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        r[i] = R::raw(static_cast<const T *>(a.r) + row * a.n, step, lane, a.n);
        dy[i] = R::raw(static_cast<const T *>(a.dy) + row * a.n, step, lane, a.n);
      }
    }
  };
  const int64_t stride = (int64_t)gridDim.x * slots;
  int64_t first = (int64_t)blockIdx.x * slots + (warp / a.wpr) * RPW;      // of the warp's rows: uniform in the warp
  if (first < a.m) fetch(first + sub);
  for (; first < a.m; first += stride) {
    const int64_t row = first + sub;
    const bool live = row < a.m;
    float xh[NV][E], g[NV][E];
    typename R::Raw dr[NV];
    float sum = 0.f;
    const float scale = rstd;
    const int64_t at = min(row, a.m - 1) * a.n;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (a.dr && w0 + i * a.wpr < steps) dr[i] = R::raw(static_cast<const T *>(a.dr) + at, w0 + i * a.wpr, lane, a.n);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        float w[E], part = 0.f;
        R::widen(r[i], xh[i]);
        R::widen(dy[i], g[i]);
        R::weight(a.w, a.w_f32, step, lane, a.n, w);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          xh[i][j] *= scale;
          if (RPW == 1 || live) dw[i][j] = fmaf(g[i][j], xh[i][j], dw[i][j]);
          g[i][j] *= w[j];
          part = fmaf(g[i][j], xh[i][j], part);
        }
        sum += part;
      }
    }
    if (first + stride < a.m) fetch(row + stride);
    const float mean = row_sum<R::LPR>(sum, a.wpr, warp, lane, s_part) / (float)a.n;
    T *dx = static_cast<T *>(a.dx) + at;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int step = w0 + i * a.wpr;
      if (step < steps) {
        float o[E];
        if (a.dr) R::widen(dr[i], o);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float t = scale * fmaf(-xh[i][j], mean, g[i][j]);
          o[j] = a.dr ? o[j] + t : t;
        }
        if (RPW == 1 || live) R::store(dx, step, lane, a.n, o);
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
      if (c < a.n) s_dw[slot * a.n + c] = dw[i][j];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < slots; ++k) s += s_dw[k * a.n + c];
    part[c] = s;
  }
}

// Rows wider than the registers of 32 warps: one block per row reads its inputs twice; dw is left to rms_norm_dw_wide_kernel.
template <typename T, typename R>
__global__ void __launch_bounds__(512) rms_norm_grad_wide_kernel(const NormGradArgs a) {
  constexpr int E = R::E;
  __shared__ float s_part[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, steps = (a.n + R::STEP - 1) / R::STEP;
  const int64_t row = blockIdx.x;
  const T *r = static_cast<const T *>(a.r) + row * a.n, *dy = static_cast<const T *>(a.dy) + row * a.n;
  const T *dr = a.dr ? static_cast<const T *>(a.dr) + row * a.n : nullptr;
  T *dx = static_cast<T *>(a.dx) + row * a.n;
  const float rstd = __ldg(a.rstd + row);
  float xh[E], g[E], w[E];
  auto read = [&](int step) {
    R::widen(R::raw(r, step, lane, a.n), xh);
    R::widen(R::raw(dy, step, lane, a.n), g);
    R::weight(a.w, a.w_f32, step, lane, a.n, w);
#pragma unroll
    for (int j = 0; j < E; ++j) xh[j] *= rstd, g[j] *= w[j];
  };
  Acc sum{0.f, 0.f};
  for (int step = warp; step < steps; step += a.wpr) {
    read(step);
    float part = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) part = fmaf(g[j], xh[j], part);
    sum.add(part);
  }
  const float mean = row_sum<32>(finite_sum(sum), a.wpr, warp, lane, s_part) / (float)a.n;
  for (int step = warp; step < steps; step += a.wpr) {
    read(step);
    float o[E];
    if (dr) R::widen(R::raw(dr, step, lane, a.n), o);
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
  Acc s{0.f, 0.f};
  for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y) {
    const int64_t i = row * a.n + c;
    s.add(to_float(static_cast<const T *>(a.dy)[i]) * (to_float(static_cast<const T *>(a.r)[i]) * __ldg(a.rstd + row)));
  }
  a.part[(int64_t)blockIdx.y * a.n + c] = finite_sum(s);
}

// dw = the partial sums' sum, in a fixed order, in double: 32 threads a column, eight loads of each under way (with eight threads a column
// and one load each, 2368 parts of 1001 columns took 42 us).
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_dw_kernel(const float *__restrict__ part, int32_t parts, int32_t n, T *__restrict__ dw) {
  __shared__ double s[32][33];
  const int lane = threadIdx.x & 31, k0 = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double v = 0.0;
  if (c < n) {
    for (int k = k0; k < parts; k += 256) {
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = k + 32 * j < parts ? __ldcs(part + (int64_t)(k + 32 * j) * n + c) : 0.f;
      // fp32 pairs of neighbours in the tree, then double
      v += (double)((t[0] + t[1]) + (t[2] + t[3])) + (double)((t[4] + t[5]) + (t[6] + t[7]));
    }
  }
  s[k0][lane] = v;
  __syncthreads();
  if (k0 == 0 && c < n) {
    for (int k = 1; k < 32; ++k) v += s[k][lane];
    dw[c] = from_float<T>((float)v);
  }
}

static int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

template <typename T, typename R, int NV, bool FP8> static void norm_launch(const NormArgs &a, int warps, cudaStream_t s) {
  const int per_block = warps / a.wpr * (32 / R::LPR);
  rms_norm_kernel<T, R, NV, FP8><<<(unsigned)((a.m + per_block - 1) / per_block), warps * 32, 0, s>>>(a);
}
template <typename T, typename R, bool FP8> static void norm_dispatch(NormArgs a, int sms, cudaStream_t s) {
  constexpr int LOW = 8 / R::E, HIGH = 16 / R::E;    // steps a warp holds: 8 or 16 values a lane
  const int steps = (a.n + R::STEP - 1) / R::STEP;
  // Few warps a row leave most loads in flight per warp and need the fewest joins (16 values a lane: 100,000 x 1024 in bf16 128 us, 8 values
  // 149); when the rows would not fill the GPU with 8 warps an SM that way, and for single columns (10007 x 1001 fp32: 29 against 31 us), a
  // row is spread over more warps instead.
  int wpr = pow2_at_least(R::SINGLE ? (steps + LOW - 1) / LOW : (steps + HIGH - 1) / HIGH);
  if (a.m * wpr < 8 * sms) wpr = pow2_at_least((steps + LOW - 1) / LOW);
  a.wpr = std::min(wpr, 16);
  const int warps = a.wpr == 1 ? 4 : a.wpr;
  if (steps <= a.wpr * LOW) norm_launch<T, R, LOW, FP8>(a, warps, s);
  else if constexpr (R::LPR == 32) {
    if (steps <= a.wpr * HIGH) norm_launch<T, R, HIGH, FP8>(a, warps, s);
    else norm_launch<T, R, 0, FP8>(a, warps, s);
  }
}
template <bool FP8> static void norm_types(const NormArgs &a, int dtype, bool vec, int sms, cudaStream_t s) {
  if (dtype == GPHL_F32) with_lanes<float>(a.n, vec, [&](auto r) { norm_dispatch<float, decltype(r), FP8>(a, sms, s); });
  else if (dtype == GPHL_BF16) with_lanes<__nv_bfloat16>(a.n, vec, [&](auto r) { norm_dispatch<__nv_bfloat16, decltype(r), FP8>(a, sms, s); });
  else with_lanes<__half>(a.n, vec, [&](auto r) { norm_dispatch<__half, decltype(r), FP8>(a, sms, s); });
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n;
}

struct GradShape {
  int wpr, warps, grid;
  size_t smem;
};
// E, LPR as in Row.  wpr == 0: wider than 32 warps hold.
static GradShape grad_shape(int64_t m, int n, int e, int lpr, int sms) {
  const int steps = (n + lpr * e - 1) / (lpr * e), hold = 8 / e;
  GradShape g{};
  const int wpr = pow2_at_least((steps + hold - 1) / hold);
  if (wpr > 32) {
    g.grid = (int)std::min<int64_t>(m, 64);          // row groups of the separate dw kernel
    return g;
  }
  g.wpr = wpr, g.warps = wpr > 1 ? wpr : 8;
  const int slots = g.warps / g.wpr * (32 / lpr);
  // as many blocks as are resident (32 warps an SM, 16 with the wider registers of fp32 rows and single columns): the partial rows of dw stay few
  g.grid = (int)std::min<int64_t>((m + slots - 1) / slots, (int64_t)sms * ((e == 4 && g.warps <= 16 ? 16 : 32) / g.warps));
  g.smem = g.wpr == 1 ? (size_t)slots * n * sizeof(float) : 0;
  return g;
}
template <typename T, typename R> static void grad_launch(NormGradArgs a, int sms, GradShape &g, cudaStream_t s) {
  g = grad_shape(a.m, a.n, R::E, R::LPR, sms);
  a.wpr = g.wpr;
  if (g.wpr > 0) {
    // Whole vectors of 16-bit rows do with 64 registers a thread (8 to 12 bytes of them spill).  fp32 rows and single columns would spill 104 to 136
    // bytes: they get up to 128 registers, and fewer warps, while 16 warps hold a row (4096 values), and spill beyond.
    if constexpr (R::E == 8 || R::LPR == 32)
      if (R::E == 8 || g.warps > 16) return rms_norm_grad_kernel<T, R, 1024><<<g.grid, g.warps * 32, g.smem, s>>>(a);
    if constexpr (R::E == 4) rms_norm_grad_kernel<T, R, 512><<<g.grid, g.warps * 32, g.smem, s>>>(a);
  } else if constexpr (R::LPR == 32) {
    a.wpr = 16;
    // dw's parts first: dx may lie over dy
    rms_norm_dw_wide_kernel<T><<<dim3((unsigned)((a.n + 255) / 256), (unsigned)g.grid), 256, 0, s>>>(a);
    rms_norm_grad_wide_kernel<T, R><<<(unsigned)a.m, 512, 0, s>>>(a);
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
  // any form may run (alignment is known at the call): the largest
  const int sms = sm_count();
  int64_t grid = grad_shape(m, (int)n, 4, 32, sms).grid;
  for (int lpr = 8; lpr <= 32; lpr *= 2) grid = std::max<int64_t>(grid, grad_shape(m, (int)n, 16 / elem_size(dtype), lpr, sms).grid);
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
  GradShape g{};
  const int sms = sm_count();
  if (dtype == GPHL_F32) with_lanes<float>(n, vec, [&](auto k) { grad_launch<float, decltype(k)>(a, sms, g, stream); });
  else if (dtype == GPHL_BF16) with_lanes<__nv_bfloat16>(n, vec, [&](auto k) { grad_launch<__nv_bfloat16, decltype(k)>(a, sms, g, stream); });
  else with_lanes<__half>(n, vec, [&](auto k) { grad_launch<__half, decltype(k)>(a, sms, g, stream); });
  int rc = launched("rms_norm_grad_kernel");
  if (rc != GPHL_OK) return rc;
  const unsigned blocks = (unsigned)((n + 31) / 32);
  if (w_dtype == GPHL_F32) rms_norm_dw_kernel<float><<<blocks, 1024, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<float *>(dw));
  else if (w_dtype == GPHL_BF16)
    rms_norm_dw_kernel<__nv_bfloat16><<<blocks, 1024, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<__nv_bfloat16 *>(dw));
  else rms_norm_dw_kernel<__half><<<blocks, 1024, 0, stream>>>(a.part, g.grid, (int32_t)n, static_cast<__half *>(dw));
  return launched("rms_norm_dw_kernel");
}

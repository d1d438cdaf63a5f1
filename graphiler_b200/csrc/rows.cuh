// Row access shared by the row-wise dense kernels (norm.cu, fp8.cu): LPR lanes walk a row in steps, every lane holding E values of
// a step.  Aligned rows: E values of one 16-byte vector; rows narrower than a warp's 32 vectors share a warp (LPR = 8 or 16).  Rows of odd
// width or base (SC): four single columns 32 apart, so that a step's loads are still whole 128- or 64-byte lines.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>

#include <type_traits>

#include "common.cuh"

namespace gphl {

#ifdef __CUDACC__

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T, bool SC, int LPR_ = 32> struct Row {
  static_assert(!SC || LPR_ == 32, "single columns are dealt to whole warps");
  static constexpr bool SINGLE = SC;
  static constexpr int LPR = LPR_, E = SC ? 4 : 16 / (int)sizeof(T), STEP = LPR * E;
  struct Raw {                                        // a lane's values of a step: four words as stored, or four single values widened
    uint32_t w[4];
  };
  // `lane`: of the row's LPR lanes
  __device__ static __forceinline__ int col(int step, int lane, int j) {
    return SC ? step * STEP + lane + 32 * j : step * STEP + lane * E + j;
  }
  __device__ static __forceinline__ Raw raw(const T *__restrict__ row, int step, int lane, int n) {
    Raw x;
    if constexpr (SC) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(step, lane, j);
        x.w[j] = c < n ? __float_as_uint(to_float(row[c])) : 0u;
      }
    } else {
      const int c = col(step, lane, 0);
      const uint4 v = c < n ? *reinterpret_cast<const uint4 *>(row + c) : make_uint4(0, 0, 0, 0);
      x.w[0] = v.x, x.w[1] = v.y, x.w[2] = v.z, x.w[3] = v.w;
    }
    return x;
  }
  __device__ static __forceinline__ void widen(const Raw &x, float (&v)[E]) {
    if constexpr (E == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(x.w[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) widen2(x.w[j], v[2 * j], v[2 * j + 1]);
    }
  }
  // Two 16-bit values of a word, and back (one instruction for the pair).
  __device__ static __forceinline__ void widen2(uint32_t w, float &lo, float &hi) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w));
      lo = f.x, hi = f.y;
    }
  }
  // Rounded to T as stored (single columns: the rounded values, widened).
  __device__ static __forceinline__ Raw round(const float (&v)[E]) {
    Raw x;
    if constexpr (E == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x.w[j] = __float_as_uint(to_float(from_float<T>(v[j])));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          x.w[j] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
          x.w[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
      }
    }
    return x;
  }
  // The sum rounded to T.  (The packed addition of 16-bit values rounds the exact sum once, like an addition in 32 bits and its rounding.)
  __device__ static __forceinline__ Raw add(const Raw &x, const Raw &y) {
    Raw z;
    if constexpr (E == 8) {
      using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const T2 s = __hadd2_rn(*reinterpret_cast<const T2 *>(&x.w[j]), *reinterpret_cast<const T2 *>(&y.w[j]));
        z.w[j] = *reinterpret_cast<const uint32_t *>(&s);
      }
    } else {
      float a[E], b[E];
      widen(x, a);
      widen(y, b);
#pragma unroll
      for (int j = 0; j < E; ++j) a[j] += b[j];
      z = round(a);
    }
    return z;
  }
  __device__ static __forceinline__ void store(T *__restrict__ row, int step, int lane, int n, const Raw &x) {
    if constexpr (SC) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(step, lane, j);
        if (c < n) row[c] = from_float<T>(__uint_as_float(x.w[j]));      // rounded already
      }
    } else {
      const int c = col(step, lane, 0);
      if (c < n) *reinterpret_cast<uint4 *>(row + c) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
    }
  }
  __device__ static __forceinline__ void store(T *__restrict__ row, int step, int lane, int n, const float (&v)[E]) { store(row, step, lane, n, round(v)); }
  // A weight row kept as T or, `f32`, in 32 bits.
  __device__ static __forceinline__ void weight(const void *w, bool f32, int step, int lane, int n, float (&v)[E]) {
    if (!f32) {
      widen(raw(static_cast<const T *>(w), step, lane, n), v);
    } else if constexpr (E == 4) {                     // single columns, or T is float
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = col(step, lane, j);
        v[j] = c < n ? static_cast<const float *>(w)[c] : 0.f;
      }
    } else {
      const int c = col(step, lane, 0);
      const float *p = static_cast<const float *>(w) + c;
      const float4 a = c < n ? *reinterpret_cast<const float4 *>(p) : make_float4(0, 0, 0, 0), b = c < n ? *reinterpret_cast<const float4 *>(p + 4) : a;
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
  }
};

// ---- e4m3 with a power-of-two scale per block of 128 -------------------------------------------------------------------------

constexpr uint32_t ABS_BITS = 0x7fffffffu, INF_BITS = 0x7f800000u;

// The exponent e >= -126 of the smallest power of two with amax <= 448 * 2^e (448 = 1.75 * 2^8, the largest e4m3 value).
__device__ __forceinline__ int fp8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
// What counts towards a block's largest magnitude: non-finite values do not (they become NaN codes by themselves).
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= FLT_MAX ? a : 0.f;
}
// Two codes, round to nearest even; NaN to the NaN code.  `e4m3x2`: infinities too.
__device__ __forceinline__ uint32_t e4m3x2_finite(float lo, float hi) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  lo = fabsf(lo) <= FLT_MAX ? lo : __int_as_float(0x7fffffff);
  hi = fabsf(hi) <= FLT_MAX ? hi : __int_as_float(0x7fffffff);
  return e4m3x2_finite(lo, hi);
}

// The codes of a lane's values of one step, stored, and their block's scale.  All lanes of the warp call it; nothing is stored unless `live`.
// Columns in [n, n_pad) are written as zero (the row's padding to 16 bytes).
template <typename R>
__device__ __forceinline__ void store_codes(const float (&y)[R::E], uint8_t *__restrict__ row, float *__restrict__ scale, int64_t scale_stride, int step, int lane,
                                            int n, int n_pad, bool live) {
  constexpr int E = R::E, BLOCK_LANES = R::STEP < 128 ? R::LPR : 128 / E;      // lanes that share a block
  uint32_t big = 0;                                    // magnitudes compare as integers, and anything from infinity up is not finite
#pragma unroll
  for (int j = 0; j < E; ++j) big = max(big, __float_as_uint(y[j]) & ABS_BITS);
#pragma unroll
  for (int d = BLOCK_LANES / 2; d >= 1; d >>= 1) big = max(big, __shfl_xor_sync(FULL, big, d));
  const bool rare = __any_sync(FULL, big >= INF_BITS);
  if (rare) {                                          // the largest finite magnitude instead
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) a = fmaxf(a, finite_abs(y[j]));
#pragma unroll
    for (int d = BLOCK_LANES / 2; d >= 1; d >>= 1) a = fmaxf(a, __shfl_xor_sync(FULL, a, d));
    big = __float_as_uint(a);
  }
  const int e = fp8_exponent(__uint_as_float(big));
  const float inv = pow2f(-e);
  uint32_t w[E / 4];
  if (rare) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) w[i] = e4m3x2(y[4 * i] * inv, y[4 * i + 1] * inv) | (e4m3x2(y[4 * i + 2] * inv, y[4 * i + 3] * inv) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
      w[i] = e4m3x2_finite(y[4 * i] * inv, y[4 * i + 1] * inv) | (e4m3x2_finite(y[4 * i + 2] * inv, y[4 * i + 3] * inv) << 16);
  }
  const int c0 = R::col(step, lane, 0);
  if (!live) return;
  if constexpr (R::SINGLE) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = R::col(step, lane, j);
      if (c < n_pad) row[c] = c < n ? (uint8_t)(w[0] >> (8 * j)) : (uint8_t)0;
    }
  } else {
    if (c0 < n_pad) {
#pragma unroll
      for (int i = 0; i < E / 4; ++i) w[i] = c0 < n ? w[i] : 0u;
      if constexpr (E == 8) *reinterpret_cast<uint2 *>(row + c0) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t *>(row + c0) = w[0];
    }
  }
  const int block = c0 / 128;
  if (lane % BLOCK_LANES == 0 && block * 128 < n) scale[block * scale_stride] = pow2f(e);
}

// Calls f with the number of lanes of a row as a constant: aligned rows of at most 8 or 16 vectors share a warp.
template <typename T, typename F> static void with_lanes(int64_t n, bool vec, F f) {
  const int64_t vectors = n * (int64_t)sizeof(T) / 16;
  if (vec && vectors <= 8) f(Row<T, false, 8>());
  else if (vec && vectors <= 16) f(Row<T, false, 16>());
  else if (vec) f(Row<T, false, 32>());
  else f(Row<T, true, 32>());
}

#endif  // __CUDACC__

}  // namespace gphl

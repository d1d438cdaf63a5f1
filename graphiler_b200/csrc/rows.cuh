// Row access shared by the row-wise dense kernels (norm.cu, fp8.cu): a warp walks a row in steps, every lane holding E values of
// a step as floats.  Aligned rows: E values of one 16-byte vector (a step is 128 fp32 or 256 16-bit columns).  Rows of odd width
// or base: four single columns 32 apart (a step is 128 columns), so that a step's loads are still whole 128- or 64-byte lines.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>

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

template <typename T, bool SC> struct Row {
  static constexpr int E = SC ? 4 : 16 / (int)sizeof(T);
  static constexpr int STEP = 32 * E;
  __device__ static __forceinline__ int col(int step, int lane, int j) {
    return SC ? step * STEP + lane + 32 * j : step * STEP + lane * E + j;
  }
  // U: the stored type, T or float (a weight kept in 32 bits beside 16-bit rows)
  template <typename U> __device__ static __forceinline__ void load(const U *__restrict__ row, int step, int lane, int n, float (&v)[E]) {
    if constexpr (SC) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(step, lane, j);
        v[j] = c < n ? to_float(row[c]) : 0.f;
      }
    } else {
      constexpr int PER = 16 / (int)sizeof(U);      // values of one 16-byte load
      const int c = col(step, lane, 0);
      if (c < n) {
#pragma unroll
        for (int q = 0; q < E / PER; ++q) {
          const uint4 raw = *reinterpret_cast<const uint4 *>(row + c + q * PER);
          const U *p = reinterpret_cast<const U *>(&raw);
#pragma unroll
          for (int j = 0; j < PER; ++j) v[q * PER + j] = to_float(p[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = 0.f;
      }
    }
  }
  __device__ static __forceinline__ void store(T *__restrict__ row, int step, int lane, int n, const float (&v)[E]) {
    if constexpr (SC) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(step, lane, j);
        if (c < n) row[c] = from_float<T>(v[j]);
      }
    } else {
      const int c = col(step, lane, 0);
      if (c < n) {
        uint4 raw;
        T *p = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int j = 0; j < E; ++j) p[j] = from_float<T>(v[j]);
        *reinterpret_cast<uint4 *>(row + c) = raw;
      }
    }
  }
};

// ---- e4m3 with a power-of-two scale per block of 128 -------------------------------------------------------------------------

// The exponent e >= -126 of the smallest power of two with amax <= 448 * 2^e (448 = 1.75 * 2^8, the largest e4m3 value).
__device__ __forceinline__ int fp8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) {      // -149 <= e <= 127
  return e >= -126 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}
// What counts towards a block's largest magnitude: non-finite values do not (they become NaN codes by themselves).
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= FLT_MAX ? a : 0.f;
}
__device__ __forceinline__ uint32_t e4m3(float v) {  // round to nearest even; infinities and NaN to the NaN code
  const float t = fabsf(v) <= FLT_MAX ? v : __int_as_float(0x7fffffff);
  return (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  lo = fabsf(lo) <= FLT_MAX ? lo : __int_as_float(0x7fffffff);
  hi = fabsf(hi) <= FLT_MAX ? hi : __int_as_float(0x7fffffff);
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// E bytes of codes of a lane's step; columns in [n, n_pad) are written as zero (the row's padding to 16 bytes).
template <typename T, bool SC>
__device__ __forceinline__ void store_codes(uint8_t *__restrict__ row, int step, int lane, int n, int n_pad, const uint32_t (&q)[Row<T, SC>::E]) {
  using R = Row<T, SC>;
  if constexpr (SC) {
#pragma unroll
    for (int j = 0; j < R::E; ++j) {
      const int c = R::col(step, lane, j);
      if (c < n_pad) row[c] = c < n ? (uint8_t)q[j] : (uint8_t)0;
    }
  } else {
    const int c = R::col(step, lane, 0);
    if (c < n_pad) {
      uint32_t w[R::E / 4];
#pragma unroll
      for (int i = 0; i < R::E / 4; ++i)
        w[i] = c < n ? (q[4 * i] | (q[4 * i + 1] << 8) | (q[4 * i + 2] << 16) | (q[4 * i + 3] << 24)) : 0u;
      if constexpr (R::E == 8) *reinterpret_cast<uint2 *>(row + c) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t *>(row + c) = w[0];
    }
  }
}

// Largest of the 128-column block that this lane's values belong to (16 lanes hold a block of a 16-bit vector step, else the warp).
template <typename T, bool SC> __device__ __forceinline__ float block_max(float a) {
  constexpr int LANES = 128 / Row<T, SC>::E;
#pragma unroll
  for (int d = LANES / 2; d >= 1; d >>= 1) a = fmaxf(a, __shfl_xor_sync(FULL, a, d));
  return a;
}

#endif  // __CUDACC__

}  // namespace gphl

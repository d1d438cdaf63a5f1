// The e4m3 product of few rows (decoding): out[i, j] = sum_k A[i, k] B[j, k] with at most 16 rows of A (8 with two weights), in one type.
//
// Bound by the bytes of B, each used for few products: what counts is how many of them are under way.  So there is no staging and no tensor
// memory: every warp loads B straight into the fragments of mma.sync, 16 bytes a lane, and the order of k inside a fragment is whatever the
// loads give, the same for A.  The warps of a block share its columns and take the blocks of 128 k in turn; their scaled fp32 sums meet in shared
// memory, in a fixed order.  1 x 4096 -> 8192 takes 6.8 us (4.9 TB/s), 1 x 16384 -> 16384 46 us (5.8).
#include "rows.cuh"
#include "tc_gemm.cuh"

namespace gphl {

constexpr int FEW_WARPS = 8;


struct FewArgs {
  const uint8_t *x, *w[2];
  const float *x_scale, *w_scale[2];
  int64_t x_stride, w_stride, x_scale_row, x_scale_block;
  int32_t m, n, k, kb;                                 // kb: blocks of 128 k
  void *out;
  int64_t ld_out, out_u;                               // out_u: from g to u (two weights: fp32)
  int32_t out_type;
};

// 16 codes of a row from column c on.  CHECKED: zero from column k on, whatever the row's padding holds.
template <bool CHECKED> __device__ __forceinline__ uint4 codes16(const uint8_t *row, int c, int k) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (!CHECKED || c < k) v = __ldg(reinterpret_cast<const uint4 *>(row + c));
  if (CHECKED) {
    auto keep = [&](uint32_t w, int at) { return at + 4 <= k ? w : at < k ? w & ((1u << (8 * (k - at))) - 1) : 0u; };
    v.x = keep(v.x, c), v.y = keep(v.y, c + 4), v.z = keep(v.z, c + 8), v.w = keep(v.w, c + 12);
  }
  return v;
}
__device__ __forceinline__ void mma_fp8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block: 16 columns of the output for all rows.  Its weight rows are the 16 rows of a fragment, eight rows of x its columns (GROUPS times); lane
// (g, t) = (lane / 4, lane % 4) holds 32 neighbouring codes of a block of 128 of weight rows g and g + 8 and of row g of x.
template <int WEIGHTS, int GROUPS>
__global__ void __launch_bounds__(32 * FEW_WARPS, GROUPS == 1 ? 3 : 2) few_rows_kernel(const FewArgs a) {
  __shared__ float s_sum[FEW_WARPS][WEIGHTS][8][17];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, n0 = blockIdx.x * 16;
  // rows past the last one: the last one's values, which are stored nowhere
  const int64_t lo = (int64_t)min(n0 + g, a.n - 1) * a.w_stride, hi = (int64_t)min(n0 + g + 8, a.n - 1) * a.w_stride;
  const int64_t ws = (int64_t)(n0 / 128) * a.kb;
  const uint8_t *x[GROUPS];
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) x[p] = a.x + min(8 * p + g, a.m - 1) * a.x_stride;
  float sum[WEIGHTS][GROUPS][4];
#pragma unroll
  for (int i = 0; i < WEIGHTS; ++i)
#pragma unroll
    for (int p = 0; p < GROUPS; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][p][j] = 0.f;
  struct Step {
    uint4 lo[WEIGHTS][2], hi[WEIGHTS][2], x[GROUPS][2];
  };
  auto load = [&](int kb, auto checked) {
    constexpr bool CHECKED = decltype(checked)::value;
    Step s;
    const int c = kb * 128 + t * 32;
#pragma unroll
    for (int i = 0; i < WEIGHTS; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.lo[i][h] = codes16<CHECKED>(a.w[i] + lo, c + 16 * h, a.k), s.hi[i][h] = codes16<CHECKED>(a.w[i] + hi, c + 16 * h, a.k);
#pragma unroll
    for (int p = 0; p < GROUPS; ++p)
#pragma unroll
      for (int h = 0; h < 2; ++h) s.x[p][h] = codes16<CHECKED>(x[p], c + 16 * h, a.k);
    return s;
  };
  auto use = [&](const Step &s, int kb) {
#pragma unroll
    for (int p = 0; p < GROUPS; ++p) {
      const float x0 = __ldg(a.x_scale + min(8 * p + 2 * t, a.m - 1) * a.x_scale_row + kb * a.x_scale_block);
      const float x1 = __ldg(a.x_scale + min(8 * p + 2 * t + 1, a.m - 1) * a.x_scale_row + kb * a.x_scale_block);
#pragma unroll
      for (int i = 0; i < WEIGHTS; ++i) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_fp8(d, s.lo[i][h].x, s.hi[i][h].x, s.lo[i][h].y, s.hi[i][h].y, s.x[p][h].x, s.x[p][h].y);
          mma_fp8(d, s.lo[i][h].z, s.hi[i][h].z, s.lo[i][h].w, s.hi[i][h].w, s.x[p][h].z, s.x[p][h].w);
        }
        const float w = __ldg(a.w_scale[i] + ws + kb), s0 = x0 * w, s1 = x1 * w;
        sum[i][p][0] = fmaf(d[0], s0, sum[i][p][0]), sum[i][p][1] = fmaf(d[1], s1, sum[i][p][1]);
        sum[i][p][2] = fmaf(d[2], s0, sum[i][p][2]), sum[i][p][3] = fmaf(d[3], s1, sum[i][p][3]);
      }
    }
  };
  const std::false_type whole;
  const int full = a.k / 128;                          // the last block of k may be a part of one
  int kb = warp;
  if (WEIGHTS == 1) {
#pragma unroll 1
    for (; kb + FEW_WARPS < full; kb += 2 * FEW_WARPS) {
      const Step s0 = load(kb, whole), s1 = load(kb + FEW_WARPS, whole);
      use(s0, kb), use(s1, kb + FEW_WARPS);
    }
  }
#pragma unroll 1
  for (; kb < full; kb += FEW_WARPS) use(load(kb, whole), kb);
  if (kb < a.kb) use(load(kb, std::true_type()), kb);
#pragma unroll
  for (int p = 0; p < GROUPS; ++p) {
    if (p > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < WEIGHTS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s_sum[warp][i][2 * t + (j & 1)][g + 8 * (j >> 1)] = sum[i][p][j];
    __syncthreads();
    const int i = threadIdx.x >> 7, row = 8 * p + ((threadIdx.x >> 4) & 7), j = threadIdx.x & 15, col = n0 + j;
    if (i < WEIGHTS && row < a.m && col < a.n) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < FEW_WARPS; ++w) v += s_sum[w][i][row & 7][j];
      const int64_t at = row * a.ld_out + i * a.out_u + col;
      if (a.out_type == GPHL_F32) static_cast<float *>(a.out)[at] = v;
      else if (a.out_type == GPHL_BF16) static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
      else static_cast<__half *>(a.out)[at] = __float2half_rn(v);
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------

// Parts of k that the product leaves in the workspace for the join (0: none, the output is finished), or -1: not for this kernel.  Against the
// tensor-core tiles, in us: 1 x 4096 -> 8192 6.8 / 13.5, 16 rows 10.0 / 13.6, 32 rows 27 / 20; gated, 8 x 4096 -> 11264 18.4 / 28.5, 16 rows 33 / 28.
int few_rows_parts(const GemmCall &c) {
  if (!c.fp8 || c.ptr || c.types != 1) return -1;
  if (c.dual == DUAL_GATED) return c.m <= 8 ? 1 : -1;
  return c.dual == DUAL_NONE && c.m <= 16 ? 0 : -1;
}

int few_rows(const GemmCall &c, float *part, int64_t ld_part, int64_t part_u, const char *what, cudaStream_t stream) {
  const bool two = c.dual == DUAL_GATED;
  FewArgs a{};
  for (int i = 0; i < (two ? 2 : 1); ++i) {
    GPHL_REQUIRE(aligned16(c.b[i].p) && aligned16(c.a[0].p) && c.b[i].ld % 16 == 0 && c.a[0].ld % 16 == 0,
                 "%s: operands must start on 16-byte boundaries and have rows a multiple of 16 bytes apart", what);
    a.w[i] = static_cast<const uint8_t *>(c.b[i].p), a.w_scale[i] = c.b_scale[i];
  }
  a.x = static_cast<const uint8_t *>(c.a[0].p), a.x_stride = c.a[0].ld, a.w_stride = c.b[0].ld;
  a.x_scale = c.a_scale, a.x_scale_row = c.a_scale_row, a.x_scale_block = c.a_scale_block;
  a.m = (int32_t)c.m, a.n = (int32_t)c.n, a.k = (int32_t)c.k, a.kb = (int32_t)((c.k + 127) / 128);
  a.out = two ? part : c.out[0], a.ld_out = two ? ld_part : c.ld_out, a.out_u = part_u, a.out_type = two ? GPHL_F32 : c.out_type;
  const unsigned grid = (unsigned)((c.n + 15) / 16);
  if (two) few_rows_kernel<2, 1><<<grid, 32 * FEW_WARPS, 0, stream>>>(a);
  else if (c.m <= 8) few_rows_kernel<1, 1><<<grid, 32 * FEW_WARPS, 0, stream>>>(a);
  else few_rows_kernel<1, 2><<<grid, 32 * FEW_WARPS, 0, stream>>>(a);
  return launched("few_rows_kernel");
}

}  // namespace gphl

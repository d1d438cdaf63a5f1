// The tensor-core product of the dense operators for sm_100a: out[i, j] = sum_k A[i, k] B[j, k], 16-bit or e4m3 operands, fp32 sums.
//
// One persistent block per SM, or one pair of blocks per two SMs, walks tiles of 128 (256) rows x BN columns of the output.  One warp brings boxes of A and B into a ring of
// shared-memory stages by TMA (128 bytes of k per stage, 128-byte swizzle), one issues tcgen05.mma into one of two accumulators in
// TMEM, eight or sixteen read the other one back and finish the tile, so that loads, products and stores of neighbouring tiles overlap.
// 16-bit: an accumulator gathers a whole tile.  e4m3: it holds one block of 128 k, which the eight warps scale (row scale x weight
// scale) and add to fp32 registers: the scales may differ from block to block, and no sum outlives a block inside the tensor core.
// GATED tiles multiply the same rows by BN/2 columns of each of two weights; both halves of the accumulator meet in the epilogue.
// When the tiles are fewer than the SMs, k is split and the parts are joined in a fixed order by a second kernel.
// Every wait is bounded: one that runs out is counted, all roles stop, wait (bounded) for what they have in flight, and the block
// frees its tensor memory and returns.
#include <algorithm>

#include "rows.cuh"
#include "tc_gemm.cuh"

namespace gphl {

constexpr int GM = 128;                                // rows of a tile = TMEM lanes
constexpr int STAGING = 4096;                          // per epilogue warp: 32 rows x 128 bytes
constexpr int GEMM_SMEM = 1024 + 224 * 1024;           // alignment, and the stages with the staging buffers
__host__ __device__ constexpr int ring_bytes(int epi_warps) { return 224 * 1024 - epi_warps * STAGING; }
constexpr int MAX_STAGES = 8;
constexpr int SCALES = 16;                             // row scales fetched at a time (blocks of k)
static_assert(2 * SCALES * 32 * 4 <= STAGING, "two groups of row scales lie in the staging buffer");
constexpr uint32_t GEMM_WAIT_LIMIT = 1u << 22;
constexpr int RASTER = 16;                             // row tiles that are walked together across the columns (L2 reuse of both operands)

__device__ int g_gemm_wait_timeouts = 0;

// n / d for n < 2^31 by one multiplication: mul = ceil(2^(32 + shift) / d) with 2^shift < d <= 2^(shift + 1) (Granlund and Montgomery, Division by
// Invariant Integers using Multiplication); d == 1 is its own case.
struct Divisor {
  uint32_t d, mul, shift;
  __host__ void set(uint32_t v) {
    d = v, mul = shift = 0;
    if (v <= 1) return;
    while ((2u << shift) < v) ++shift;
    mul = (uint32_t)(((1ull << (32 + shift)) + v - 1) / v);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d <= 1 ? n : __umulhi(n, mul) >> shift; }
};

struct __align__(64) GemmArgs {
  CUtensorMap a[2], b[2];
  int64_t m, n;
  uint32_t tiles_m, tiles_n, work;                     // work = tiles_m * tiles_n * batch * splits < 2^31
  Divisor by_plane, by_band, by_last;                  // tiles of a plane, of a band of RASTER row tiles, row tiles of the last band
  int32_t batch, splits, kt, kt_first;                 // steps of 128 bytes of k; kt_first: steps of the first pair (CONCAT)
  int32_t a_mn, b_mn, types, a_bytes;                  // a_bytes: of one step's box of A (fewer rows than a tile where m is smaller)
  uint32_t idesc;
  const int32_t *ptr;
  void *out[2];
  int64_t ld_out;
  int32_t out_type, out_vec, act, dh_vec;
  const void *dh;
  float *g, *u;
  int64_t ld_gu;
  uint8_t *q;
  float *q_scale;
  int64_t q_scale_stride;
  float *part;                                         // splits > 1: ((split * batch + b) * m + row) * ld_part + column
  int64_t ld_part, part_u;                             // part_u: column offset of u
  const float *a_scale, *b_scale[2];
  int64_t a_scale_row, a_scale_block;
  int32_t scale_kb, scale_nb;                          // blocks of 128 along k and n
};

namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
// The same barrier in block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(uint32_t bar, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(bar), "r"(rank));
  return r;
}
template <int CTAS> __device__ __forceinline__ void arrive(uint32_t bar) {
  if constexpr (CTAS == 2) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
  else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CTAS> __device__ __forceinline__ void alloc(uint32_t to, uint32_t cols) {
  if constexpr (CTAS == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <int CTAS> __device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t cols) {
  if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait for the phase of `parity`; false when the limit ran out or another role has given up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *failed, uint32_t limit = GEMM_WAIT_LIMIT) {
  for (uint32_t i = 0; i < limit; ++i) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255) == 255 && *failed) return false;
  }
  *failed = 1;
  return false;
}
// One lane of the (converged) warp.  Loops over steps run in all lanes alike and only the issue itself hangs on this: operands of TMA and
// tensor-core instructions must be known to be uniform, and a loop inside `if (lane == 0)` hides that (500 cycles a step for four products).
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
// One box into this block's shared memory; its bytes are counted on `bar`, which may lie in the pair's even block.
template <int CTAS> __device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
// 16 bytes, or zeros
__device__ __forceinline__ void copy16(void *dst, const void *src, bool in_range) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in_range ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(float *dst, const float *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Shared-memory operand descriptor, 128-byte swizzle.  K-major: rows of 128 bytes, groups of 8 rows 1024 B apart.  MN-major: rows
// of 64 i (or j) for one k, groups of 8 k 1024 B apart, the next 64 i 8192 B on (a box is 64 x 64).
__device__ __forceinline__ uint64_t operand(uint32_t saddr, bool mn) {
  uint64_t d = (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(mn ? 8192 >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
#define GPHL_MMA(group, kind)                                                             \
  asm volatile(                                                                           \
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"                                         \
      "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], %1, %2, %3, p;\n}" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(acc)                                                \
      : "memory")
template <int CTAS, bool FP8> __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (CTAS == 2) {
    if constexpr (FP8) GPHL_MMA("2", "f8f6f4");
    else GPHL_MMA("2", "f16");
  } else {
    if constexpr (FP8) GPHL_MMA("1", "f8f6f4");
    else GPHL_MMA("1", "f16");
  }
}
#undef GPHL_MMA
// Arrives on `bar` (of a pair: of both blocks) once the products issued so far are done.
template <int CTAS> __device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 fp32 columns of the warp's 32 lanes: one row's 32 values per thread, to be read only behind ld_wait of the same array (which names
// the registers, so that no use moves up).
__device__ __forceinline__ void ld32(uint32_t taddr, float (&f)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]), "=f"(f[4]), "=f"(f[5]), "=f"(f[6]), "=f"(f[7]), "=f"(f[8]), "=f"(f[9]), "=f"(f[10]), "=f"(f[11]), "=f"(f[12]), "=f"(f[13]), "=f"(f[14]), "=f"(f[15]), "=f"(f[16]), "=f"(f[17]), "=f"(f[18]), "=f"(f[19]), "=f"(f[20]), "=f"(f[21]), "=f"(f[22]), "=f"(f[23]), "=f"(f[24]), "=f"(f[25]), "=f"(f[26]), "=f"(f[27]), "=f"(f[28]), "=f"(f[29]), "=f"(f[30]), "=f"(f[31])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void ld_wait(float (&f)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(f[0]), "+f"(f[1]), "+f"(f[2]), "+f"(f[3]), "+f"(f[4]), "+f"(f[5]), "+f"(f[6]), "+f"(f[7]), "+f"(f[8]), "+f"(f[9]), "+f"(f[10]), "+f"(f[11]), "+f"(f[12]), "+f"(f[13]), "+f"(f[14]), "+f"(f[15]), "+f"(f[16]), "+f"(f[17]), "+f"(f[18]), "+f"(f[19]), "+f"(f[20]), "+f"(f[21]), "+f"(f[22]), "+f"(f[23]), "+f"(f[24]), "+f"(f[25]), "+f"(f[26]), "+f"(f[27]), "+f"(f[28]), "+f"(f[29]), "+f"(f[30]), "+f"(f[31])
               :
               : "memory");
}

}  // namespace tc

// ---- tiles -------------------------------------------------------------------------------------------------------------------------

struct Tile {
  int split, batch, n0, seg, rows;                     // rows == 0: nothing to do (typed: past the last tile)
  int64_t row0;
};

// Work item `w`, found by a whole warp.  Typed: row tile `mt` is looked up in the type pointer, 32 types at a time (tile counts, prefix
// sum, one hit); pointer values outside [0, m] are clamped.
template <int CTAS> __device__ __forceinline__ Tile find_tile(const GemmArgs &a, uint32_t w, int bn_out, int lane) {
  constexpr int TM = GM * CTAS;                          // rows of a tile; t.rows counts those of the whole tile
  Tile t;
  const uint32_t plane = a.tiles_m * a.tiles_n;
  t.split = t.batch = 0;
  if (w >= plane) {
    const uint32_t p = a.by_plane.div(w);
    w -= p * plane;
    t.split = (int)(a.batch == 2 ? p >> 1 : p), t.batch = (int)(a.batch == 2 ? p & 1 : 0);
  }
  const uint32_t band = a.by_band.div(w), in = w - band * RASTER * a.tiles_n;
  const bool whole = (band + 1) * RASTER <= a.tiles_m;
  const uint32_t high = whole ? RASTER : a.tiles_m - band * RASTER;
  const uint32_t nt = whole ? in / RASTER : a.by_last.div(in);
  const int64_t mt = band * RASTER + (in - nt * high);
  t.n0 = (int)nt * bn_out;
  t.seg = 0;
  if (!a.ptr) {
    t.row0 = mt * TM;
    t.rows = (int)min((int64_t)TM, a.m - t.row0);
    return t;
  }
  t.rows = 0, t.row0 = 0;
  int64_t base = 0;
  for (int t0 = 0; t0 < a.types; t0 += 32) {
    const int k = t0 + lane;
    int64_t lo = 0, hi = 0;
    if (k < a.types) {
      lo = min(max((int64_t)__ldg(a.ptr + k), (int64_t)0), a.m);
      hi = min(max((int64_t)__ldg(a.ptr + k + 1), lo), a.m);
    }
    const int64_t nt_ = (hi - lo + TM - 1) / TM;
    int64_t incl = nt_;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t v = __shfl_up_sync(FULL, incl, d);
      if (lane >= d) incl += v;
    }
    const int64_t first = base + incl - nt_;
    const bool hit = mt >= first && mt < first + nt_;
    const unsigned who = __ballot_sync(FULL, hit);
    if (who) {
      const int src = __ffs(who) - 1;
      const int64_t row = lo + (mt - first) * TM;
      t.seg = __shfl_sync(FULL, k, src);
      t.row0 = __shfl_sync(FULL, row, src);
      t.rows = (int)__shfl_sync(FULL, min((int64_t)TM, hi - row), src);
      return t;
    }
    base += __shfl_sync(FULL, incl, 31);
  }
  return t;
}

// ---- storing a chunk: 32 columns of the warp's 32 rows, one row per thread ------------------------------------------------------------

// A thread's values lie in one row; stored directly every instruction would touch 32 rows.  The chunk goes through a swizzled staging
// buffer and leaves as row segments of 128 (fp32) or 64 bytes.
__device__ __forceinline__ void store_chunk(const float (&v)[32], int type, bool vec, void *out, int64_t ld, int64_t row0, int rows, int64_t col0,
                                            int64_t ncols, uint8_t *stg, int lane) {
  if (type == GPHL_F32) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      *reinterpret_cast<float4 *>(stg + lane * 128 + ((q ^ (lane & 7)) << 4)) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
    float *o = static_cast<float *>(out);
    if (vec && col0 + 32 <= ncols) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = (lane >> 3) + 4 * j, ch = lane & 7;
        if (r < rows) *reinterpret_cast<float4 *>(o + (row0 + r) * ld + col0 + ch * 4) = *reinterpret_cast<const float4 *>(stg + r * 128 + ((ch ^ (r & 7)) << 4));
      }
    } else if (col0 + lane < ncols) {
      for (int r = 0; r < rows; ++r)
        o[(row0 + r) * ld + col0 + lane] = *reinterpret_cast<const float *>(stg + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
    }
  } else {
    uint32_t p[16];
    if (type == GPHL_BF16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        p[i] = *reinterpret_cast<uint32_t *>(&h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        p[i] = *reinterpret_cast<uint32_t *>(&h);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<uint4 *>(stg + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = make_uint4(p[4 * q], p[4 * q + 1], p[4 * q + 2], p[4 * q + 3]);
    __syncwarp();
    uint16_t *o = static_cast<uint16_t *>(out);
    if (vec && col0 + 32 <= ncols) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (lane >> 2) + 8 * j, ch = lane & 3;
        if (r < rows) *reinterpret_cast<uint4 *>(o + (row0 + r) * ld + col0 + ch * 8) = *reinterpret_cast<const uint4 *>(stg + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
      }
    } else if (col0 + lane < ncols) {
      for (int r = 0; r < rows; ++r)
        o[(row0 + r) * ld + col0 + lane] = *reinterpret_cast<const uint16_t *>(stg + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
    }
  }
  __syncwarp();
}

// The reverse for 16-bit rows: 32 columns of the warp's rows, one row per thread, two values a word; 0 outside.  Aligned rows come by
// asynchronous copies (fetch_chunk) that are under way while the previous tile is finished.
__device__ __forceinline__ void fetch_chunk(const void *in, int64_t ld, int64_t row0, int rows, int64_t col0, int64_t ncols, uint8_t *stg, int lane) {
  const uint16_t *src = static_cast<const uint16_t *>(in);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = (lane >> 2) + 8 * j, ch = lane & 3;
    const bool in_range = r < rows && col0 + ch * 8 < ncols;         // rows are whole 16-byte pieces
    tc::copy16(stg + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4), in_range ? src + (row0 + r) * ld + col0 + ch * 8 : src, in_range);
  }
}
__device__ __forceinline__ void load_chunk(uint32_t (&v)[16], bool fetched, const void *in, int64_t ld, int64_t row0, int rows, int64_t col0, int64_t ncols,
                                           uint8_t *stg, int lane) {
  if (fetched) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    const uint16_t *src = static_cast<const uint16_t *>(in);
    for (int r = 0; r < 32; ++r)
      *reinterpret_cast<uint16_t *>(stg + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2) =
          r < rows && col0 + lane < ncols ? __ldg(src + (row0 + r) * ld + col0 + lane) : (uint16_t)0;
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint4 p = *reinterpret_cast<const uint4 *>(stg + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4));
    v[4 * q] = p.x, v[4 * q + 1] = p.y, v[4 * q + 2] = p.z, v[4 * q + 3] = p.w;
  }
  __syncwarp();
}
template <int TYPE> __device__ __forceinline__ void unpack16(uint32_t w, float &lo, float &hi) {
  if constexpr (TYPE == GPHL_BF16) lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
  else {
    const __half2 h = *reinterpret_cast<const __half2 *>(&w);
    lo = __low2float(h), hi = __high2float(h);
  }
}

// 32 e4m3 codes per row; code rows are padded to 16 bytes, so a 16-byte piece is inside the row whenever its first column is.
__device__ __forceinline__ void store_code_chunk(const float (&v)[32], float inv, uint8_t *out, int64_t ld, int64_t row0, int rows, int64_t col0,
                                                 int64_t ncols, uint8_t *stg, int lane) {
  uint32_t p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t w = e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | (e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + 4 * i + j >= ncols) w &= ~(0xffu << (8 * j));
    p[i] = w;
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
    *reinterpret_cast<uint4 *>(stg + lane * 32 + ((q ^ ((lane >> 2) & 1)) << 4)) = make_uint4(p[4 * q], p[4 * q + 1], p[4 * q + 2], p[4 * q + 3]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = (lane >> 1) + 16 * j, ch = lane & 1;
    if (r < rows && col0 + ch * 16 < ld)
      *reinterpret_cast<uint4 *>(out + (row0 + r) * ld + col0 + ch * 16) = *reinterpret_cast<const uint4 *>(stg + r * 32 + ((ch ^ ((r >> 2) & 1)) << 4));
  }
  __syncwarp();
}

// ---- the kernel --------------------------------------------------------------------------------------------------------------------

enum Mode { LINEAR, GATED, GATED_GRAD };

// CTAS == 2: a pair of blocks on neighbouring SMs shares a tile of 256 rows: each brings its own 128 rows of A and half of B's columns, the
// even block issues products over both shared memories (cta_group::2), so that an SM's share of a step is 32 KB instead of 48 (gated 8192 x 4096 ->
// 11264 in bf16: 0.97 against 1.09 ms).
__host__ __device__ constexpr int gemm_threads(int epi_warps, bool fp8) { return 32 * (epi_warps + (fp8 ? 4 : 2)); }

template <int BN, int CTAS, int EPI_WARPS, bool FP8, int MODE>
__global__ void __launch_bounds__(gemm_threads(EPI_WARPS, FP8), 1) gemm_kernel(const __grid_constant__ GemmArgs a) {
  constexpr bool PAIRED = MODE != LINEAR;                // two weights, their columns side by side in the accumulator
  constexpr int BROWS = BN / CTAS;                       // columns of B in this block's shared memory
  constexpr int STAGE = GM * 128 + BROWS * 128;
  constexpr int RING_BYTES = ring_bytes(EPI_WARPS);
  constexpr int STAGES = RING_BYTES / STAGE < MAX_STAGES ? RING_BYTES / STAGE : MAX_STAGES;
  constexpr int BN_OUT = PAIRED ? BN / 2 : BN;           // output columns of a tile
  constexpr int PARTS = EPI_WARPS / 4;                   // the accumulator's columns are split among so many warps per 32 rows
  constexpr int NCH = BN / PARTS / 32;                   // chunks of 32 accumulator columns of a thread
  constexpr int KE = FP8 ? 128 : 64;                     // k of a step
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t s_full[MAX_STAGES], s_empty[MAX_STAGES], s_acc_full[2], s_acc_empty[2], s_pair[4], s_drain;
  __shared__ int8_t s_exp[2][FP8 ? EPI_WARPS : 1][32];   // codes: the exponent of a row's scale as each warp sees it, in -126 .. 120
  __shared__ uint32_t s_tmem;
  __shared__ int s_failed;

  const int warp = __shfl_sync(FULL, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0;
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const uint32_t ring_u = tc::smem_u32(ring), full = tc::smem_u32(s_full), empty = tc::smem_u32(s_empty);
  const uint32_t acc_full = tc::smem_u32(s_acc_full), acc_empty = tc::smem_u32(s_acc_empty), drain = tc::smem_u32(&s_drain);
  const uint32_t pair = tc::smem_u32(s_pair);
  volatile int *failed = &s_failed;
  uint32_t issued = 0;                                   // TMA warp: steps brought in

  if (warp == EPI_WARPS + 1) tc::alloc<CTAS>(tc::smem_u32(&s_tmem), 2 * BN);
  if (threadIdx.x == 0) {
    s_failed = 0;
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(full + 8 * i, 1), tc::mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(acc_full + 8 * i, 1), tc::mbar_init(acc_empty + 8 * i, CTAS * EPI_WARPS);
    for (int i = 0; i < 4; ++i) tc::mbar_init(pair + 8 * i, PARTS);
    tc::mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  tc::before_sync();
  if (CTAS == 2) tc::cluster_sync();                     // the other block's barriers exist before anything arrives there
  else __syncthreads();
  tc::after_sync();
  const uint32_t tmem = s_tmem;
  const uint32_t w0 = blockIdx.x / CTAS, wstep = gridDim.x / CTAS;
  // e4m3: 12 warps start with 168 registers a thread (64512 of them); the 8 that hold sums take 232 and the 4 others give theirs up
  static_assert(!FP8 || EPI_WARPS == 8, "the register split is for 8 + 4 warps");
  if (warp >= EPI_WARPS) {
    if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == EPI_WARPS) {
      // ---- TMA: step i goes to stage i % STAGES; the bytes of both blocks are counted on the even block's barrier
      uint32_t i = 0;
      bool ok = true;
      const uint32_t lead_full = CTAS == 2 ? tc::in_block(full, 0) : full;
      for (uint32_t w = w0; w < a.work && ok; w += wstep) {
        const Tile t = find_tile<CTAS>(a, w, BN_OUT, lane);
        if (t.rows == 0) continue;
        const int k0 = (int)((int64_t)a.kt * t.split / a.splits), k1 = (int)((int64_t)a.kt * (t.split + 1) / a.splits);
        const int row0 = (int)t.row0 + rank * GM, n0 = t.n0 + (PAIRED ? 0 : rank * BROWS);
        const int brow = t.seg * (int)a.n + n0;
        for (int kt = k0; kt < k1; ++kt, ++i) {
          const uint32_t s = i % STAGES, bar = lead_full + 8 * s, sa = ring_u + s * STAGE, sb = sa + GM * 128;
          if (!(ok = __all_sync(FULL, tc::mbar_wait(empty + 8 * s, ((i / STAGES) & 1) ^ 1, failed)))) break;
          if (tc::elect()) {
            if (rank == 0) tc::mbar_expect_tx(full + 8 * s, CTAS * (a.a_bytes + BROWS * 128));
            const int sel = a.batch > 1 ? t.batch : (kt >= a.kt_first), x = (a.batch == 1 && kt >= a.kt_first ? kt - a.kt_first : kt) * KE;
            if (a.a_mn) {
#pragma unroll
              for (int c = 0; c < GM / 64; ++c) tc::tma_2d<CTAS>(sa + c * 8192, &a.a[sel], row0 + 64 * c, x, bar);
            } else {
              tc::tma_2d<CTAS>(sa, &a.a[sel], x, row0, bar);
            }
            if constexpr (PAIRED && CTAS == 2) {           // each block brings one of the two weights
              if (a.b_mn) {
#pragma unroll
                for (int c = 0; c < BROWS / 64; ++c) tc::tma_2d<CTAS>(sb + c * 8192, &a.b[rank], n0 + 64 * c, x, bar);
              } else {
                tc::tma_2d<CTAS>(sb, &a.b[rank], x, n0, bar);
              }
            } else if constexpr (PAIRED) {
              if (a.b_mn) {
#pragma unroll
                for (int c = 0; c < BN / 64; ++c)
                  tc::tma_2d<CTAS>(sb + c * 8192, &a.b[c >= BN / 128], n0 + 64 * (c % (BN / 128)), x, bar);
              } else {
                tc::tma_2d<CTAS>(sb, &a.b[0], x, n0, bar);
                tc::tma_2d<CTAS>(sb + BN * 64, &a.b[1], x, n0, bar);
              }
            } else if (a.b_mn) {
#pragma unroll
              for (int c = 0; c < BROWS / 64; ++c) tc::tma_2d<CTAS>(sb + c * 8192, &a.b[sel], n0 + 64 * c, x, bar);
            } else {
              tc::tma_2d<CTAS>(sb, &a.b[sel], x, brow, bar);
            }
          }
          __syncwarp();
        }
      }
      issued = i;
      // the last steps' stages are given back: after this no commit of the tensor core is on its way to this block's barriers
      if (ok)
        for (uint32_t j = i > STAGES ? i - STAGES : 0; j < i; ++j) tc::mbar_wait(empty + 8 * (j % STAGES), (j / STAGES) & 1, failed);
    } else if (warp == EPI_WARPS + 1) {
      // ---- tensor core (of a pair: the even block's)
      uint32_t i = 0, acc = 0;                             // acc: accumulators begun (tiles, or blocks of k)
      bool ok = true;
      const uint32_t adv_a = a.a_mn ? 2048 >> 4 : 32 >> 4, adv_b = a.b_mn ? 2048 >> 4 : 32 >> 4;   // one mma's k within a stage
      for (uint32_t w = w0; rank == 0 && w < a.work && ok; w += wstep) {
        const Tile t = find_tile<CTAS>(a, w, BN_OUT, lane);
        if (t.rows == 0) continue;
        const int k0 = (int)((int64_t)a.kt * t.split / a.splits), k1 = (int)((int64_t)a.kt * (t.split + 1) / a.splits);
        for (int kt = k0; kt < k1; ++kt, ++i) {
          const uint32_t s = i % STAGES, d = tmem + (acc & 1) * BN;
          // the step's operands and, where an accumulator begins, its release: odd lanes wait for the one, even lanes for the other
          const bool mine = (FP8 || kt == k0) && (lane & 1) == 0;
          const uint32_t bar = mine ? acc_empty + 8 * (acc & 1) : full + 8 * s, parity = mine ? ((acc >> 1) & 1) ^ 1 : (i / STAGES) & 1;
          if (!(ok = __all_sync(FULL, tc::mbar_wait(bar, parity, failed)))) break;
          tc::after_sync();
          const bool last = FP8 || kt == k1 - 1;
          if (tc::elect()) {
            const uint64_t da = tc::operand(ring_u + s * STAGE, a.a_mn), db = tc::operand(ring_u + s * STAGE + GM * 128, a.b_mn);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) tc::mma<CTAS, FP8>(d, da + kk * adv_a, db + kk * adv_b, a.idesc, (kk > 0 || (!FP8 && kt > k0)) ? 1u : 0u);
            tc::commit<CTAS>(empty + 8 * s);
            if (last) tc::commit<CTAS>(acc_full + 8 * (acc & 1));
          }
          __syncwarp();
          if (last) ++acc;
        }
      }
    }
  } else {
    if constexpr (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ---- epilogue: warp w reads lanes 32 (w % 4) .. and part w / 4 of the columns
    const int cpart = warp >> 2, quad = warp & 3;
    uint8_t *stg = ring + RING_BYTES + warp * STAGING;
    const uint32_t lead_empty = CTAS == 2 ? tc::in_block(acc_empty, 0) : acc_empty;
    uint32_t acc = 0, tiles = 0;                         // accumulators read; tiles of codes finished
    bool ok = true;
    // GATED_GRAD: chunk c of work item w of dh, on its way into the upper half of the staging buffer
    auto fetch_dh = [&](const Tile &t, int c) {
      if (t.rows > 0) {
        fetch_chunk(a.dh, a.n, t.row0 + rank * GM + quad * 32, t.rows - rank * GM - quad * 32, (int64_t)t.n0 + cpart * (BN_OUT / PARTS) + 32 * c, a.n, stg + 2048, lane);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    Tile next{};
    if (w0 < a.work) next = find_tile<CTAS>(a, w0, BN_OUT, lane);
    if (MODE == GATED_GRAD && a.dh_vec && a.splits == 1) fetch_dh(next, 0);
    for (uint32_t w = w0; w < a.work && ok; w += wstep) {
      const Tile t = next;
      next.rows = 0;
      if (w + wstep < a.work) next = find_tile<CTAS>(a, w + wstep, BN_OUT, lane);
      if (t.rows == 0) continue;
      const int k0 = (int)((int64_t)a.kt * t.split / a.splits), k1 = (int)((int64_t)a.kt * (t.split + 1) / a.splits);
      const int rows = min(32, t.rows - rank * GM - quad * 32);     // of this warp; may be <= 0
      const int64_t row0 = t.row0 + rank * GM + quad * 32;
      // accumulator column of chunk c, and the output column that it stands for
      auto acc_col = [&](int c) {
        return PAIRED ? (c < NCH / 2 ? 0 : BN / 2) + cpart * (BN / 2 / PARTS) + 32 * (c % (NCH / 2 ? NCH / 2 : 1)) : cpart * (BN / PARTS) + 32 * c;
      };
      auto out_col = [&](int c) { return (int64_t)t.n0 + cpart * (BN_OUT / PARTS) + 32 * c; };
      float *part = a.splits > 1 ? a.part + ((int64_t)(t.split * a.batch + t.batch) * a.m) * a.ld_part : nullptr;
      auto release = [&] {
        tc::before_sync();
        __syncwarp();
        if (lane == 0) tc::arrive<CTAS>(lead_empty + 8 * (acc & 1));
      };

      // one finished chunk of a plain product
      auto put = [&](float (&v)[32], int c) {
        if (part) store_chunk(v, GPHL_F32, true, part, a.ld_part, row0, rows, out_col(c), a.n, stg, lane);
        else store_chunk(v, a.out_type, a.out_vec, a.out[t.batch], a.ld_out, row0, rows, out_col(c), a.n, stg, lane);
      };
      // one finished pair of chunks (g is overwritten by the result)
      auto put_pair = [&](float (&g)[32], float (&u)[32], int c) {
        if (part) {
          store_chunk(g, GPHL_F32, true, part, a.ld_part, row0, rows, out_col(c), a.n, stg, lane);
          store_chunk(u, GPHL_F32, true, part + a.part_u, a.ld_part, row0, rows, out_col(c), a.n, stg, lane);
          return;
        }
        if constexpr (MODE == GATED_GRAD) {
          uint32_t dh[16];
          load_chunk(dh, a.dh_vec, a.dh, a.n, row0, rows, out_col(c), a.n, stg + 2048, lane);
          if (a.dh_vec) fetch_dh(c + 1 < NCH / 2 ? t : next, c + 1 < NCH / 2 ? c + 1 : 0);
          auto grads = [&](auto type) {
            with_activation(a.act, [&](auto k) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float lo, hi;
                unpack16<decltype(type)::value>(dh[i], lo, hi);
                gate_grads2<decltype(k)::value>(lo, hi, g[2 * i], g[2 * i + 1], u[2 * i], u[2 * i + 1]);
              }
            });
          };
          if (a.out_type == GPHL_BF16) grads(std::integral_constant<int, GPHL_BF16>());
          else grads(std::integral_constant<int, GPHL_F16>());
          store_chunk(g, a.out_type, true, a.out[0], a.ld_out, row0, rows, out_col(c), a.ld_out, stg, lane);
          store_chunk(u, a.out_type, true, a.out[1], a.ld_out, row0, rows, out_col(c), a.ld_out, stg, lane);
          return;
        }
        if (a.g) {
          store_chunk(g, GPHL_F32, true, a.g, a.ld_gu, row0, rows, out_col(c), a.n, stg, lane);
          store_chunk(u, GPHL_F32, true, a.u, a.ld_gu, row0, rows, out_col(c), a.n, stg, lane);
        }
        with_activation(a.act, [&](auto k) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) gate2<decltype(k)::value>(g[i], g[i + 1], u[i], u[i + 1]);
        });
        if (!FP8 || !a.q) store_chunk(g, a.out_type, a.out_vec, a.out[0], a.ld_out, row0, rows, out_col(c), a.n, stg, lane);
      };

      if constexpr (FP8) {
        uint64_t sum[NCH][16];                           // pairs of neighbouring columns: packed multiply-adds
#pragma unroll
        for (int c = 0; c < NCH; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[c][i] = 0;
        // The row scales of SCALES blocks ahead come into the warp's staging buffer by asynchronous 4-byte copies, two groups in turn (a
        // load per block into a register left its latency between any two accumulators: 0.72 us a block of a 128 x 256 tile).
        // Rows that are stored nowhere read the scale of one that is.
        const float *sx = a.a_scale + (rows > 0 ? row0 + min(lane, rows - 1) : 0) * a.a_scale_row;
        float *const held = reinterpret_cast<float *>(stg) + lane;                        // block kt at ((kt - k0) % (2 SCALES)) * 32
        auto fetch = [&](int first) {
          for (int kt = first; kt < min(first + SCALES, k1); ++kt) tc::copy4(held + ((kt - k0) % (2 * SCALES)) * 32, sx + kt * a.a_scale_block);
          asm volatile("cp.async.commit_group;" ::: "memory");
        };
        fetch(k0);
        fetch(k0 + SCALES);
        // the columns of one part lie inside one 128-block of the weight's scales
        const int nb = min((t.n0 + (PAIRED ? 0 : cpart * (BN / PARTS))) / 128, a.scale_nb - 1);
        const float *sw0 = a.b_scale[0] + ((int64_t)t.seg * a.scale_nb + nb) * a.scale_kb;
        const float *sw1 = PAIRED ? a.b_scale[1] + (int64_t)nb * a.scale_kb : sw0;
        float next_w0 = __ldg(sw0 + k0), next_w1 = PAIRED ? __ldg(sw1 + k0) : 0.f;
        auto ready = [&] {
          ok = __all_sync(FULL, tc::mbar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1, failed));
          tc::after_sync();
        };
        // Two chunks in registers in turn: while one is scaled and added, the next is on its way from tensor memory, the first of the next
        // accumulator included.
        auto addr = [&](int c) { return tmem + (acc & 1) * BN + ((uint32_t)(quad * 32) << 16) + acc_col(c); };
        float v[2][32];
        ready();
        if (ok) tc::ld32(addr(0), v[0]);
        for (int kt = k0; kt < k1 && ok; ++kt) {
          if ((kt - k0) % SCALES == 0) {
            if (kt > k0) fetch(kt + SCALES);             // into the group that has just been used up (by this thread alone)
            asm volatile("cp.async.wait_group 1;" ::: "memory");
          }
          const float x = held[((kt - k0) % (2 * SCALES)) * 32];
          const float s0 = x * next_w0, s1 = PAIRED ? x * next_w1 : s0;
          const uint64_t p0 = pack2(s0, s0), p1 = PAIRED ? pack2(s1, s1) : p0;
          if (kt + 1 < k1) {
            next_w0 = __ldg(sw0 + kt + 1);
            if (PAIRED) next_w1 = __ldg(sw1 + kt + 1);
          }
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            constexpr int LAST = NCH - 1;
            float (&u)[32] = v[NCH == 1 ? 0 : c & 1];
            tc::ld_wait(u);
            if (c < LAST) {
              tc::ld32(addr(c + 1), v[(c + 1) & 1]);
            } else {
              release();
              ++acc;
              if (NCH > 1 && kt + 1 < k1) {
                ready();
                if (ok) tc::ld32(addr(0), v[0]);
              }
            }
            const uint64_t s = PAIRED && c >= NCH / 2 ? p1 : p0;
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[c][i] = ffma2(pack2(u[2 * i], u[2 * i + 1]), s, sum[c][i]);
            if (NCH == 1 && kt + 1 < k1) {
              ready();
              if (ok) tc::ld32(addr(0), v[0]);
            }
          }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        if (!ok) break;
        __syncwarp();                                    // the staging buffer changes hands
        auto unpack = [](const uint64_t (&p)[16], float (&v)[32]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) unpack2(p[i], v[2 * i], v[2 * i + 1]);
        };
        if constexpr (PAIRED) {
          float g[NCH / 2][32];
#pragma unroll
          for (int c = 0; c < NCH / 2; ++c) {
            float u[32];
            unpack(sum[c], g[c]);
            unpack(sum[c + NCH / 2], u);
            put_pair(g[c], u, c);
          }
          if (a.q && !part) {
            // the tile's columns are one block of 128 of the codes, shared by the warps of these rows
            float big = 0.f;
#pragma unroll
            for (int c = 0; c < NCH / 2; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i) big = fmaxf(big, out_col(c) + i < a.n ? finite_abs(g[c][i]) : 0.f);
            // Joined as exponents, in memory of their own (the staging buffer's row scales of the next tile may be on their way before the other warp
            // has read).  Two slots in turn: one is written again only after the others' next arrivals, which follow their reads.
            int e = fp8_exponent(big);
            s_exp[tiles & 1][warp][lane] = (int8_t)e;
            __syncwarp();
            if (lane == 0) tc::arrive<1>(pair + 8 * quad);
            ok = __all_sync(FULL, tc::mbar_wait(pair + 8 * quad, tiles & 1, failed));
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) e = max(e, (int)s_exp[tiles & 1][quad + 4 * i][lane]);
            ++tiles;
            if (cpart == 0 && lane < rows) a.q_scale[(int64_t)(t.n0 / 128) * a.q_scale_stride + row0 + lane] = pow2f(e);
#pragma unroll
            for (int c = 0; c < NCH / 2; ++c) store_code_chunk(g[c], pow2f(-e), a.q, a.ld_out, row0, rows, out_col(c), a.n, stg, lane);
          }
        } else {
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            float v[32];
            unpack(sum[c], v);
            put(v, c);
          }
        }
      } else {
        ok = __all_sync(FULL, tc::mbar_wait(acc_full + 8 * (acc & 1), (acc >> 1) & 1, failed));
        if (!ok) break;
        tc::after_sync();
        const uint32_t taddr = tmem + (acc & 1) * BN + ((uint32_t)(quad * 32) << 16);
        if constexpr (PAIRED) {
#pragma unroll
          for (int c = 0; c < NCH / 2; ++c) {
            float g[32], u[32];
            tc::ld32(taddr + acc_col(c), g);
            tc::ld32(taddr + acc_col(c + NCH / 2), u);
            tc::ld_wait(g);
            tc::ld_wait(u);
            if (c == NCH / 2 - 1) release();
            put_pair(g, u, c);
          }
        } else {
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            float v[32];
            tc::ld32(taddr + acc_col(c), v);
            tc::ld_wait(v);
            if (c == NCH - 1) release();
            put(v, c);
          }
        }
        ++acc;
      }
    }
  }
  __syncwarp();
  tc::before_sync();
  __syncthreads();
  if (s_failed) {                                        // what is in flight lands before the block leaves
    int unused = 0;
    if (threadIdx.x == 0) atomicAdd(&g_gemm_wait_timeouts, 1);
    if (rank == 0 && warp == EPI_WARPS && lane == 0)     // (the bytes of both blocks are counted on the even block's barriers)
      for (uint32_t j = issued > STAGES ? issued - STAGES : 0; j < issued; ++j) tc::mbar_wait(full + 8 * (j % STAGES), (j / STAGES) & 1, &unused);
    if (rank == 0 && warp == EPI_WARPS + 1 && lane == 0) {
      tc::commit<CTAS>(drain);
      tc::mbar_wait(drain, 0, &unused);
    }
    __syncwarp();
  }
  if (CTAS == 2) tc::cluster_sync();                     // neither block leaves while the other may reach into its shared memory
  else __syncthreads();
  if (warp == EPI_WARPS + 1) tc::dealloc<CTAS>(tmem, 2 * BN);
}

// ---- joining the parts of a split k ------------------------------------------------------------------------------------------------

// A warp per (row, 128 columns), 4 neighbouring columns a lane; the parts are added in order, in groups, so that a sum over very many rows (3052
// parts for 100 million) rounds a running sum about as often as a group is long and groups are many.
constexpr int JOIN_GROUP = 64;
template <int MODE> __global__ void __launch_bounds__(256) gemm_join_kernel(const GemmArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t blocks = (a.n + 127) / 128, item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t row_b = item / blocks, c0 = (item - row_b * blocks) * 128 + lane * 4;
  const int b = (int)(row_b / a.m);
  const int64_t row = row_b - (int64_t)b * a.m;
  if (b >= a.batch) return;
  if (a.ptr && (row < __ldg(a.ptr) || row >= __ldg(a.ptr + a.types))) return;      // a row of no type
  float4 g = make_float4(0, 0, 0, 0), u = g;
  if (c0 < a.n) {
    for (int s0 = 0; s0 < a.splits; s0 += JOIN_GROUP) {
      float4 pg = make_float4(0, 0, 0, 0), pu = pg;
      for (int s = s0; s < min(s0 + JOIN_GROUP, a.splits); ++s) {
        const float *p = a.part + ((int64_t)(s * a.batch + b) * a.m + row) * a.ld_part + c0;
        const float4 v = *reinterpret_cast<const float4 *>(p);
        pg.x += v.x, pg.y += v.y, pg.z += v.z, pg.w += v.w;
        if (MODE != LINEAR) {
          const float4 t = *reinterpret_cast<const float4 *>(p + a.part_u);
          pu.x += t.x, pu.y += t.y, pu.z += t.z, pu.w += t.w;
        }
      }
      g.x += pg.x, g.y += pg.y, g.z += pg.z, g.w += pg.w;
      u.x += pu.x, u.y += pu.y, u.z += pu.z, u.w += pu.w;
    }
  }
  float o[4] = {g.x, g.y, g.z, g.w};
  if (MODE == GATED_GRAD) {
    float gg[4] = {g.x, g.y, g.z, g.w}, uu[4] = {u.x, u.y, u.z, u.w}, dh[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = row * a.n + c0 + j;
      dh[j] = c0 + j >= a.n ? 0.f : a.out_type == GPHL_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(a.dh)[i]) : __half2float(static_cast<const __half *>(a.dh)[i]);
    }
    with_activation(a.act, [&](auto k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) gate_grads<decltype(k)::value>(dh[j], gg[j], uu[j]);
    });
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j < a.n) {
        const int64_t i = row * a.ld_out + c0 + j;
        if (a.out_type == GPHL_BF16) {
          static_cast<__nv_bfloat16 *>(a.out[0])[i] = __float2bfloat16_rn(gg[j]);
          static_cast<__nv_bfloat16 *>(a.out[1])[i] = __float2bfloat16_rn(uu[j]);
        } else {
          static_cast<__half *>(a.out[0])[i] = __float2half_rn(gg[j]);
          static_cast<__half *>(a.out[1])[i] = __float2half_rn(uu[j]);
        }
      }
    return;
  }
  if (MODE == GATED) {
    const float gg[4] = {g.x, g.y, g.z, g.w}, uu[4] = {u.x, u.y, u.z, u.w};
    if (a.g && c0 < a.n) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < a.n) a.g[row * a.ld_gu + c0 + j] = gg[j], a.u[row * a.ld_gu + c0 + j] = uu[j];
    }
    with_activation(a.act, [&](auto k) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = activate<decltype(k)::value>(gg[j]) * uu[j];
    });
    if (a.q) {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (c0 + j >= a.n) o[j] = 0.f;
        big = fmaxf(big, finite_abs(o[j]));
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) big = fmaxf(big, __shfl_xor_sync(FULL, big, d));
      const int e = fp8_exponent(big);
      const float inv = pow2f(-e);
      if (c0 < a.ld_out)
        *reinterpret_cast<uint32_t *>(a.q + row * a.ld_out + c0) = e4m3x2(o[0] * inv, o[1] * inv) | (e4m3x2(o[2] * inv, o[3] * inv) << 16);
      if (lane == 0) a.q_scale[(c0 / 128) * a.q_scale_stride + row] = pow2f(e);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c0 + j < a.n) {
      const int64_t i = row * a.ld_out + c0 + j;
      if (a.out_type == GPHL_F32) static_cast<float *>(a.out[b])[i] = o[j];
      else if (a.out_type == GPHL_BF16) static_cast<__nv_bfloat16 *>(a.out[b])[i] = __float2bfloat16_rn(o[j]);
      else static_cast<__half *>(a.out[b])[i] = __float2half_rn(o[j]);
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}
// Boxes of 128 bytes (the swizzle span) x `box_rows` rows.  The inner coordinate of every load is a multiple of 64 16-bit or 128 8-bit
// elements, which keeps each copy on a 16-byte boundary.
static int encode(CUtensorMap *map, const Matrix &x, int type, bool fp8, int box_rows, const char *what) {
  const int size = fp8 ? 1 : 2;
  if (!aligned16(x.p) || (x.ld * size) % 16 != 0)
    return fail(GPHL_ERR_UNSUPPORTED, "%s: operands must start on 16-byte boundaries and have rows a multiple of 16 bytes apart", what);
  const cuuint64_t dim[2] = {(cuuint64_t)x.cols, (cuuint64_t)x.rows}, stride[1] = {(cuuint64_t)(x.ld * size)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUtensorMapDataType t = fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : type == GPHL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = encode_fn()(map, t, 2, const_cast<void *>(x.p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GPHL_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return GPHL_OK;
}

struct Shape {
  int bn, ctas, splits;
  int64_t tiles_m, tiles_n;
  int32_t kt, batch;
};
// Tile width, blocks per tile and parts of k by an estimate of the time, in microseconds: waves of tiles times steps times the measured
// time of a step (128 bytes of k: 0.40 for a pair of blocks with 256 columns in 16 bits, 0.48 in e4m3, 0.50 for one block, less for narrower
// tiles, which read A more often, but 0.41 in e4m3, where an accumulator's way to the epilogue and back takes that long), at least the time of the
// operands' bytes at the rate that tiles of that width, or the SMs at work, were seen to stream them (5 x 4096 -> 11264 in bf16 on 88 SMs 41.8,
// in 3 parts on all 38.6; 64 x 4096 -> 8192 in e4m3 with 64 columns a tile 19.2, with 128 and 2 parts 16.2), and for parts their join (3, and the parts' fp32 sums written and read at 5 TB/s).  In e4m3: 2048 x 11264 -> 4096 takes 112 with k whole, 141 in
// 2 parts; 1 x 4096 -> 8192 18.7 in 2 parts, 14.0 in 4; 1 x 16384 -> 16384 73 with 128 columns a tile, 59 with 256 and 2 parts.
// The tensor core truncates when it adds to an fp32 accumulator: over k values of one sign a sum loses 5.4e-9 k of itself (65,536: 3.5e-4,
// 524,288: 3.0e-3), so in 16 bits no part is longer than CHAIN (1.8e-4, below half a step of the results), however many parts that makes (both
// weights' gradients over m rows: m k f / 4096 bytes of parts, at most k / 16384 of the operands' own); the join adds with rounding.
constexpr int64_t CHAIN = 32768;
static bool paired(const GemmCall &c) { return c.dual == DUAL_GATED || c.dual == DUAL_GATED_GRAD; }
static int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}
static Shape shape_of(const GemmCall &c, int sms) {
  const int ke = c.fp8 ? 128 : 64;
  const bool two = paired(c);
  const int64_t per = (c.k + ke - 1) / ke, wide = two ? 2 * c.n : c.n;
  const double size = c.fp8 ? 1.0 : 2.0, pairs = c.dual == DUAL_NONE ? 1.0 : 2.0;
  const double bytes = ((two ? 1.0 : pairs) * c.m * c.k + pairs * c.types * c.n * c.k) * size;
  Shape best{};
  double best_us = 1e30;
  for (int bn = 256; bn >= 64; bn /= 2) {
    if (two && bn == 64) continue;
    if (c.q && bn != 256) continue;                      // a tile is one block of 128 codes
    if (bn > 64 && wide <= bn / 2 && !(two && bn == 128) && !c.q) continue;
    for (int ctas = 1; ctas <= 2; ++ctas) {
      // pairs of blocks where the tiles of 256 rows are whole but for the last
      if (ctas == 2 && (bn != 256 || c.m <= GM || (c.ptr && c.m < 4 * GM * c.types))) continue;
      Shape s{};
      s.bn = bn, s.ctas = ctas, s.batch = c.dual == DUAL_BATCH ? 2 : 1;
      s.kt = (int32_t)(c.dual == DUAL_CONCAT ? 2 * per : per);
      s.tiles_m = (c.m + ctas * GM - 1) / (ctas * GM) + (c.ptr ? std::min<int64_t>(c.types, c.m) : 0);
      const int out = two ? bn / 2 : bn, units = sms / ctas;
      s.tiles_n = (c.n + out - 1) / out;
      const int64_t items = s.tiles_m * s.tiles_n * s.batch;
      const double most = bn == 256 ? 5.5e6 : bn == 128 ? 4.0e6 : 3.2e6, each = 0.052e6;      // bytes a microsecond, of all SMs and of one
      const double step = bn == 256 ? (ctas == 1 ? 0.50 : c.fp8 ? 0.48 : 0.40) : c.fp8 ? 0.41 : bn == 128 ? 0.32 : 0.24;
      const double finish = c.fp8 ? bn * (3.0 / 256) : 1.5;       // a tile's end (e4m3: the sums are in registers, no accumulator hides it)
      const int least = c.fp8 ? 1 : (int)((s.kt * (int64_t)ke + CHAIN - 1) / CHAIN);
      for (int p = least; p == least || (p <= 64 && p * 4 <= s.kt && items < 2 * units && items * p <= 8 * units); ++p) {
        const double waves = (double)((items * p + units - 1) / units);
        const double rate = std::min(most, each * ctas * (double)std::min<int64_t>(items * p, units));
        double us = std::max(waves * ((double)s.kt / p * step + finish), bytes / rate);
        if (p > 1) us += 3.0 + (double)p * s.batch * c.m * wide * 8.0 / 5e6;
        if (us < best_us * 0.999) best_us = us, best = s, best.splits = p;
      }
    }
  }
  return best;
}
static int64_t part_ld(const GemmCall &c) { return (c.n + 3) / 4 * 4 * (paired(c) ? 2 : 1); }

int64_t gemm_workspace_bytes(const GemmCall &c) {
  if (c.m <= 0 || c.n <= 0 || c.k <= 0) return 0;
  const int few = few_rows_parts(c);
  if (few >= 0) return (int64_t)few * c.m * part_ld(c) * (int64_t)sizeof(float);
  const Shape s = shape_of(c, sm_count());
  return s.splits > 1 ? (int64_t)s.splits * s.batch * c.m * part_ld(c) * (int64_t)sizeof(float) : 0;
}

template <int BN, int CTAS, int EPI_WARPS, bool FP8, int MODE> static int run(const GemmArgs &a, int sms, cudaStream_t stream) {
  const auto kernel = gemm_kernel<BN, CTAS, EPI_WARPS, FP8, MODE>;
  // a per-device attribute of the function: set on every call (a process may use several GPUs)
  GPHL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GEMM_SMEM));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(a.work, sms / CTAS) * CTAS)), cfg.blockDim = dim3(gemm_threads(EPI_WARPS, FP8));
  cfg.dynamicSmemBytes = GEMM_SMEM, cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CTAS, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = CTAS > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, a);
  return launched("gemm_kernel");
}
template <bool FP8, int MODE> static int run_shape(const Shape &s, const GemmArgs &a, int sms, cudaStream_t stream) {
  // 16 epilogue warps where they have an activation to compute (300,000 x 256 -> 1024 forward: 337 us, with 8 warps 391, an element at a time; 320 since
  // silu takes two), 8 where they only store or hold sums
  constexpr int WARPS = FP8 || MODE == LINEAR ? 8 : 16;
  if (s.ctas == 2) return run<256, 2, WARPS, FP8, MODE>(a, sms, stream);
  if (s.bn == 256) return run<256, 1, WARPS, FP8, MODE>(a, sms, stream);
  if constexpr (MODE == LINEAR)
    if (s.bn == 64) return run<64, 1, 8, FP8, MODE>(a, sms, stream);
  return run<128, 1, 8, FP8, MODE>(a, sms, stream);
}

// What finishes a tile, or joins parts.
static GemmArgs finish_args(const GemmCall &c) {
  GemmArgs a{};
  a.m = c.m, a.n = c.n, a.batch = c.dual == DUAL_BATCH ? 2 : 1, a.types = (int32_t)c.types, a.ptr = c.ptr;
  a.out[0] = c.out[0], a.out[1] = c.out[1], a.ld_out = c.ld_out, a.out_type = c.out_type, a.act = c.act;
  a.out_vec = aligned16(c.out[0]) && aligned16(c.out[1]) && (c.ld_out * (c.out_type == GPHL_F32 ? 4 : 2)) % 16 == 0;
  a.dh = c.dh, a.dh_vec = aligned16(c.dh) && c.n % 8 == 0;
  a.g = c.g, a.u = c.u, a.ld_gu = c.ld_gu, a.q = c.q, a.q_scale = c.q_scale, a.q_scale_stride = c.q_scale_stride;
  a.part = static_cast<float *>(c.workspace), a.ld_part = part_ld(c), a.part_u = (c.n + 3) / 4 * 4;
  return a;
}
static int join(const GemmCall &c, GemmArgs &a, int parts, cudaStream_t stream) {
  a.splits = parts;
  const unsigned blocks = (unsigned)((a.batch * c.m * ((c.n + 127) / 128) + 7) / 8);
  if (c.dual == DUAL_GATED_GRAD) gemm_join_kernel<GATED_GRAD><<<blocks, 256, 0, stream>>>(a);
  else if (c.dual == DUAL_GATED) gemm_join_kernel<GATED><<<blocks, 256, 0, stream>>>(a);
  else gemm_join_kernel<LINEAR><<<blocks, 256, 0, stream>>>(a);
  return launched("gemm_join_kernel");
}

int gemm(const GemmCall &c, const char *what, cudaStream_t stream) {
  int dev = 0, sms = 0;
  GPHL_CUDA(cudaGetDevice(&dev));
  GPHL_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  GemmArgs a = finish_args(c);
  if (c.k == 0) return join(c, a, 0, stream);            // no parts: sums of nothing
  const int few = few_rows_parts(c);
  if (few >= 0) {
    GPHL_REQUIRE(few == 0 || (a.part && aligned16(a.part)), "%s: the workspace is missing or not 16-byte aligned", what);
    const int rc = few_rows(c, a.part, a.ld_part, a.part_u, what, stream);
    return rc != GPHL_OK || few == 0 ? rc : join(c, a, few, stream);
  }
  if (!encode_fn()) return fail(GPHL_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available from this driver", what);
  GPHL_CUDA(cudaSetDevice(dev));       // tensor maps are made by the driver, which wants a context: a thread's first call (of an autograd thread) finds none
  const Shape s = shape_of(c, sms);
  const bool pairs_of_b = paired(c);
  const int pairs = c.dual == DUAL_NONE ? 1 : 2;
  // With fewer rows than a tile, only they are brought: the tensor core multiplies whatever the stage's other rows hold into rows of the
  // accumulator that nobody reads.  (A box of 128 rows costs its time even where it is zeros: 5 x 4096 -> 11264 47 us.)
  const int a_rows = c.a_mn ? 64 : (int)std::min<int64_t>(GM, (c.m + 7) / 8 * 8);
  a.a_bytes = c.a_mn ? GM * 128 : a_rows * 128;
  for (int i = 0; i < pairs; ++i) {
    if (i == 0 || !pairs_of_b) {
      int rc = encode(&a.a[i], c.a[i], c.in_type, c.fp8, a_rows, what);
      if (rc != GPHL_OK) return rc;
    }
    int rc = encode(&a.b[i], c.b[i], c.in_type, c.fp8, c.b_mn ? 64 : pairs_of_b ? s.bn / 2 : s.bn / s.ctas, what);
    if (rc != GPHL_OK) return rc;
  }
  const int64_t work = s.tiles_m * s.tiles_n * s.batch * s.splits;
  GPHL_REQUIRE(work + 65536 < INT32_MAX, "%s: too many tiles", what);
  a.tiles_m = (uint32_t)s.tiles_m, a.tiles_n = (uint32_t)s.tiles_n, a.work = (uint32_t)work;
  a.by_plane.set(a.tiles_m * a.tiles_n), a.by_band.set(RASTER * a.tiles_n), a.by_last.set(a.tiles_m % RASTER ? a.tiles_m % RASTER : RASTER);
  a.splits = s.splits, a.kt = s.kt, a.kt_first = c.dual == DUAL_CONCAT ? s.kt / 2 : s.kt;
  a.a_mn = c.a_mn, a.b_mn = c.b_mn;
  a.idesc = (1u << 4) | ((uint32_t)(s.bn >> 3) << 17) | ((uint32_t)(GM * s.ctas >> 4) << 24);
  if (!c.fp8) a.idesc |= (c.in_type == GPHL_BF16 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)c.a_mn << 15) | ((uint32_t)c.b_mn << 16);
  a.a_scale = c.a_scale, a.b_scale[0] = c.b_scale[0], a.b_scale[1] = c.b_scale[1];
  a.a_scale_row = c.a_scale_row, a.a_scale_block = c.a_scale_block;
  a.scale_kb = (int32_t)((c.k + 127) / 128), a.scale_nb = (int32_t)((c.n + 127) / 128);
  GPHL_REQUIRE(s.splits == 1 || (a.part && aligned16(a.part)), "%s: the workspace is missing or not 16-byte aligned", what);
  int rc;
  if (c.dual == DUAL_GATED_GRAD) rc = run_shape<false, GATED_GRAD>(s, a, sms, stream);
  else if (c.dual == DUAL_GATED) rc = c.fp8 ? run_shape<true, GATED>(s, a, sms, stream) : run_shape<false, GATED>(s, a, sms, stream);
  else rc = c.fp8 ? run_shape<true, LINEAR>(s, a, sms, stream) : run_shape<false, LINEAR>(s, a, sms, stream);
  return rc != GPHL_OK || s.splits == 1 ? rc : join(c, a, s.splits, stream);
}

int gemm_wait_timeouts(int *count) {
  GPHL_CUDA(cudaMemcpyFromSymbol(count, g_gemm_wait_timeouts, sizeof(int)));
  return GPHL_OK;
}
int gemm_reset_wait_timeouts() {
  const int zero = 0;
  GPHL_CUDA(cudaMemcpyToSymbol(g_gemm_wait_timeouts, &zero, sizeof(int)));
  return GPHL_OK;
}

}  // namespace gphl

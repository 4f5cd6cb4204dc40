// b200_gemm_blocks: matrix products of 8-bit operands with a scale for each block of 128 (quantize.cu).
//
// C[m, n] = act(sum over k-blocks of sa(m, kb) sb(n, kb) (sum over the block's k of a[m, k] b[n, k]) + bias): the
// inner sum is of products of 8-bit values, which fp32 holds exactly; it is taken to fp32 registers once per
// block of 128 and multiplied by the product of the two scales there, or by one after the other where their product is out
// of range (Scaling).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "engine.h"
#include "epilogue.cuh"
#include "ptx.cuh"
#include "tc_common.cuh"

namespace b200 {

// An operand as the kernels see it: element (i, k), i = m or n, at data[i * si + k * sk]; its scale at
// scales[(i >> shift) * ss_i + (k >> 7) * ss_k].
struct BlockOperand {
  const uint8_t *data;
  long long si, sk;
  const float *scales;
  long long ss_i, ss_k;
  int shift;  // 0: a scale per row or column, 7: per 128 x 128 tile
  int e5m2;
};

struct BlocksParams {
  long long M, N, K;
  void *C;
  long long ldc;
  int c_bf16;
  Epilogue ep;
};

__device__ __forceinline__ float f8_to_float(uint8_t v, int e5m2) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, e5m2 ? __NV_E5M2 : __NV_E4M3)));
}

// Whether the product of two scales is a normal number, and can multiply a block's sum as it is. As one comparison: the magnitude's
// bits less those of the least normal number, both doubled, so that what lies below wraps round.
constexpr uint32_t RANGE = 254u << 24;
__device__ __forceinline__ uint32_t away_from_range(float product) { return (__float_as_uint(product) << 1) - (1u << 24); }
__device__ __forceinline__ bool in_range(float product) { return away_from_range(product) < RANGE; }

// The product of two scales in a form that can be applied in any case. The sum `part` of a block is 0 or between 2^-32 and 2^39
// (or no finite number). Of two scales whose product is out of range, the one that is farther out is brought nearer by
// 2^64, which is exact, and the result is put back as it is added: a product above the range has a scale above 2^63 and the
// other one is 1 or more, one below has a scale below 2^-63 and the other one is 2^23 at most, so nothing in between
// leaves the range unless the result has by far. Which form is taken depends on the two scales alone.
struct Scaling {
  float first, second, last;  // 1, 1 and the product where that is in range
  __device__ __forceinline__ Scaling(float a, float b) {
    const float product = __fmul_rn(a, b);
    const bool fine = in_range(product), above = fabsf(product) > 1.f, swap = (fabsf(a) > fabsf(b)) != above;
    first = fine ? 1.f : (swap ? b : a) * (above ? 0x1p-64f : 0x1p64f);
    second = fine ? 1.f : (swap ? a : b);
    last = fine ? product : (above ? 0x1p64f : 0x1p-64f);
  }
  __device__ __forceinline__ float near(float part) const { return __fmul_rn(__fmul_rn(part, first), second); }
  __device__ __forceinline__ float add(float acc, float part) const { return __fmaf_rn(near(part), last, acc); }
};

// Any layout, alignment and size: 64 x 64 outputs per CTA, 4 x 4 per thread, 32 k at a time through shared memory.
constexpr int GB_T = 64, GB_K = 32;
__global__ void __launch_bounds__(256) gemm_blocks_simt_kernel(const BlockOperand a, const BlockOperand b, const BlocksParams p) {
  ptx::grid_begin();
  __shared__ float sa[GB_K][GB_T + 1], sb[GB_K][GB_T + 1];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const long long tiles_m = (p.M + GB_T - 1) / GB_T, tiles = tiles_m * ((p.N + GB_T - 1) / GB_T);
  for (long long t = blockIdx.x; t < tiles; t += gridDim.x) {
    const long long m0 = t % tiles_m * GB_T, n0 = t / tiles_m * GB_T;
    float acc[4][4] = {};
    for (long long k0 = 0; k0 < p.K; k0 += 128) {
      float part[4][4] = {};
      for (long long k1 = k0; k1 < min(k0 + 128, p.K); k1 += GB_K) {
        __syncthreads();
        // consecutive threads along whichever index is contiguous
        for (int i = threadIdx.x; i < GB_T * GB_K; i += 256) {
          const int ka = a.sk == 1 ? i % GB_K : i / GB_T, ra = a.sk == 1 ? i / GB_K : i % GB_T;
          const int kb = b.sk == 1 ? i % GB_K : i / GB_T, rb = b.sk == 1 ? i / GB_K : i % GB_T;
          sa[ka][ra] = m0 + ra < p.M && k1 + ka < p.K ? f8_to_float(a.data[(m0 + ra) * a.si + (k1 + ka) * a.sk], a.e5m2) : 0.f;
          sb[kb][rb] = n0 + rb < p.N && k1 + kb < p.K ? f8_to_float(b.data[(n0 + rb) * b.si + (k1 + kb) * b.sk], b.e5m2) : 0.f;
        }
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < GB_K; ++k) {
          float va[4], vb[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            va[j] = sa[k][ty + 16 * j];
            vb[j] = sb[k][tx + 16 * j];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[i][j] = __fmaf_rn(va[i], vb[j], part[i][j]);
        }
      }
      float ra[4], rb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long m = m0 + ty + 16 * j, n = n0 + tx + 16 * j;
        ra[j] = m < p.M ? a.scales[(m >> a.shift) * a.ss_i + (k0 >> 7) * a.ss_k] : 1.f;
        rb[j] = n < p.N ? b.scales[(n >> b.shift) * b.ss_i + (k0 >> 7) * b.ss_k] : 1.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = Scaling(ra[i], rb[j]).add(acc[i][j], part[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const long long m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
        if (m >= p.M || n >= p.N) continue;
        const float v = apply_epilogue<float>(acc[i][j], p.ep, m, n);
        const long long at = m * p.ldc + n;
        if (p.c_bf16) ((__nv_bfloat16 *)p.C)[at] = __float2bfloat16_rn(v);
        else ((float *)p.C)[at] = p.ep.accumulate ? __fadd_rn(((float *)p.C)[at], v) : v;
      }
  }
}

// ------------------------------------------------------------------------------------------
// up to 16 rows of A, both operands with k contiguous: B is read, nothing else counts
// ------------------------------------------------------------------------------------------

// D += A B for 16 x 8 x 32 8-bit values, in fp32. (tcgen05 has no business here: a tile's way through shared and tensor
// memory costs more than the reading of B itself. 1 x 4096 x 4096 there: 11.5 us.)
template <bool A5, bool B5>
__device__ __forceinline__ void mma_16x8x32(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1) {
#define B200_MMA_F8(TA, TB)                                                                                                 \
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32." TA "." TB ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "      \
               "{%0, %1, %2, %3};"                                                                                         \
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                                            \
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1))
  if (A5 && B5) B200_MMA_F8("e5m2", "e5m2");
  else if (A5) B200_MMA_F8("e5m2", "e4m3");
  else if (B5) B200_MMA_F8("e4m3", "e5m2");
  else B200_MMA_F8("e4m3", "e4m3");
#undef B200_MMA_F8
}

// A block takes 16 rows of the weights w and all of x; its eight warps share the k-blocks, and their sums are added in the
// order of the warps. In a warp, lane 4 g + t holds the 16 bytes from 16 t on of every 64 of rows g and g + 8: which k an
// instruction's operands belong to does not matter as long as both operands agree. 1 x 4096 x 4096: 5.4 us in a row of calls,
// which is the host's call; reading B takes 2.6 at the copy rate.
template <int NT, bool W5, bool X5>
__global__ void __launch_bounds__(256, 2)
    gemm_blocks_skinny_kernel(const BlockOperand w, const BlockOperand x, const BlocksParams p) {
  ptx::grid_begin();
  __shared__ float s_sum[8][16][NT * 8 + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const long long n0 = (long long)blockIdx.x * 16;  // rows of w, columns of C
  const int nk = (int)((p.K + 127) / 128);
  const uint8_t *row[2 + NT];
#pragma unroll
  for (int r = 0; r < 2; ++r) row[r] = w.data + min(n0 + g + 8 * r, p.N - 1) * w.si;
#pragma unroll
  for (int j = 0; j < NT; ++j) row[2 + j] = x.data + min((long long)(j * 8 + g), p.M - 1) * x.si;
  const float *ws[2], *xs[NT][2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    ws[r] = w.scales + (min(n0 + g + 8 * r, p.N - 1) >> w.shift) * w.ss_i;
#pragma unroll
    for (int j = 0; j < NT; ++j) xs[j][r] = x.scales + (min((long long)(j * 8 + 2 * t + r), p.M - 1) >> x.shift) * x.ss_i;
  }
  const int K = (int)p.K;  // a multiple of 16
  auto bytes = [&](int r, int k) -> uint4 {
    return k < K ? __ldg(reinterpret_cast<const uint4 *>(row[r] + k)) : make_uint4(0, 0, 0, 0);
  };
  // k-blocks of w in flight per warp, 2 KB each (with two column tiles four do not fit the registers: 16 x 4096 x 4096 in the
  // loop of calls 8.0 us instead of 7.1)
  constexpr int AHEAD = NT == 1 ? 4 : 3;
  float acc[NT][4];
  // The k-blocks are added without asking whether a product of two scales is in range: how far the products go is
  // kept, and a warp that has met one out of range begins again with care.
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[j][c] = 0.f;
  for (int kb0 = warp; kb0 < nk; kb0 += 8 * AHEAD) {
    uint4 v[AHEAD][2][2];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) v[i][h][r] = bytes(r, (kb0 + 8 * i) * 128 + h * 64 + t * 16);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int kb = kb0 + 8 * i;
      if (kb >= nk) continue;
      const float sw[2] = {__ldg(ws[0] + kb * w.ss_k), __ldg(ws[1] + kb * w.ss_k)};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float sx[2] = {__ldg(xs[j][0] + kb * x.ss_k), __ldg(xs[j][1] + kb * x.ss_k)};
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 &a0 = v[i][h][0], &a1 = v[i][h][1], b = bytes(2 + j, kb * 128 + h * 64 + t * 16);
          mma_16x8x32<W5, X5>(part, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
          mma_16x8x32<W5, X5>(part, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float product = __fmul_rn(sw[c >> 1], sx[c & 1]);
          most = max(most, away_from_range(product));
          acc[j][c] = __fmaf_rn(part[c], product, acc[j][c]);
        }
      }
    }
  }
  if (__any_sync(0xffffffffu, most >= RANGE)) {
    long long first = n0;
    asm volatile("" : "+l"(first));  // addresses are worked out again: kept over the loop above they cost it registers
    auto load = [&](const BlockOperand &o, long long i, int k) -> uint4 {
      return k < K ? __ldg(reinterpret_cast<const uint4 *>(o.data + i * o.si + k)) : make_uint4(0, 0, 0, 0);
    };
    auto scale = [](const BlockOperand &o, long long i, int kb) { return __ldg(o.scales + (i >> o.shift) * o.ss_i + kb * o.ss_k); };
    auto wrow = [&](int i) { return min(first + g + 8 * i, p.N - 1); };
    auto xrow = [&](int i) { return min((long long)i, p.M - 1); };
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[j][c] = 0.f;
    for (int kb = warp; kb < nk; kb += 8) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = kb * 128 + h * 64 + t * 16;
          const uint4 a0 = load(w, wrow(0), k), a1 = load(w, wrow(1), k), b = load(x, xrow(j * 8 + g), k);
          mma_16x8x32<W5, X5>(part, a0.x, a1.x, a0.y, a1.y, b.x, b.y);
          mma_16x8x32<W5, X5>(part, a0.z, a1.z, a0.w, a1.w, b.z, b.w);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          acc[j][c] = Scaling(scale(w, wrow(c >> 1), kb), scale(x, xrow(j * 8 + 2 * t + (c & 1)), kb)).add(acc[j][c], part[c]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_sum[warp][g + 8 * (i >> 1)][j * 8 + 2 * t + (i & 1)] = acc[j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * NT * 8; i += 256) {
    const int r = i & 15, m = i >> 4;
    const long long n = n0 + r;
    if (m >= p.M || n >= p.N) continue;
    float sum = s_sum[0][r][m];
#pragma unroll
    for (int q = 1; q < 8; ++q) sum = __fadd_rn(sum, s_sum[q][r][m]);
    const float out = apply_epilogue<float>(sum, p.ep, m, n);
    const long long at = m * p.ldc + n;
    if (p.c_bf16) ((__nv_bfloat16 *)p.C)[at] = __float2bfloat16_rn(out);
    else ((float *)p.C)[at] = p.ep.accumulate ? __fadd_rn(((float *)p.C)[at], out) : out;
  }
}

// ------------------------------------------------------------------------------------------
// tensor cores
// ------------------------------------------------------------------------------------------

constexpr int GB_BM = 128;     // rows of a tile
constexpr int GB_BK = 128;     // k of a block of scales, of a ring stage and of an accumulator
constexpr int GB_SLAB = GB_BK * 128;  // bytes of 128 rows (or columns) of a k-block

struct BlocksTcParams {
  int M, N;                     // rows and columns of the tiles: M and N of the product, or N and M (swapped)
  int a_mn, b_mn;               // the operand is stored with its m / n index contiguous
  uint32_t idesc;
  const float *a_scales, *b_scales;
  long long as_i, as_k, bs_i, bs_k;  // BlockOperand's ss_i, ss_k
  int a_shift, b_shift;
  void *C;
  long long c_row, c_col;       // elements between rows and columns; one of them is 1
  int c_bf16;
  int c_tma;                    // the tile leaves by TMA stores
  int tiles_m, tiles_n, num_k, group_m;
  int stages, stage_bytes;
  // how the work is shared between the CTAs (TilePieces, tc_common.cuh)
  int streamk, units, sk_first, sk_workers;
  float *ws;
  int *tile_count;
  Epilogue ep;                  // bias_kind in terms of the tiles' rows and columns
  int *err_flag;
};

constexpr int gb_epi_warps(int bn) { return bn >= 64 ? 8 : 4; }
constexpr int gb_max_stages(int bn) { return bn >= 128 ? 6 : 12; }
constexpr int gb_threads(int bn) { return 128 + 32 * gb_epi_warps(bn); }
constexpr int GB_OUT = 8192;   // bytes of a warp's buffer for the store: two boxes of 32 rows of 128 bytes

// acc += part * scale for two values at a time: the fp32 units take 64-bit operand pairs, and with one fused
// multiply-add for each value of each k-block they are as busy as the tensor core.
__device__ __forceinline__ void fma_pair(float &a0, float &a1, uint32_t p0, uint32_t p1, float s0, float s1) {
  asm("{\n\t"
      ".reg .b64 a, p, s;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 p, {%2, %3};\n\t"
      "mov.b64 s, {%4, %5};\n\t"
      "fma.rn.f32x2 a, p, s, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t"
      "}"
      : "+f"(a0), "+f"(a1)
      : "r"(p0), "r"(p1), "f"(s0), "f"(s1));
}
// acc += part * (row * col), the scales multiplied first.
__device__ __forceinline__ void scale_fma_pair(float &a0, float &a1, uint32_t p0, uint32_t p1, float row, float c0, float c1) {
  asm("{\n\t"
      ".reg .b64 a, p, s, r;\n\t"
      "mov.b64 a, {%0, %1};\n\t"
      "mov.b64 p, {%2, %3};\n\t"
      "mov.b64 r, {%4, %4};\n\t"
      "mov.b64 s, {%5, %6};\n\t"
      "mul.rn.f32x2 s, r, s;\n\t"
      "fma.rn.f32x2 a, p, s, a;\n\t"
      "mov.b64 {%0, %1}, a;\n\t"
      "}"
      : "+f"(a0), "+f"(a1)
      : "r"(p0), "r"(p1), "f"(row), "f"(c0), "f"(c1));
}

// Persistent: a CTA takes tiles of 128 x BN, k-block by k-block. Warps: 0 loads (TMA), 1 issues MMAs and owns tensor
// memory, 2 and 3 bring the scales of the k-blocks into shared memory, the others (8, or 4 where a tile is 32 columns or
// fewer) take each k-block's accumulator to registers, scaled, and store the tile at its end. A ring stage and an
// accumulator are one k-block each; there are at least as many stages as accumulators, so that one commit per
// k-block, on the stage's "done" barrier, serves the loader and the epilogue: that barrier's next phase cannot
// complete before the epilogue has let go of the accumulator that this one announced.
// PAIR: two CTAs of a cluster share a tile of 256 x 256. Each loads its own 128 rows of A and half of B's, the even one
// issues the MMAs for both (cta_group::2) and keeps their barriers, each scales and stores its own 128 rows.
// COLS: a scale for each of the tile's columns, else one for each 128. (An argument of the template, not of the launch:
// 4096 x 4096 x 8192 summed down columns 223 -> 210 us, the question after products out of range included.)
//
// What bounds it: the epilogue's way from one k-block to the next. Scales that change from block to block keep the tensor core
// from accumulating over k, so each 128 x 256 sums of a k-block are loaded from tensor memory and added once per 514 cycles
// of MMAs (4.27 PFLOP/s on their own). 8192^3 takes 555 us (2.0 PFLOP/s) in short bursts, 640 under the power limit: 0.63 us a k-block,
// some 1,200 cycles. Loads and additions on their own are 270 of them; without the additions the product takes 456 us,
// without the wait for the scales, which are long there, 499. So the k-block is a chain of waits (scales, MMAs, two loads, the
// arrival at the pair's even CTA), of which the parts that were measured do not make up the whole.
template <int BN, bool PAIR, bool COLS>
__global__ void __launch_bounds__(gb_threads(BN), 1)
    gemm_blocks_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ CUtensorMap tmC, const __grid_constant__ BlocksTcParams p) {
  ptx::grid_begin();
  constexpr int EPI_WARPS = gb_epi_warps(BN);
  constexpr int HALF = BN / (EPI_WARPS / 4);    // columns an epilogue warp takes
  constexpr int NBUF = BN == 256 ? 2 : 4;       // accumulators in tensor memory
  constexpr int CH = HALF >= 64 ? 64 : HALF;    // columns of the accumulator in registers at a time
  constexpr int RANKS = PAIR ? 2 : 1;
  constexpr int MAX_STAGES = gb_max_stages(BN);
  extern __shared__ __align__(1024) unsigned char gb_smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], done_bar[MAX_STAGES], acc_empty[NBUF];
  __shared__ __align__(8) uint64_t epi_bar;  // the epilogue warps meet here when a partial tile is handed over
  constexpr int SLOTS = 8, SLOT = GB_BM + BN;   // a ring of its own: scales of the tile's rows and columns, one slot per k-block
  __shared__ __align__(16) float s_scale[SLOTS][SLOT];
  __shared__ __align__(8) uint64_t scale_full[SLOTS], scale_empty[SLOTS];
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_fail, s_last;

  unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)gb_smem_raw + 1023) & ~(uintptr_t)1023);
  unsigned char *stage_out = smem + (size_t)p.stages * p.stage_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? ptx::cluster_ctarank() : 0u;  // 0: the CTA that issues the pair's MMAs
  const int stages = p.stages, worker = (int)blockIdx.x / RANKS, workers = (int)gridDim.x / RANKS;
  const int total_tiles = p.tiles_m * p.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&done_bar[s], 1);
    }
    for (int b = 0; b < NBUF; ++b) ptx::mbar_init(&acc_empty[b], EPI_WARPS * RANKS);
    for (int b = 0; b < SLOTS; ++b) {
      ptx::mbar_init(&scale_full[b], 64);
      ptx::mbar_init(&scale_empty[b], EPI_WARPS);
    }
    ptx::mbar_init(&epi_bar, EPI_WARPS);
    ptx::fence_mbar_init();
    s_fail = 0;
    s_last = 0;
  }
  if (warp == 1) {
    if (PAIR) {
      ptx::tmem_alloc_pair(&tmem_base_s, NBUF * BN);
      ptx::tmem_relinquish_pair();
    } else {
      ptx::tmem_alloc(&tmem_base_s, NBUF * BN);
      ptx::tmem_relinquish();
    }
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmA);
    ptx::prefetch_tmap(&tmB);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (PAIR) ptx::cluster_sync();  // the other CTA's barriers are initialised before anything reaches them
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  auto at_leader = [&](uint64_t *bar) { return ptx::map_to_rank(ptx::smem_addr(bar), 0u); };

  // m blocks are walked in groups so that the CTAs of one wave share columns of B and rows of A in L2
  auto decode = [&](int tile, int &mb, int &nb) {
    const int per_group = p.group_m * p.tiles_n;
    const int g = tile / per_group, first_m = g * p.group_m;
    const int gm = min(p.tiles_m - first_m, p.group_m), r = tile % per_group;
    mb = first_m + r % gm;
    nb = r / gm;
  };

  // 128 sums per thread and what is being added to them need more than an even share of the registers:
  // 128 x 40 + 256 x 232 = 384 x 168
  if (warp < 4) {
    if (BN == 256) ptx::setmaxnreg_dec<40>();
    // ---------------- loads ----------------
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      TilePieces pieces(p.streamk, p.units, p.num_k, total_tiles, worker, workers, p.sk_first, p.sk_workers);
      int tile, kb0, kb1;
      while (ok && pieces.next(tile, kb0, kb1)) {
        int mb, nb;
        decode(tile, mb, nb);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&done_bar[stage], phase ^ 1)) {
            ok = false;
            break;
          }
          unsigned char *sa = smem + (size_t)stage * p.stage_bytes, *sb = sa + GB_SLAB;
          const int k0 = kb * GB_BK;
          if (PAIR) {
            // the even CTA arms the stage for both CTAs' bytes; the odd one's may land first, which only drives the
            // pending count below zero for a moment
            if (rank == 0) ptx::mbar_arrive_expect_tx(&full_bar[stage], 2u * (uint32_t)p.stage_bytes);
            const uint32_t fb = at_leader(&full_bar[stage]);
            const int m0 = (mb * 2 + (int)rank) * GB_BM, n0 = nb * BN + (int)rank * (BN / 2);
            if (!p.a_mn) ptx::tma_load_3d_pair(sa, &tmA, k0, m0, 0, fb);
            else ptx::tma_load_3d_pair(sa, &tmA, m0, k0, 0, fb);
            if (!p.b_mn) ptx::tma_load_3d_pair(sb, &tmB, k0, n0, 0, fb);
            else ptx::tma_load_3d_pair(sb, &tmB, n0, k0, 0, fb);
            if (++stage == stages) {
              stage = 0;
              phase ^= 1;
            }
            continue;
          }
          ptx::mbar_arrive_expect_tx(&full_bar[stage], (uint32_t)p.stage_bytes);
          if (!p.a_mn) ptx::tma_load_3d(sa, &tmA, k0, mb * GB_BM, 0, &full_bar[stage]);
          else ptx::tma_load_3d(sa, &tmA, mb * GB_BM, k0, 0, &full_bar[stage]);
          if (!p.b_mn) {
            ptx::tma_load_3d(sb, &tmB, k0, nb * BN, 0, &full_bar[stage]);
          } else {
            // whole boxes of 128 columns, also for a narrower tile: the swizzle wants rows of 128 bytes
#pragma unroll
            for (int q = 0; q < (BN + 127) / 128; ++q)
              ptx::tma_load_3d(sb + q * GB_SLAB, &tmB, nb * BN + q * 128, k0, 0, &full_bar[stage]);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) s_fail = 1;
    }
    // ---------------- scales ----------------
    // Rows and columns beyond the matrix get a scale of the last one: they are not stored.
    if (warp >= 2) {
      const int t = threadIdx.x - 64;
      const bool row_each = p.a_shift == 0;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      TilePieces pieces(p.streamk, p.units, p.num_k, total_tiles, worker, workers, p.sk_first, p.sk_workers);
      int tile, kb0, kb1;
      while (ok && pieces.next(tile, kb0, kb1)) {
        int mb, nb;
        decode(tile, mb, nb);
        const int m0 = (mb * RANKS + (int)rank) * GB_BM, n0 = nb * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait_relaxed(&scale_empty[slot], phase ^ 1, 32)) {
            ok = false;
            break;
          }
          float *to = s_scale[slot];
          const float *a = p.a_scales + kb * p.as_k, *b = p.b_scales + kb * p.bs_k;
          if (row_each) {
#pragma unroll
            for (int i = 0; i < GB_BM; i += 64) ptx::copy_async_4(to + i + t, a + (long long)min(m0 + i + t, p.M - 1) * p.as_i);
          } else if (t == 0) {
            ptx::copy_async_4(to, a + (long long)(min(m0, p.M - 1) >> 7) * p.as_i);
          }
          to += GB_BM;
          if (COLS) {
#pragma unroll
            for (int i = 0; i < BN; i += 64)
              if (i + t < BN) ptx::copy_async_4(to + i + t, b + (long long)min(n0 + i + t, p.N - 1) * p.bs_i);
          } else if (t * 128 < BN) {
            ptx::copy_async_4(to + t, b + (long long)(min(n0 + t * 128, p.N - 1) >> 7) * p.bs_i);
          }
          ptx::copy_async_arrive(&scale_full[slot]);
          if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      ptx::copy_async_wait_all();
      if (!ok) s_fail = 1;
    }
    // ---------------- MMAs (of a pair: the even CTA's only) ----------------
    if (warp == 1 && rank == 0) {  // all lanes, see kblock_f8
      // a k-slice is 32 bytes of a K-major row, or 32 rows of 128 bytes of an MN-major block
      const uint64_t a_step = (p.a_mn ? 32 * 128 : 32) >> 4, b_step = (p.b_mn ? 32 * 128 : 32) >> 4;
      const uint32_t st0 = ptx::smem_addr(smem), stage_step = (uint32_t)p.stage_bytes >> 4;
      const uint64_t a_desc0 = make_smem_desc(st0, p.a_mn ? GB_SLAB : 16, 1024, 2);
      const uint64_t b_desc0 = make_smem_desc(st0 + GB_SLAB, p.b_mn ? GB_SLAB : 16, 1024, 2);
      const uint32_t done0 = ptx::smem_addr(&done_bar[0]), lead = lane == 0 ? 1u : 0u;
      // how many k-blocks this CTA takes in all: which tiles they belong to is no concern of this thread
      int blocks = 0, tile, kb0, kb1;
      TilePieces pieces(p.streamk, p.units, p.num_k, total_tiles, worker, workers, p.sk_first, p.sk_workers);
      while (pieces.next(tile, kb0, kb1)) blocks += kb1 - kb0;
      int stage = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 1, soff = 0;
      bool ok = true, full = false, empty = false;  // polled ahead: the next stage is there, the next accumulator is free
      for (; blocks > 0; --blocks) {
        if (!__all_sync(0xffffffffu, empty)) ok = __all_sync(0xffffffffu, ptx::mbar_wait(&acc_empty[buf], acc_phase));
        if (ok && !__all_sync(0xffffffffu, full)) ok = __all_sync(0xffffffffu, ptx::mbar_wait(&full_bar[stage], phase));
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint64_t off = soff;
        const uint32_t d = tmem_base + (uint32_t)(buf * BN), done = done0 + (uint32_t)stage * 8u;
        soff += stage_step;
        if (++stage == stages) {
          stage = 0;
          soff = 0;
          phase ^= 1;
        }
        if (++buf == NBUF) {
          buf = 0;
          acc_phase ^= 1;
        }
        full = ptx::mbar_test_wait(&full_bar[stage], phase);
        ptx::kblock_f8<PAIR>(lead, d, a_desc0 + off, b_desc0 + off, a_step, b_step, p.idesc, done);
        empty = ptx::mbar_test_wait(&acc_empty[buf], acc_phase);
      }
      if (!ok) s_fail = 1;
    }
  } else {
    if (BN == 256) ptx::setmaxnreg_inc<232>();
    // ---------------- scaling, sums and stores ----------------
    const int ew = warp - 4;
    const int quarter = warp & 3;        // the TMEM lanes this warp may read: 32*quarter .. +31
    const int ch0 = (ew >> 2) * HALF;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)ch0;
    const uint32_t acc_empty0 = at_leader(&acc_empty[0]);
    int stage = 0, buf = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0, epi_phase = 0;
    // Whether some product of a scale of the warp's rows and one of its columns is out of range: the rows' times the least and
    // the greatest magnitude of the columns', zeros apart.
    auto any_far = [&](float row, const float *cols) -> bool {
      float least = 3.40282347e38f, most = 0.f;
      for (int j = lane; j < (COLS ? HALF : 1); j += 32) {
        const float c = fabsf(cols[j]);
        if (c != 0.f) least = fminf(least, c);
        most = fmaxf(most, c);
      }
      least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      return __any_sync(0xffffffffu, row != 0.f && most != 0.f && !(in_range(__fmul_rn(row, least)) && in_range(__fmul_rn(row, most))));
    };
    bool ok = true;
    auto epi_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&epi_bar);
      const bool done = ptx::mbar_wait_relaxed(&epi_bar, epi_phase, 32);
      epi_phase ^= 1;
      return done;
    };
    TilePieces pieces(p.streamk, p.units, p.num_k, total_tiles, worker, workers, p.sk_first, p.sk_workers);
    int tile, kb0, kb1;
    while (ok && pieces.next(tile, kb0, kb1)) {
      int mb, nb;
      decode(tile, mb, nb);
      const int m = (mb * RANKS + (int)rank) * GB_BM + quarter * 32 + lane, n0 = nb * BN + ch0;
      const int row_at = p.a_shift == 0 ? quarter * 32 + lane : 0, col_at = GB_BM + (COLS ? ch0 : ch0 >> 7);
      float acc[HALF];
#pragma unroll
      for (int j = 0; j < HALF; ++j) acc[j] = 0.f;
      // An accumulator is taken in pieces of CH columns: the fewer waits for tensor memory, the better (8192^3 with
      // 32 columns a piece 587 us, with 64 551).
      uint32_t r[CH];
      auto load = [&](int c) {
        const uint32_t at = lane_addr + (uint32_t)(buf * BN + c);
        if constexpr (CH == 16) {
          ptx::tmem_ld_32x16(at, r);
        } else {
#pragma unroll
          for (int q = 0; q < CH; q += 32) ptx::tmem_ld_32x32(at + (uint32_t)q, *reinterpret_cast<uint32_t(*)[32]>(&r[q]));
        }
      };
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!ptx::mbar_wait(&scale_full[slot], slot_phase)) ok = false;  // long there
        const float *cols = s_scale[slot] + col_at;
        const float row = s_scale[slot][row_at], both = __fmul_rn(row, *cols);
        if (!ok || !ptx::mbar_wait(&done_bar[stage], phase)) {
          ok = false;
          break;
        }
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
        __syncwarp();
        ptx::tc_fence_after_sync();
        auto take = [&](bool last) {  // what was loaded is in registers; after the last piece the accumulator is free
          ptx::tmem_ld_wait();
          if (last) {
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) ptx::mbar_arrive_cluster_tmem(acc_empty0 + (uint32_t)buf * 8u);
              else ptx::mbar_arrive(&acc_empty[buf]);
            }
          }
        };
        load(0);
        // Seldom: scales whose product is out of range, or may be. (Asked without a branch while the first piece is on its way:
        // a k-block of the epilogue is one chain of waits, and 100 cycles in front of it are 9 % of 512 x 4096 x 4096.)
        bool odd;
        if constexpr (COLS) {
          // every scale in [2^-63, 2^63), a column or more to a lane: then the product of any two is in range
          auto away = [](float v) { return (__float_as_uint(v) << 1) - (64u << 24); };
          uint32_t most = away(row);
          if constexpr (HALF <= 32) {
            most = max(most, away(cols[lane & (HALF - 1)]));
          } else if constexpr (HALF == 64) {
            const float2 v = *reinterpret_cast<const float2 *>(cols + 2 * lane);
            most = max(most, max(away(v.x), away(v.y)));
          } else {
            const float4 v = *reinterpret_cast<const float4 *>(cols + 4 * lane);
            most = max(max(most, away(v.x)), max(away(v.y), max(away(v.z), away(v.w))));
          }
          odd = most >= (126u << 24);
        } else {
          odd = !in_range(both);
        }
        odd = __any_sync(0xffffffffu, odd);
        take(CH == HALF);
        if constexpr (COLS) {
          auto add_block = [&](auto careful) {
#pragma unroll
            for (int c = 0; c < HALF; c += CH) {
              if (c > 0) {
                load(c);
                take(c + CH == HALF);
              }
              if constexpr (decltype(careful)::value) {
#pragma unroll
                for (int j = 0; j < CH; ++j) acc[c + j] = Scaling(row, cols[c + j]).add(acc[c + j], __uint_as_float(r[j]));
              } else {
#pragma unroll
                for (int j = 0; j < CH; j += 4) {
                  const float4 s = *reinterpret_cast<const float4 *>(cols + c + j);
                  scale_fma_pair(acc[c + j], acc[c + j + 1], r[j], r[j + 1], row, s.x, s.y);
                  scale_fma_pair(acc[c + j + 2], acc[c + j + 3], r[j + 2], r[j + 3], row, s.z, s.w);
                }
              }
            }
          };
          if (__builtin_expect(odd, 0) && any_far(row, cols)) add_block(std::true_type());
          else add_block(std::false_type());
        } else {
          // (two forms of the sums, as above, made the compiler move them about: 8192^3 615 us instead of 564)
          float last = both;
#pragma unroll
          for (int c = 0; c < HALF; c += CH) {
            if (c > 0) {
              load(c);
              take(c + CH == HALF);
            }
            if (__builtin_expect(odd, 0)) {
              const Scaling by(s_scale[slot][row_at], s_scale[slot][col_at]);
              last = by.last;
#pragma unroll
              for (int j = 0; j < CH; ++j) r[j] = __float_as_uint(by.near(__uint_as_float(r[j])));
            }
#pragma unroll
            for (int j = 0; j < CH; j += 2) fma_pair(acc[c + j], acc[c + j + 1], r[j], r[j + 1], last, last);
          }
        }
        if (++buf == NBUF) buf = 0;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&scale_empty[slot]);
        if (++slot == SLOTS) {
          slot = 0;
          slot_phase ^= 1;
        }
      }
      if (kb0 != 0 || kb1 != p.num_k) {
        // part of a tile: leave it in the workspace; the CTA that delivers the last part finishes the tile
        const int tile_u0 = (tile - p.sk_first) * p.num_k;
        const size_t slot_floats = (size_t)GB_BM * BN * RANKS;
        const size_t within = (size_t)rank * GB_BM * BN + (size_t)ew * HALF * 32 + lane;
        if (ok) {
          float *wsp = p.ws + (size_t)share_slot(worker, tile_u0, p.units, p.sk_workers) * slot_floats + within;
#pragma unroll
          for (int j = 0; j < HALF; ++j) __stcg(wsp + j * 32, acc[j]);
        } else {
          s_fail = 1;
        }
        __threadfence();
        const int c_first = share_of_unit(tile_u0, p.units, p.sk_workers);
        const int c_last = share_of_unit(tile_u0 + p.num_k - 1, p.units, p.sk_workers);
        bool met = epi_sync();
        if (ew == 0 && lane == 0) {  // each CTA of a pair counts for its own rows
          int *count = p.tile_count + (tile - p.sk_first) * RANKS + (int)rank;
          s_last = atomicAdd(count, 1) == c_last - c_first ? 1 : 0;
          if (s_last) *count = 0;  // zero again for the next launch
        }
        met = epi_sync() && met;
        if (!met || *(volatile int *)&s_fail) {
          ok = false;
          break;
        }
        if (!*(volatile int *)&s_last) continue;
        __threadfence();
#pragma unroll
        for (int j = 0; j < HALF; ++j) acc[j] = 0.f;
        // k order: CTA c's share precedes CTA c + 1's. A part is a latency of about a microsecond: on narrow tiles
        // several are on their way at once
        constexpr int PF = HALF <= 16 ? 8 : (HALF <= 32 ? 2 : 1);
        for (int c = c_first; c <= c_last; c += PF) {
          if constexpr (PF > 1) {
            float in[PF][HALF];
#pragma unroll
            for (int q = 0; q < PF; ++q) {
              const float *src = p.ws + (size_t)share_slot(min(c + q, c_last), tile_u0, p.units, p.sk_workers) * slot_floats + within;
#pragma unroll
              for (int j = 0; j < HALF; ++j) in[q][j] = __ldcg(src + j * 32);
            }
#pragma unroll
            for (int q = 0; q < PF; ++q) {
              if (c + q <= c_last) {
#pragma unroll
                for (int j = 0; j < HALF; ++j) acc[j] = __fadd_rn(acc[j], in[q][j]);
              }
            }
          } else {
            const float *src = p.ws + (size_t)share_slot(c, tile_u0, p.units, p.sk_workers) * slot_floats + within;
#pragma unroll
            for (int j = 0; j < HALF; ++j) acc[j] = __fadd_rn(acc[j], ptx::ld_cg_ordered(src + j * 32));
          }
        }
      }
      if (!ok) break;
      const int mw = m - lane;  // the warp's first row
      if (mw >= p.M || n0 >= p.N) continue;
      const int valid = min(HALF, p.N - n0);
      const float *bias = reinterpret_cast<const float *>(p.ep.bias);
      if (p.ep.bias_kind == B200_BIAS_COL) {
#pragma unroll
        for (int j = 0; j < HALF; ++j)
          if (j < valid) acc[j] = __fadd_rn(acc[j], __ldg(bias + n0 + j));
      } else if (p.ep.bias_kind == B200_BIAS_ROW) {
        const float bm = __ldg(bias + min(m, p.M - 1));
#pragma unroll
        for (int j = 0; j < HALF; ++j) acc[j] = __fadd_rn(acc[j], bm);
      }
      const float alpha = (float)p.ep.alpha;
      if (p.ep.act == B200_ACT_RECTIFY) {
#pragma unroll
        for (int j = 0; j < HALF; ++j) acc[j] = apply_act<float>(acc[j], B200_ACT_RECTIFY, alpha);
      } else if (p.ep.act == B200_ACT_LEAKY) {
#pragma unroll
        for (int j = 0; j < HALF; ++j) acc[j] = apply_act<float>(acc[j], B200_ACT_LEAKY, alpha);
      }
      if (p.c_row == 1) {
        // swapped: the lanes hold neighbours already
        if (m < p.M) {
          const long long at = (long long)n0 * p.c_col + m;
#pragma unroll
          for (int j = 0; j < HALF; ++j) {
            if (j < valid) {
              const long long x = at + j * p.c_col;
              if (p.c_bf16) reinterpret_cast<__nv_bfloat16 *>(p.C)[x] = __float2bfloat16_rn(acc[j]);
              else {
                float *f = reinterpret_cast<float *>(p.C) + x;
                *f = p.ep.accumulate ? __fadd_rn(*f, acc[j]) : acc[j];
              }
            }
          }
        }
      } else {
        if (HALF >= 32 && p.c_tma) {
          // A lane holds a row. The warp's part of the tile goes to shared memory, boxes of 32 rows of 128 bytes in the
          // 128-byte swizzle, and from there by TMA stores that drain while the next tile is multiplied: all SMs
          // come to the end of their tiles together, and stores that were waited for held the accumulators up.
          const int per = p.c_bf16 ? 64 : 32;
          unsigned char *out = stage_out + ew * GB_OUT;
          const int sw = lane & 7;
          auto send = [&](int c, int boxes) {  // columns c .. of the warp's, in boxes from `out` on
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              for (int i = 0; i < boxes && c + i * per < valid; ++i)
                ptx::tma_store_3d(&tmC, out + i * 4096, n0 + c + i * per, mw, 0);
              ptx::bulk_commit();
            }
          };
          auto reuse = [&]() {  // what was sent before has been read
            if (lane == 0) ptx::bulk_wait_read<0>();
            __syncwarp();
          };
          if (HALF >= 64 && p.c_bf16) {
            reuse();
#pragma unroll
            for (int j = 0; j < HALF; j += 8) {
              uint4 w;
              uint32_t *ww = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(acc[j + 2 * t], acc[j + 2 * t + 1]);
                ww[t] = *reinterpret_cast<const uint32_t *>(&h);
              }
              *reinterpret_cast<uint4 *>(out + (j / 64) * 4096 + lane * 128 + ((((j % 64) / 8) ^ sw) << 4)) = w;
            }
            send(0, (HALF + 63) / 64);
          } else {
#pragma unroll
            for (int c = 0; c < HALF; c += 64) {
              reuse();
#pragma unroll
              for (int j = c; j < c + 64 && j < HALF; j += 4)
                *reinterpret_cast<float4 *>(out + ((j - c) / 32) * 4096 + lane * 128 + ((((j % 32) / 4) ^ sw) << 4)) =
                    make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
              send(c, 2);
            }
          }
        } else {
          // Anything else (rows that do not start on 16-byte boundaries, results that are added) goes through shared
          // memory too, 32 columns at a time, and leaves row by row: from the lanes' registers an instruction would
          // touch 32 rows (1000 x 625 x 1152 float32 16.1 -> 13.2 us).
          constexpr int W = HALF < 32 ? HALF : 32, PITCH = W + 1;
          float *out = reinterpret_cast<float *>(stage_out + ew * GB_OUT);
#pragma unroll
          for (int c = 0; c < HALF; c += W) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < W; ++j) out[lane * PITCH + j] = acc[c + j];
            __syncwarp();
            const int j = lane % W, rows = min(32, p.M - mw);
            if (c + j < valid) {
              const long long first = (long long)mw * p.c_row + n0 + c + j;
#pragma unroll 8
              for (int r = lane / W; r < rows; r += 32 / W) {
                const float v = out[r * PITCH + j];
                const long long x = first + r * p.c_row;
                if (p.c_bf16) {
                  reinterpret_cast<__nv_bfloat16 *>(p.C)[x] = __float2bfloat16_rn(v);
                } else {  // Incr mode: the rounded result is added to what C holds
                  float *f = reinterpret_cast<float *>(p.C) + x;
                  *f = p.ep.accumulate ? __fadd_rn(*f, v) : v;
                }
              }
            }
          }
        }
      }
    }
    if (!ok) s_fail = 1;
    if (lane == 0) ptx::bulk_wait<0>();  // what was sent has been written
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  // neither CTA of a pair leaves, or gives its tensor memory back, while the other may still read its shared memory
  // or arrive on its barriers (every wait above is bounded, so both get here)
  if (PAIR) ptx::cluster_sync();
  if (threadIdx.x == 0 && s_fail) atomicExch(p.err_flag, 1);
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    if (PAIR) ptx::tmem_dealloc_pair(tmem_base, NBUF * BN);
    else ptx::tmem_dealloc(tmem_base, NBUF * BN);
  }
}

// Rows of bytes to a pitch that the TMA unit takes: both operands in one launch (rows of the second follow those of
// the first), 16 bytes of the copy per thread and step.
struct RepackJob {
  const uint8_t *src;
  uint8_t *dst;
  long long rows, cols, ld, ldo;  // ldo a multiple of 16
};
__global__ void __launch_bounds__(256) repack_kernel(const RepackJob j0, const RepackJob j1) {
  ptx::grid_begin();
  const long long n0 = j0.rows * (j0.ldo / 16), n = n0 + j1.rows * (j1.ldo / 16);
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    const RepackJob &j = i < n0 ? j0 : j1;
    const long long w = i < n0 ? i : i - n0, per = j.ldo / 16, r = w / per, c = (w - r * per) * 16;
    const uint8_t *s = j.src + r * j.ld + c;
    union {
      uint8_t b[16];
      uint4 v;
    } o;
    if (c >= 4 && c + 20 <= j.cols) {
      // five aligned words around the sixteen bytes, all of them inside the row (4095^3: 134 -> 126 us)
      const uint32_t *w4 = reinterpret_cast<const uint32_t *>((uintptr_t)s & ~(uintptr_t)3);
      const unsigned by = ((unsigned)(uintptr_t)s & 3u) * 8u;
      uint32_t in[5];
#pragma unroll
      for (int t = 0; t < 5; ++t) in[t] = t < 4 || by ? __ldg(w4 + t) : 0u;
      o.v = make_uint4(__funnelshift_r(in[0], in[1], by), __funnelshift_r(in[1], in[2], by), __funnelshift_r(in[2], in[3], by),
                       __funnelshift_r(in[3], in[4], by));
    } else {
#pragma unroll
      for (int t = 0; t < 16; ++t) o.b[t] = c + t < j.cols ? s[t] : 0;
    }
    *reinterpret_cast<uint4 *>(j.dst + r * j.ldo + c) = o.v;
  }
}

// grid: CTAs; pairs launch as clusters of two.
template <int BN, bool PAIR, bool COLS>
static int launch_blocks_tc_as(b200_engine *e, const CUtensorMap *tm, const BlocksTcParams &p, int grid) {
  auto kern = gemm_blocks_tc_kernel<BN, PAIR, COLS>;
  const size_t smem = (size_t)p.stages * p.stage_bytes + (p.c_row != 1 ? gb_epi_warps(BN) * GB_OUT : 0) + 1024;
  static std::atomic<int> attr_dev_mask{0};
  if (!(attr_dev_mask & (1 << (e->device & 31)))) {
    cudaFuncAttributes fa;
    B200_CHECK_CUDA(e, cudaFuncGetAttributes(&fa, kern));
    // what the widest tiles' warpgroups ask for has to be there, or they would wait for it for good
    if (BN == 256 && fa.numRegs * gb_threads(BN) < 128 * 40 + 256 * 232)
      return set_error(e, B200_ERR_CUDA, "gemm_blocks_tc_kernel was built with %d registers per thread", fa.numRegs);
    const size_t optin = std::min<size_t>(e->smem_optin, 227 * 1024);
    B200_CHECK_CUDA(e, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(optin - fa.sharedSizeBytes)));
    attr_dev_mask |= 1 << (e->device & 31);
  }
  if (PAIR) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_kernel does
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(gb_threads(BN));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = e->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    B200_CHECK_CUDA(e, cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], tm[2], p));
  } else {
    launch_kernel(e, kern, grid, gb_threads(BN), smem, tm[0], tm[1], tm[2], p);
  }
  B200_CHECK_LAUNCH(e, "gemm_blocks_tc_kernel");
  e->flags_dirty = true;
  return B200_OK;
}

template <int BN, bool PAIR = false>
static int launch_blocks_tc(b200_engine *e, const CUtensorMap *tm, const BlocksTcParams &p, int grid) {
  return p.b_shift == 0 ? launch_blocks_tc_as<BN, PAIR, true>(e, tm, p, grid) : launch_blocks_tc_as<BN, PAIR, false>(e, tm, p, grid);
}

// One operand in the form that the TMA unit reads: rows x cols bytes as stored, pitch a multiple of 16.
struct StoredOperand {
  const uint8_t *data;
  long long rows, cols, ld;
};

static int gemm_blocks_tc(b200_engine *e, StoredOperand sa, StoredOperand sb, BlockOperand a, BlockOperand b, bool a_mn,
                          bool b_mn, const BlocksParams &q) {
  long long M = q.M, N = q.N;
  // Few rows: the tile's 128 rows are the weights' then, and its columns the rows of A, 16 at least
  const bool swap = M <= 64 && N > M;
  Epilogue ep = q.ep;
  if (swap) {
    std::swap(M, N);
    std::swap(sa, sb);
    std::swap(a, b);
    std::swap(a_mn, b_mn);
    if (ep.bias_kind != B200_BIAS_NONE) ep.bias_kind = ep.bias_kind == B200_BIAS_COL ? B200_BIAS_ROW : B200_BIAS_COL;
  }
  BlocksTcParams p;
  memset((void *)&p, 0, sizeof p);
  p.M = (int)M;
  p.N = (int)N;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.a_scales = a.scales;
  p.as_i = a.ss_i;
  p.as_k = a.ss_k;
  p.a_shift = a.shift;
  p.b_scales = b.scales;
  p.bs_i = b.ss_i;
  p.bs_k = b.ss_k;
  p.b_shift = b.shift;
  p.C = q.C;
  p.c_row = swap ? 1 : q.ldc;
  p.c_col = swap ? q.ldc : 1;
  p.c_bf16 = q.c_bf16;
  p.ep = ep;
  p.err_flag = e->d_flags + 2;
  p.num_k = (int)((q.K + GB_BK - 1) / GB_BK);
  p.tiles_m = (int)((M + GB_BM - 1) / GB_BM);
  // Tile width. A k-block costs a CTA about as much on 64 columns as on 128 (four instructions and a commit take 514
  // cycles to issue, whatever their width), a pair of CTAs on 256 x 256 one and a half times that: the width is the one
  // whose rounds of tiles take least, the widest of equals. (The widest that gives every SM a tile, which
  // bf16 products take, made 512 x 4096 x 4096 in two rounds of 64 columns, 32 us, and 1024 x 4096 x 4096 in two of 128, 34.)
  const bool may_pair = !(e->flags & B200_ENGINE_NO_PAIRS), may_share = !(e->flags & B200_ENGINE_NO_STREAMK);
  auto tiles_of = [&](int width) {
    const long long rows = width == 256 && may_pair ? 256 : 128;
    return (M + rows - 1) / rows * ((N + width - 1) / width);
  };
  auto cost = [&](int width) {  // us
    const bool paired = width == 256 && may_pair;
    const long long workers = paired ? e->sm_count / 2 : e->sm_count, tiles = tiles_of(width);
    const double block = width == 256 ? 0.62 : (width == 128 ? 0.42 : 0.39);
    const double whole = (double)((tiles + workers - 1) / workers) * p.num_k * block;
    if (!may_share || tiles >= workers) return whole;
    const long long shares = std::min(workers, (3 * tiles >= workers ? 2 : 4) * tiles);
    return std::min(whole, (double)(tiles * p.num_k) / shares * block + 4.0);
  };
  int bn = 256;
  for (int width : {128, 64})
    if (cost(width) < cost(bn) || bn / 2 >= N) bn = width;
  while (bn > 16 && bn / 2 >= N) bn /= 2;
  p.c_tma = !swap && (uintptr_t)q.C % 16 == 0 && q.ldc % (q.c_bf16 ? 8 : 4) == 0 && !ep.accumulate &&
            bn >= (q.c_bf16 ? 128 : 64);  // a warp's columns fill a box of 128 bytes
  p.tiles_n = (int)((N + bn - 1) / bn);
  const bool pair = may_pair && bn == 256;  // the widest tiles are shared by pairs of CTAs
  if (pair) p.tiles_m = (p.tiles_m + 1) / 2;
  const int ranks = pair ? 2 : 1, max_workers = e->sm_count / ranks;
  const long long total_tiles = (long long)p.tiles_m * p.tiles_n;
  if (total_tiles >= (1LL << 31))
    return set_error(e, B200_ERR_UNSUPPORTED, "b200_gemm_blocks: %lld output tiles are more than one launch takes", total_tiles);
  p.group_m = std::min(p.tiles_m, 8 / ranks);
  p.stage_bytes = GB_SLAB + (b_mn ? std::max(bn / ranks, 128) : bn / ranks) * 128;
  const int budget = (int)std::min<size_t>(e->smem_optin, 227 * 1024) - 1024 - 14 * 1024 -
                     (p.c_row != 1 ? gb_epi_warps(bn) * GB_OUT : 0);  // alignment, static part, the stores' buffers
  p.stages = std::min(gb_max_stages(bn), budget / p.stage_bytes);
  p.idesc = make_idesc(0, a_mn, b_mn, GB_BM * ranks, bn) | ((uint32_t)a.e5m2 << 7) | ((uint32_t)b.e5m2 << 10);

  // operands that the TMA unit cannot read in place
  void *blk[2] = {nullptr, nullptr};
  RepackJob jobs[2];
  StoredOperand *ops[2] = {&sa, &sb};
  int rc = B200_OK;
  for (int i = 0; i < 2; ++i) {
    RepackJob &j = jobs[i];
    j = RepackJob{nullptr, nullptr, 0, 0, 0, 16};
    StoredOperand &o = *ops[i];
    if ((uintptr_t)o.data % 16 == 0 && o.ld % 16 == 0) continue;
    const long long ldo = (o.cols + 15) / 16 * 16;
    rc = b200_get(e, o.rows * ldo, &blk[i]);
    if (rc != B200_OK) break;
    j = RepackJob{o.data, (uint8_t *)blk[i], o.rows, o.cols, o.ld, ldo};
    o.data = (const uint8_t *)blk[i];
    o.ld = ldo;
  }
  if (rc == B200_OK && (blk[0] || blk[1])) {
    const long long n = (jobs[0].rows * jobs[0].ldo + jobs[1].rows * jobs[1].ldo) / 16;
    launch_kernel(e, repack_kernel, (unsigned)std::max<long long>(1, std::min<long long>((n + 255) / 256, e->sm_count * 16)), 256, 0,
                  jobs[0], jobs[1]);
    if (cudaGetLastError() != cudaSuccess) rc = set_error(e, B200_ERR_CUDA, "launch of repack_kernel failed");
    else e->launches++;
  }
  CUtensorMap tm[3];
  if (rc == B200_OK) rc = encode_map(e, &tm[0], 1, sa.data, sa.cols, sa.rows, 1, sa.ld, 0, 128, 128, false);
  if (rc == B200_OK) rc = encode_map(e, &tm[1], 1, sb.data, sb.cols, sb.rows, 1, sb.ld, 0, 128, b_mn ? 128 : bn / ranks, false);
  tm[2] = tm[1];
  if (rc == B200_OK && p.c_tma)
    rc = encode_map(e, &tm[2], q.c_bf16 ? 2 : 4, q.C, N, M, 1, q.ldc, 0, q.c_bf16 ? 64 : 32, 32, false);
  int workers = (int)std::min<long long>(total_tiles, max_workers);
  p.sk_workers = workers;
  void *ws = nullptr;
  if (rc == B200_OK && may_share) {
    // whole tiles per CTA would leave SMs idle: share out the k range instead (TilePieces)
    // (Where two parts of each tile occupy most SMs, no tile is cut into more: 64 x 8192 x 4096, 64 tiles, in up to four
    // parts 22 us, in two 18; 64 x 4096 x 4096, 32 tiles, 15.1 and 16.9.)
    int shares = workers, first = 0;
    const int most = 3 * total_tiles >= max_workers ? (int)std::min<long long>(max_workers, 2 * total_tiles) : max_workers;
    if (total_tiles <= b200_engine::kSkCounters / 2 && streamk_pays(total_tiles, p.num_k, max_workers, &shares)) {
      shares = std::min(shares, most);
      if (b200_get(e, 2LL * shares * ranks * GB_BM * bn * 4, &ws) == B200_OK) {
        p.streamk = 1;
        p.units = (int)(total_tiles * p.num_k);
        workers = p.sk_workers = shares;
      }
    } else if (streamk_tail_pays(total_tiles, p.num_k, max_workers, &first, &shares)) {
      if (b200_get(e, 2LL * shares * ranks * GB_BM * bn * 4, &ws) == B200_OK) {
        p.streamk = 1;
        p.sk_first = first;
        p.sk_workers = shares;
        p.units = (int)((total_tiles - first) * p.num_k);
      }
    }
    p.tile_count = e->sk_counters;
    p.ws = (float *)ws;
  }
  if (rc == B200_OK) {
    switch (bn) {
      case 256: rc = pair ? launch_blocks_tc<256, true>(e, tm, p, 2 * workers) : launch_blocks_tc<256>(e, tm, p, workers); break;
      case 128: rc = launch_blocks_tc<128>(e, tm, p, workers); break;
      case 64: rc = launch_blocks_tc<64>(e, tm, p, workers); break;
      case 32: rc = launch_blocks_tc<32>(e, tm, p, workers); break;
      default: rc = launch_blocks_tc<16>(e, tm, p, workers); break;
    }
  }
  // stream order makes handing the scratch back safe: later users run after this kernel
  for (void *s : {blk[0], blk[1], ws})
    if (s) b200_put(e, s, 0);
  return rc;
}

template <int NT>
static void launch_skinny(b200_engine *e, const BlockOperand &w, const BlockOperand &x, const BlocksParams &p) {
  auto kern = w.e5m2 ? (x.e5m2 ? gemm_blocks_skinny_kernel<NT, true, true> : gemm_blocks_skinny_kernel<NT, true, false>)
                     : (x.e5m2 ? gemm_blocks_skinny_kernel<NT, false, true> : gemm_blocks_skinny_kernel<NT, false, false>);
  launch_kernel(e, kern, (unsigned)((p.N + 15) / 16), 256, 0, w, x, p);
}

static BlockOperand block_operand(const void *data, int type, int block, bool k_contiguous, long long ld, const float *scales,
                                  long long i_extent, long long k_extent) {
  BlockOperand o;
  o.data = (const uint8_t *)data;
  o.si = k_contiguous ? ld : 1;
  o.sk = k_contiguous ? 1 : ld;
  o.scales = scales;
  o.shift = block == B200_BLOCK_TILE ? 7 : 0;
  const long long nk = (k_extent + 127) / 128, ni = o.shift ? (i_extent + 127) / 128 : i_extent;
  o.ss_i = k_contiguous ? nk : 1;
  o.ss_k = k_contiguous ? 1 : ni;
  o.e5m2 = type == B200_E5M2;
  return o;
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_gemm_blocks(b200_engine *e, int ctype, int transA, int transB, int64_t M, int64_t N, int64_t K, const void *A,
                     int a_type, int a_block, int64_t lda, const float *a_scales, const void *B, int b_type, int b_block,
                     int64_t ldb, const float *b_scales, void *C, int64_t ldc, const b200_epilogue *epi) {
  if (!e) return B200_ERR_INVALID;
  std::lock_guard<std::recursive_mutex> lk(e->mu);
  B200_REQUIRE(e, ctype == B200_F32 || ctype == B200_BF16, "b200_gemm_blocks: dtype %d not supported for C", ctype);
  B200_REQUIRE(e, (a_type == B200_E4M3 || a_type == B200_E5M2) && (b_type == B200_E4M3 || b_type == B200_E5M2),
               "b200_gemm_blocks: an operand's dtype (%d, %d) is no 8-bit one", a_type, b_type);
  B200_REQUIRE(e, a_block == B200_BLOCK_TILE || a_block == (transA ? B200_BLOCK_COL : B200_BLOCK_ROW),
               "b200_gemm_blocks: A's blocks (%d) do not lie along k", a_block);
  B200_REQUIRE(e, b_block == B200_BLOCK_TILE || b_block == (transB ? B200_BLOCK_ROW : B200_BLOCK_COL),
               "b200_gemm_blocks: B's blocks (%d) do not lie along k", b_block);
  B200_REQUIRE(e, M >= 0 && N >= 0 && K >= 0, "b200_gemm_blocks: negative extent");
  B200_REQUIRE(e, M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31), "b200_gemm_blocks: an extent is 2^31 or more");
  if (M == 0 || N == 0) return B200_OK;
  B200_REQUIRE(e, C != nullptr, "b200_gemm_blocks: C is null");
  B200_REQUIRE(e, lda >= (transA ? M : K) && ldb >= (transB ? K : N) && ldc >= N,
               "b200_gemm_blocks: leading dimension too small (%lld %lld %lld)", (long long)lda, (long long)ldb, (long long)ldc);
  B200_REQUIRE(e, K == 0 || (A && B && a_scales && b_scales), "b200_gemm_blocks: null operand");
  B200_REQUIRE(e, (uintptr_t)C % dtype_size(ctype) == 0 && ((uintptr_t)a_scales | (uintptr_t)b_scales) % 4 == 0,
               "b200_gemm_blocks: a pointer is not aligned to its type");
  if (epi) {
    B200_REQUIRE(e, epi->bias_kind >= 0 && epi->bias_kind <= 2 && epi->act >= 0 && epi->act <= 2,
                 "b200_gemm_blocks: bad epilogue");
    B200_REQUIRE(e, epi->bias_kind == 0 || (epi->bias != nullptr && (uintptr_t)epi->bias % 4 == 0),
                 "b200_gemm_blocks: bias is null or not aligned");
    B200_REQUIRE(e, !epi->accumulate || ctype == B200_F32, "b200_gemm_blocks: only a float32 C can be added to");
  }
  DeviceGuard g(e);
  int rc = flush_pending(e);
  if (rc != B200_OK) return rc;
  const BlockOperand a = block_operand(A, a_type, a_block, !transA, lda, a_scales, M, K);
  const BlockOperand b = block_operand(B, b_type, b_block, transB, ldb, b_scales, N, K);
  BlocksParams p;
  p.M = M;
  p.N = N;
  p.K = K;
  p.C = C;
  p.ldc = ldc;
  p.c_bf16 = ctype == B200_BF16;
  p.ep = make_epilogue(epi);
  if (K > 0) {
    const StoredOperand sa{(const uint8_t *)A, transA ? K : M, transA ? M : K, lda};
    const StoredOperand sb{(const uint8_t *)B, transB ? N : K, transB ? K : N, ldb};
    // Few rows, k contiguous and 16-byte loads possible: the kernel for these, as long as B is not so large that the tensor
    // cores' longer way is hidden behind its reading. us in a row of calls, this kernel / the other: 1 x 4096 x 4096 5.4 / 11.5,
    // 8 x 8192 x 4096 8.7 / 14.8, 1 x 4096 x 16384 13.7 / 21.6, 8 x 16384 x 8192 34.8 / 28.9; two column tiles: 16 x 4096 x 4096 7.1 / 11.8,
    // 16 x 8192 x 4096 12.7 / 14.9 (the line lies where the kernel's former loop lost, 18.3 / 16.6, and is kept: results on
    // either side of it differ in their last bits). Not where a result may not depend on the batch.
    const long long most = M <= 8 ? 100LL << 20 : 16LL << 20;
    if (M <= 16 && (long long)N * K <= most && !transA && transB && !(e->flags & B200_ENGINE_NO_STREAMK) &&
        (((uintptr_t)A | (uintptr_t)B | (uintptr_t)lda | (uintptr_t)ldb | (uintptr_t)K) & 15) == 0) {
      if (M <= 8) launch_skinny<1>(e, b, a, p);
      else launch_skinny<2>(e, b, a, p);
      B200_CHECK_LAUNCH(e, "gemm_blocks_skinny_kernel");
      return B200_OK;
    }
    rc = gemm_blocks_tc(e, sa, sb, a, b, transA != 0, transB == 0, p);
    if (rc != B200_ERR_OOM) return rc;
  }
  // the empty sum, or an arena without room for copies of operands that the TMA unit cannot read in place
  const long long tiles = (M + GB_T - 1) / GB_T * ((N + GB_T - 1) / GB_T);
  launch_kernel(e, gemm_blocks_simt_kernel, (unsigned)std::min<long long>(tiles, 1 << 20), 256, 0, a, b, p);
  B200_CHECK_LAUNCH(e, "gemm_blocks_simt_kernel");
  return B200_OK;
}

}  // extern "C"

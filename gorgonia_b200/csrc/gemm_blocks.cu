// b200_gemm_blocks: matrix products of 8-bit operands with a scale for each block of 128 (quantize.cu).
//
// C[m, n] = act(sum over k-blocks of sa(m, kb) sb(n, kb) (sum over the block's k of a[m, k] b[n, k]) + bias): the
// inner sum is of products of 8-bit values, which fp32 holds exactly; it is taken to fp32 registers once per
// block of 128 and multiplied by the product of the two scales there.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstring>

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
        ra[j] = m < p.M ? a.scales[(m >> a.shift) * a.ss_i + (k0 >> 7) * a.ss_k] : 0.f;
        rb[j] = n < p.N ? b.scales[(n >> b.shift) * b.ss_i + (k0 >> 7) * b.ss_k] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(part[i][j], ra[i] * rb[j], acc[i][j]);
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
  int c_bf16, c_vec;            // c_vec: rows can be stored 16 bytes at a time
  int tiles_m, tiles_n, num_k, group_m;
  int stages, stage_bytes;
  // how the work is shared between the CTAs (TilePieces, tc_common.cuh)
  int streamk, units, sk_first, sk_workers;
  float *ws;
  int *tile_count;
  Epilogue ep;                  // bias_kind in terms of the tiles' rows and columns
  int *err_flag;
};

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

// Warps: 0 loads (TMA), 1 issues MMAs and owns tensor memory, the others (8, or 4 where a tile is 32 columns or
// fewer) take each k-block's accumulator to registers, scaled, and store the tile at its end. A ring stage and an
// accumulator are one k-block each; there are at least as many stages as accumulators, so that one commit per
// k-block, on the stage's "done" barrier, serves the loader and the epilogue: that barrier's next phase cannot
// complete before the epilogue has let go of the accumulator that this one announced.
template <int BN>
__global__ void __launch_bounds__(BN >= 64 ? 320 : 192, 1)
    gemm_blocks_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                          const __grid_constant__ BlocksTcParams p) {
  ptx::grid_begin();
  constexpr int EPI_WARPS = BN >= 64 ? 8 : 4;
  constexpr int HALF = BN / (EPI_WARPS / 4);    // columns an epilogue warp takes
  constexpr int NBUF = BN == 256 ? 2 : 4;       // accumulators in tensor memory
  constexpr int CH = HALF < 32 || HALF == 128 ? 16 : 32;  // columns per tcgen05.ld; 128 sums leave no registers for 32
  constexpr int MAX_STAGES = 12;
  extern __shared__ __align__(1024) unsigned char gb_smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[MAX_STAGES], done_bar[MAX_STAGES], acc_empty[NBUF];
  __shared__ __align__(8) uint64_t epi_bar;  // the epilogue warps meet here when a partial tile is handed over
  __shared__ __align__(16) float s_col[EPI_WARPS][2][HALF];
  __shared__ uint32_t tmem_base_s;
  __shared__ int s_fail, s_last;

  unsigned char *smem = reinterpret_cast<unsigned char *>(((uintptr_t)gb_smem_raw + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stages = p.stages, worker = (int)blockIdx.x, workers = (int)gridDim.x;
  const int total_tiles = p.tiles_m * p.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(&full_bar[s], 1);
      ptx::mbar_init(&done_bar[s], 1);
    }
    for (int b = 0; b < NBUF; ++b) ptx::mbar_init(&acc_empty[b], EPI_WARPS);
    ptx::mbar_init(&epi_bar, EPI_WARPS);
    ptx::fence_mbar_init();
    s_fail = 0;
    s_last = 0;
  }
  if (warp == 1) {
    ptx::tmem_alloc(&tmem_base_s, NBUF * BN);
    ptx::tmem_relinquish();
  }
  if (warp == 0 && lane == 0) {
    ptx::prefetch_tmap(&tmA);
    ptx::prefetch_tmap(&tmB);
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;

  // m blocks are walked in groups so that the CTAs of one wave share columns of B and rows of A in L2
  auto decode = [&](int tile, int &mb, int &nb) {
    const int per_group = p.group_m * p.tiles_n;
    const int g = tile / per_group, first_m = g * p.group_m;
    const int gm = min(p.tiles_m - first_m, p.group_m), r = tile % per_group;
    mb = first_m + r % gm;
    nb = r / gm;
  };

  if (warp == 0) {
    // ---------------- loads ----------------
    if (lane == 0) {
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
  } else if (warp == 1) {
    // ---------------- MMAs ----------------
    if (lane == 0) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      // a k-slice is 32 bytes of a K-major row, or 32 rows of 128 bytes of an MN-major block
      const uint64_t a_step = (p.a_mn ? 32 * 128 : 32) >> 4, b_step = (p.b_mn ? 32 * 128 : 32) >> 4;
      const uint32_t st0 = ptx::smem_addr(smem);
      const uint64_t a_desc0 = make_smem_desc(st0, p.a_mn ? GB_SLAB : 16, 1024, 2);
      const uint64_t b_desc0 = make_smem_desc(st0 + GB_SLAB, p.b_mn ? GB_SLAB : 16, 1024, 2);
      const uint32_t full0 = ptx::smem_addr(&full_bar[0]), done0 = ptx::smem_addr(&done_bar[0]);
      uint32_t ready = 0;
      TilePieces pieces(p.streamk, p.units, p.num_k, total_tiles, worker, workers, p.sk_first, p.sk_workers);
      int tile, kb0, kb1;
      while (ok && pieces.next(tile, kb0, kb1)) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ptx::mbar_wait(&acc_empty[buf], acc_phase ^ 1) || (!ready && !ptx::mbar_wait(&full_bar[stage], phase))) {
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const int ns = stage + 1 == stages ? 0 : stage + 1;
          const uint32_t nphase = ns == 0 ? phase ^ 1u : phase;
          const uint64_t soff = (uint64_t)((uint32_t)stage * (uint32_t)(p.stage_bytes >> 4));
          ready = ptx::kblock_f8(tmem_base + (uint32_t)(buf * BN), a_desc0 + soff, b_desc0 + soff, a_step, b_step, p.idesc,
                                 done0 + (uint32_t)stage * 8u, full0 + (uint32_t)ns * 8u, nphase);
          stage = ns;
          phase = nphase;
          if (++buf == NBUF) {
            buf = 0;
            acc_phase ^= 1;
          }
        }
      }
      if (!ok) s_fail = 1;
    }
  } else {
    // ---------------- scaling, sums and stores ----------------
    const int ew = warp - 2;
    const int quarter = warp & 3;        // the TMEM lanes this warp may read: 32*quarter .. +31
    const int ch0 = (ew >> 2) * HALF;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)ch0;
    int stage = 0, buf = 0;
    uint32_t phase = 0, epi_phase = 0;
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
      const int m = mb * GB_BM + quarter * 32 + lane, n0 = nb * BN + ch0;
      // this thread's row scale, and the warp's column scale(s): one where a tile of scales covers the columns,
      // else one for each, which the lanes fetch and the warp shares through shared memory. Both are fetched a
      // k-block ahead. Rows and columns beyond the matrix read a scale of the last one and are not stored.
      const float *pa = p.a_scales + (long long)(min(m, p.M - 1) >> p.a_shift) * p.as_i;
      const bool per_col = p.b_shift == 0;
      const float *pb = p.b_scales + (per_col ? 0 : (long long)(min(n0, p.N - 1) >> 7) * p.bs_i);
      constexpr int PER = (HALF + 31) / 32;
      float sa = 0.f, sb = 0.f, sc[PER];
      auto fetch = [&](int kb) {
        sa = __ldg(pa + kb * p.as_k);
        if (per_col) {
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (j * 32 + lane < HALF) sc[j] = __ldg(p.b_scales + (long long)min(n0 + j * 32 + lane, p.N - 1) * p.bs_i + kb * p.bs_k);
        } else {
          sb = __ldg(pb + kb * p.bs_k);
        }
      };
      float acc[HALF];
#pragma unroll
      for (int j = 0; j < HALF; ++j) acc[j] = 0.f;
      if (kb0 < kb1) fetch(kb0);
      for (int kb = kb0; kb < kb1; ++kb) {
        const float row = sa, both = __fmul_rn(sa, sb);
        float *cols = s_col[ew][kb & 1];
        if (per_col) {
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (j * 32 + lane < HALF) cols[j * 32 + lane] = sc[j];
          __syncwarp();
        }
        if (kb + 1 < kb1) fetch(kb + 1);
        if (!ptx::mbar_wait(&done_bar[stage], phase)) {
          ok = false;
          break;
        }
        __syncwarp();
        ptx::tc_fence_after_sync();
#pragma unroll
        for (int c = 0; c < HALF; c += CH) {
          uint32_t r[CH];
          if constexpr (CH == 32) ptx::tmem_ld_32x32(lane_addr + (uint32_t)(buf * BN + c), r);
          else ptx::tmem_ld_32x16(lane_addr + (uint32_t)(buf * BN + c), r);
          ptx::tmem_ld_wait();
          if (per_col) {
#pragma unroll
            for (int j = 0; j < CH; j += 4) {
              const float4 s = *reinterpret_cast<const float4 *>(cols + c + j);
              fma_pair(acc[c + j], acc[c + j + 1], r[j], r[j + 1], __fmul_rn(row, s.x), __fmul_rn(row, s.y));
              fma_pair(acc[c + j + 2], acc[c + j + 3], r[j + 2], r[j + 3], __fmul_rn(row, s.z), __fmul_rn(row, s.w));
            }
          } else {
#pragma unroll
            for (int j = 0; j < CH; j += 2) fma_pair(acc[c + j], acc[c + j + 1], r[j], r[j + 1], both, both);
          }
        }
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&acc_empty[buf]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
        if (++buf == NBUF) buf = 0;
      }
      if (kb0 != 0 || kb1 != p.num_k) {
        // part of a tile: leave it in the workspace; the CTA that delivers the last part finishes the tile
        const int tile_u0 = (tile - p.sk_first) * p.num_k;
        const size_t slot_floats = (size_t)GB_BM * BN;
        const size_t within = (size_t)ew * HALF * 32 + lane;
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
        if (warp == 2 && lane == 0) {
          s_last = (atomicAdd(p.tile_count + (tile - p.sk_first), 1) == c_last - c_first) ? 1 : 0;
          if (s_last) p.tile_count[tile - p.sk_first] = 0;  // zero again for the next launch
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
        for (int c = c_first; c <= c_last; ++c) {  // k order: CTA c's share precedes CTA c + 1's
          const float *src = p.ws + (size_t)share_slot(c, tile_u0, p.units, p.sk_workers) * slot_floats + within;
          if constexpr (HALF <= 32) {
            float part[HALF];
#pragma unroll
            for (int j = 0; j < HALF; ++j) part[j] = __ldcg(src + j * 32);
#pragma unroll
            for (int j = 0; j < HALF; ++j) acc[j] = __fadd_rn(acc[j], part[j]);
          } else {
#pragma unroll
            for (int j = 0; j < HALF; ++j) acc[j] = __fadd_rn(acc[j], ptx::ld_cg_ordered(src + j * 32));
          }
        }
      }
      if (ok && m < p.M && n0 < p.N) {
        const int valid = min(HALF, p.N - n0);
        const float *bias = reinterpret_cast<const float *>(p.ep.bias);
        if (p.ep.bias_kind == B200_BIAS_COL) {
  #pragma unroll
          for (int j = 0; j < HALF; ++j)
            if (j < valid) acc[j] = __fadd_rn(acc[j], __ldg(bias + n0 + j));
        } else if (p.ep.bias_kind == B200_BIAS_ROW) {
          const float bm = __ldg(bias + m);
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
        const long long at = (long long)m * p.c_row + (long long)n0 * p.c_col;
        if (p.c_bf16) {
          __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(p.C) + at;
          if (p.c_vec && valid == HALF) {
  #pragma unroll
            for (int j = 0; j < HALF; j += 8) {
              uint4 w;
              uint32_t *ww = reinterpret_cast<uint32_t *>(&w);
  #pragma unroll
              for (int t = 0; t < 4; ++t) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(acc[j + 2 * t], acc[j + 2 * t + 1]);
                ww[t] = *reinterpret_cast<const uint32_t *>(&h);
              }
              *reinterpret_cast<uint4 *>(out + j) = w;
            }
          } else {
  #pragma unroll
            for (int j = 0; j < HALF; ++j)
              if (j < valid) out[j * p.c_col] = __float2bfloat16_rn(acc[j]);
          }
        } else {
          float *out = reinterpret_cast<float *>(p.C) + at;
          if (p.c_vec && valid == HALF) {
            if (p.ep.accumulate) {  // Incr mode: the rounded result is added to what C holds
  #pragma unroll
              for (int j = 0; j < HALF; j += 4) {
                const float4 old = *reinterpret_cast<const float4 *>(out + j);
                *reinterpret_cast<float4 *>(out + j) = make_float4(__fadd_rn(old.x, acc[j]), __fadd_rn(old.y, acc[j + 1]),
                                                                   __fadd_rn(old.z, acc[j + 2]), __fadd_rn(old.w, acc[j + 3]));
              }
            } else {
  #pragma unroll
              for (int j = 0; j < HALF; j += 4)
                *reinterpret_cast<float4 *>(out + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            }
          } else {
  #pragma unroll
            for (int j = 0; j < HALF; ++j)
              if (j < valid) out[j * p.c_col] = p.ep.accumulate ? __fadd_rn(out[j * p.c_col], acc[j]) : acc[j];
          }
        }
      }
    }
    if (!ok) s_fail = 1;
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && s_fail) atomicExch(p.err_flag, 1);
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, NBUF * BN);
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
#pragma unroll
    for (int t = 0; t < 16; ++t) o.b[t] = c + t < j.cols ? s[t] : 0;
    *reinterpret_cast<uint4 *>(j.dst + r * j.ldo + c) = o.v;
  }
}

template <int BN>
static int launch_blocks_tc(b200_engine *e, const CUtensorMap *tm, const BlocksTcParams &p, int grid) {
  auto kern = gemm_blocks_tc_kernel<BN>;
  const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
  static std::atomic<int> attr_dev_mask{0};
  if (!(attr_dev_mask & (1 << (e->device & 31)))) {
    cudaFuncAttributes fa;
    B200_CHECK_CUDA(e, cudaFuncGetAttributes(&fa, kern));
    const size_t optin = std::min<size_t>(e->smem_optin, 227 * 1024);
    B200_CHECK_CUDA(e, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(optin - fa.sharedSizeBytes)));
    attr_dev_mask |= 1 << (e->device & 31);
  }
  launch_kernel(e, kern, grid, BN >= 64 ? 320 : 192, smem, tm[0], tm[1], p);
  B200_CHECK_LAUNCH(e, "gemm_blocks_tc_kernel");
  e->flags_dirty = true;
  return B200_OK;
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
  p.c_vec = !swap && (uintptr_t)q.C % 16 == 0 && q.ldc % (q.c_bf16 ? 8 : 4) == 0;
  p.ep = ep;
  p.err_flag = e->d_flags + 2;
  p.num_k = (int)((q.K + GB_BK - 1) / GB_BK);
  p.tiles_m = (int)((M + GB_BM - 1) / GB_BM);
  // tile width: the widest that still gives every SM a tile
  int bn = 256;
  while (bn > 64 && (long long)p.tiles_m * ((N + bn - 1) / bn) < e->sm_count) bn /= 2;
  while (bn > 16 && bn / 2 >= N) bn /= 2;
  p.tiles_n = (int)((N + bn - 1) / bn);
  const long long total_tiles = (long long)p.tiles_m * p.tiles_n;
  if (total_tiles >= (1LL << 31))
    return set_error(e, B200_ERR_UNSUPPORTED, "b200_gemm_blocks: %lld output tiles are more than one launch takes", total_tiles);
  p.group_m = std::min(p.tiles_m, 8);
  p.stage_bytes = GB_SLAB + (b_mn ? std::max(bn, 128) : bn) * 128;
  const int budget = (int)std::min<size_t>(e->smem_optin, 227 * 1024) - 1024 - 9 * 1024;  // static part, alignment
  p.stages = std::min(12, budget / p.stage_bytes);
  p.idesc = make_idesc(0, a_mn, b_mn, GB_BM, bn) | ((uint32_t)a.e5m2 << 7) | ((uint32_t)b.e5m2 << 10);

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
  CUtensorMap tm[2];
  if (rc == B200_OK) rc = encode_map(e, &tm[0], 1, sa.data, sa.cols, sa.rows, 1, sa.ld, 0, 128, 128, false);
  if (rc == B200_OK) rc = encode_map(e, &tm[1], 1, sb.data, sb.cols, sb.rows, 1, sb.ld, 0, 128, b_mn ? 128 : bn, false);
  int grid = (int)std::min<long long>(total_tiles, e->sm_count);
  p.sk_workers = grid;
  void *ws = nullptr;
  if (rc == B200_OK && !(e->flags & B200_ENGINE_NO_STREAMK)) {
    // whole tiles per CTA would leave SMs idle: share out the k range instead (TilePieces)
    int sk_grid = grid, first = 0;
    if (total_tiles <= b200_engine::kSkCounters && streamk_pays(total_tiles, p.num_k, e->sm_count, &sk_grid)) {
      if (b200_get(e, 2LL * sk_grid * GB_BM * bn * 4, &ws) == B200_OK) {
        p.streamk = 1;
        p.units = (int)(total_tiles * p.num_k);
        grid = p.sk_workers = sk_grid;
      }
    } else if (streamk_tail_pays(total_tiles, p.num_k, e->sm_count, &first, &sk_grid)) {
      if (b200_get(e, 2LL * sk_grid * GB_BM * bn * 4, &ws) == B200_OK) {
        p.streamk = 1;
        p.sk_first = first;
        p.sk_workers = sk_grid;
        p.units = (int)((total_tiles - first) * p.num_k);
      }
    }
    p.tile_count = e->sk_counters;
    p.ws = (float *)ws;
  }
  if (rc == B200_OK) {
    switch (bn) {
      case 256: rc = launch_blocks_tc<256>(e, tm, p, grid); break;
      case 128: rc = launch_blocks_tc<128>(e, tm, p, grid); break;
      case 64: rc = launch_blocks_tc<64>(e, tm, p, grid); break;
      case 32: rc = launch_blocks_tc<32>(e, tm, p, grid); break;
      default: rc = launch_blocks_tc<16>(e, tm, p, grid); break;
    }
  }
  // stream order makes handing the scratch back safe: later users run after this kernel
  for (void *s : {blk[0], blk[1], ws})
    if (s) b200_put(e, s, 0);
  return rc;
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

// b200_gemm_blocks: matrix products of 8-bit operands with a scale for each block of 128 (quantize.cu).
//
// C[m, n] = act(sum over k-blocks of sa(m, kb) sb(n, kb) (sum over the block's k of a[m, k] b[n, k]) + bias): the
// inner sum is of products of 8-bit values, which fp32 holds exactly; it is taken to fp32 registers once per
// block of 128 and multiplied by the two scales there.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "engine.h"
#include "epilogue.cuh"
#include "ptx.cuh"

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
        for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(part[i][j] * ra[i], rb[j], acc[i][j]);
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
  const long long tiles = (M + GB_T - 1) / GB_T * ((N + GB_T - 1) / GB_T);
  launch_kernel(e, gemm_blocks_simt_kernel, (unsigned)std::min<long long>(tiles, 1 << 20), 256, 0, a, b, p);
  B200_CHECK_LAUNCH(e, "gemm_blocks_simt_kernel");
  return B200_OK;
}

}  // extern "C"

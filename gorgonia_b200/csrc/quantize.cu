// b200_quantize_blocks: float32 or bfloat16 matrices rounded to 8 bits with a scale for each block of 128.
//
// A block's scale is the least power of two s >= 2^-126 with amax / s <= qmax, amax the largest finite magnitude of
// the block. Both formats' largest value has the significand 1.75 (448 = 1.75 * 2^8, 57344 = 1.75 * 2^15), so s is
// read off amax's bits: its exponent less 8 (15), and one more where its significand lies above 1.75. x / s is exact
// as a product with 1 / s (a result too small for that lies far below half of the format's least value), and
// the conversion to 8 bits is the only rounding.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "engine.h"
#include "ptx.cuh"

namespace b200 {

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// The bits of |v|, or 0 for NaN and infinities.
__device__ __forceinline__ uint32_t finite_magnitude(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// A block's scale, from the bits of its largest finite magnitude.
template <bool E5M2>
__device__ __forceinline__ float block_scale(uint32_t amax) {
  if (amax == 0) return 1.f;
  const int e = (int)(amax >> 23) + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0) - (E5M2 ? 15 : 8);
  return __uint_as_float((uint32_t)max(e, 1) << 23);
}

template <bool E5M2>
__device__ __forceinline__ uint32_t to_f8(float v) {
  if (fabsf(v) == INFINITY) return (E5M2 ? 0x7cu : 0x7fu) | (v < 0.f ? 0x80u : 0u);
  return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, E5M2 ? __NV_E5M2 : __NV_E4M3);
}

// One CTA per block, whatever its shape; two reads of the block.
template <typename T, bool E5M2>
__global__ void __launch_bounds__(128) quantize_kernel(const T *__restrict__ x, long long ldx, long long rows, long long cols,
                                                       uint8_t *__restrict__ q, long long ldq, float *__restrict__ scales,
                                                       int br, int bc, long long col_blocks) {
  ptx::grid_begin();
  __shared__ uint32_t s_amax;
  const long long rb = blockIdx.x / col_blocks, cb = blockIdx.x % col_blocks;
  const int nr = (int)min((long long)br, rows - rb * br), nc = (int)min((long long)bc, cols - cb * bc);
  x += rb * br * ldx + cb * bc;
  q += rb * br * ldq + cb * bc;
  if (threadIdx.x == 0) s_amax = 0;
  __syncthreads();
  uint32_t amax = 0;
  for (int i = threadIdx.x; i < nr * nc; i += blockDim.x) amax = max(amax, finite_magnitude(widen<T>(x[i / nc * ldx + i % nc])));
  atomicMax(&s_amax, amax);
  __syncthreads();
  const float scale = block_scale<E5M2>(s_amax), inv = 1.f / scale;
  for (int i = threadIdx.x; i < nr * nc; i += blockDim.x)
    q[i / nc * ldq + i % nc] = (uint8_t)to_f8<E5M2>(widen<T>(x[i / nc * ldx + i % nc]) * inv);
  if (threadIdx.x == 0) scales[blockIdx.x] = scale;
}

template <typename T>
static int launch_quantize(b200_engine *e, int qtype, int block, const T *x, long long ldx, long long rows, long long cols,
                           uint8_t *q, long long ldq, float *scales) {
  const int br = block == B200_BLOCK_ROW ? 1 : 128, bc = block == B200_BLOCK_COL ? 1 : 128;
  const long long rbs = (rows + br - 1) / br, cbs = (cols + bc - 1) / bc;
  if (rbs * cbs >= (1LL << 31))
    return set_error(e, B200_ERR_UNSUPPORTED, "b200_quantize_blocks: %lld blocks are more than one launch takes", rbs * cbs);
  if (qtype == B200_E5M2)
    launch_kernel(e, quantize_kernel<T, true>, (unsigned)(rbs * cbs), 128, 0, x, ldx, rows, cols, q, ldq, scales, br, bc, cbs);
  else
    launch_kernel(e, quantize_kernel<T, false>, (unsigned)(rbs * cbs), 128, 0, x, ldx, rows, cols, q, ldq, scales, br, bc, cbs);
  B200_CHECK_LAUNCH(e, "quantize_kernel");
  return B200_OK;
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_quantize_blocks(b200_engine *e, int dtype, int qtype, int block, const void *x, int64_t ldx, int64_t rows,
                         int64_t cols, void *q, int64_t ldq, float *scales) {
  if (!e) return B200_ERR_INVALID;
  std::lock_guard<std::recursive_mutex> lk(e->mu);
  B200_REQUIRE(e, dtype == B200_F32 || dtype == B200_BF16, "b200_quantize_blocks: dtype %d not supported", dtype);
  B200_REQUIRE(e, qtype == B200_E4M3 || qtype == B200_E5M2, "b200_quantize_blocks: %d is no 8-bit dtype", qtype);
  B200_REQUIRE(e, block >= B200_BLOCK_ROW && block <= B200_BLOCK_TILE, "b200_quantize_blocks: unknown block %d", block);
  B200_REQUIRE(e, rows >= 0 && cols >= 0, "b200_quantize_blocks: negative extent");
  if (rows == 0 || cols == 0) return B200_OK;
  B200_REQUIRE(e, ldx >= cols && ldq >= cols, "b200_quantize_blocks: leading dimension too small (%lld %lld)",
               (long long)ldx, (long long)ldq);
  B200_REQUIRE(e, x && q && scales, "b200_quantize_blocks: null pointer");
  B200_REQUIRE(e, (uintptr_t)x % dtype_size(dtype) == 0 && (uintptr_t)scales % 4 == 0,
               "b200_quantize_blocks: a pointer is not aligned to its type");
  DeviceGuard g(e);
  int rc = flush_pending(e);
  if (rc != B200_OK) return rc;
  if (dtype == B200_F32) return launch_quantize<float>(e, qtype, block, (const float *)x, ldx, rows, cols, (uint8_t *)q, ldq, scales);
  return launch_quantize<__nv_bfloat16>(e, qtype, block, (const __nv_bfloat16 *)x, ldx, rows, cols, (uint8_t *)q, ldq, scales);
}

}  // extern "C"

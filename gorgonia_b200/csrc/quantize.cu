// b200_quantize_blocks: float32 or bfloat16 matrices rounded to 8 bits with a scale for each block of 128.
//
// A block's scale is the least power of two s >= 2^-126 with amax / s <= qmax, amax the largest finite magnitude of
// the block. Both formats' largest value has the significand 1.75 (448 = 1.75 * 2^8, 57344 = 1.75 * 2^15), so s is
// read off amax's bits: its exponent less 8 (15), and one more where its significand lies above 1.75. x / s is exact
// as a product with 1 / s (a result too small for that lies far below half of the format's least value), and
// the conversion to 8 bits is the only rounding.
//
// One pass: a block's values stay in registers between the search for its largest and the rounding. Float32 is bound
// by HBM (8192 x 4096 to e4m3 by rows 33 us, by columns or tiles 29: 78 and 89 % of the copy rate), and so is bfloat16 by tiles
// (17.4 us, 89 %). By rows (20.3) and columns (23.8) bfloat16 is at no unit's limit: by rows 60 % of the issue slots, 39 % of the
// DRAM rate and 42 % of the warps are in use (by columns it has not been looked at), so there are too few loads in flight.
// Rows that do not start on 16-byte boundaries are read value by value (8191 x 4095 bf16 by rows 35 us).
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

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

// 1 / scale, a power of two from 2^-126 to 2^120.
__device__ __forceinline__ float inverse(float scale) { return __uint_as_float((254u << 23) - __float_as_uint(scale)); }

// Four values to four bytes. ODD: an infinity may be among them. (Chosen by a branch of the warp's, not of the lanes':
// the few instructions are otherwise made conditional and issued always.)
template <bool E5M2, bool ODD>
__device__ __forceinline__ uint32_t to_f8x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  if (E5M2) {
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  } else {
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  }
  uint32_t r = (uint32_t)lo | (uint32_t)hi << 16;
  if (ODD) {
    const float v[4] = {a, b, c, d};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (fabsf(v[j]) == INFINITY) r = (r & ~(0x7fu << (8 * j))) | (E5M2 ? 0x7cu : 0x7fu) << (8 * j);
  }
  return r;
}

// Values as they are loaded: 16 bytes, or fewer where the rows do not start on 16-byte boundaries (V = 1).
template <typename T, int V>
struct alignas(V * sizeof(T)) Values {
  T v[V];
};

// V values to V bytes.
template <typename T, int V, bool E5M2, bool ODD>
__device__ __forceinline__ void store_f8(uint8_t *q, const Values<T, V> &x, float inv) {
  if constexpr (V == 8) {
    const uint4 p = *reinterpret_cast<const uint4 *>(&x);
    const auto low = [&](uint32_t w) { return __uint_as_float(w << 16) * inv; };
    const auto high = [&](uint32_t w) { return __uint_as_float(w & 0xffff0000u) * inv; };
    *reinterpret_cast<uint2 *>(q) = make_uint2(to_f8x4<E5M2, ODD>(low(p.x), high(p.x), low(p.y), high(p.y)),
                                               to_f8x4<E5M2, ODD>(low(p.z), high(p.z), low(p.w), high(p.w)));
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint32_t *>(q) =
        to_f8x4<E5M2, ODD>(widen<T>(x.v[0]) * inv, widen<T>(x.v[1]) * inv, widen<T>(x.v[2]) * inv, widen<T>(x.v[3]) * inv);
  } else {
    *q = (uint8_t)to_f8x4<E5M2, ODD>(widen<T>(x.v[0]) * inv, 0.f, 0.f, 0.f);
  }
}

// The larger of two pairs of 16-bit numbers each.
__device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The largest magnitude of V values as float32 bits, NaN and infinities above all numbers. Two bfloat16 values to an
// instruction: their bits are in the order of the magnitudes as float32's are.
template <typename T, int V>
__device__ __forceinline__ uint32_t largest_of(const Values<T, V> &x) {
  if constexpr (sizeof(T) == 2 && V == 8) {
    const uint4 w = *reinterpret_cast<const uint4 *>(&x);
    const uint32_t m = max_pairs(max_pairs(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), max_pairs(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) m = max(m, __float_as_uint(widen<T>(x.v[j])) & 0x7fffffffu);
    return m;
  }
}

// 1 x 128 blocks: 128 / V lanes hold a block (32 of four values where V = 1), the largest magnitude by shuffles. A
// warp takes `U` steps of 32 * V consecutive values of a row at a time, all loads first.
template <typename T, int V, bool E5M2>
__global__ void __launch_bounds__(256, 4) quantize_rows_kernel(const T *__restrict__ x, long long ldx, long long rows, long long cols,
                                                            uint8_t *__restrict__ q, long long ldq, float *__restrict__ scales) {
  ptx::grid_begin();
  constexpr int U = 4;
  constexpr int STEP = V == 1 ? 128 : 32 * V;      // values of a row per warp and step
  constexpr int PER = V == 1 ? 4 : 1;              // loads per lane and step
  constexpr int LANES = V == 1 ? 32 : 128 / V;     // lanes of a block
  const int lane = threadIdx.x & 31;
  const long long blocks = (cols + 127) / 128, c0 = (long long)blockIdx.x * (U * STEP);
  const int n = (int)min((long long)(U * STEP), cols - c0);  // of the row that are this warp's
  const int at = V == 1 ? lane : lane * V;                   // the lane's first, of each step
  for (long long r = blockIdx.y * 8LL + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8LL) {
    const T *xr = x + r * ldx + c0 + at;
    uint8_t *qr = q + r * ldq + c0 + at;
    float *sr = scales + r * blocks + c0 / 128 + (V == 1 ? 0 : lane / LANES);
    Values<T, V> v[U][PER];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (u * STEP + i * 32 + at < n) {
          v[u][i] = *reinterpret_cast<const Values<T, V> *>(xr + u * STEP + i * 32);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) v[u][i].v[j] = (T)0.f;
        }
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * STEP >= n) break;
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) amax = max(amax, largest_of<T, V>(v[u][i]));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const bool any_odd = __any_sync(0xffffffffu, amax >= 0x7f800000u);
      if (any_odd) {  // NaN or infinities: the largest of the others
        amax = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) amax = max(amax, finite_magnitude(widen<T>(v[u][i].v[j])));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      }
      const float scale = block_scale<E5M2>(amax), inv = inverse(scale);
      if (lane % LANES == 0 && u * STEP + at < n) sr[u * (STEP / 128)] = scale;
      auto store = [&](auto any) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (u * STEP + i * 32 + at < n) store_f8<T, V, E5M2, decltype(any)::value>(qr + u * STEP + i * 32, v[u][i], inv);
      };
      if (any_odd) store(std::true_type());
      else store(std::false_type());
    }
  }
}

// 128 x 1 blocks (COL) and 128 x 128 ones: a block of 256 threads holds a tile of 128 rows and 16 * V columns (V > 1;
// 32 columns where V = 1) in registers; columns' maxima are joined through shared memory.
template <typename T, int V, bool E5M2, bool COL>
__global__ void __launch_bounds__(256) quantize_tiles_kernel(const T *__restrict__ x, long long ldx, long long rows, long long cols,
                                                             uint8_t *__restrict__ q, long long ldq, float *__restrict__ scales) {
  ptx::grid_begin();
  constexpr int TX = COL ? (V == 1 ? 32 : 16) : (V == 1 ? 32 : 128 / V);  // threads across the columns
  constexpr int REP = (!COL && V == 1) ? 4 : 1;                           // steps across them
  constexpr int WIDE = TX * V * REP, TY = 256 / TX, R = 128 / TY;
  __shared__ uint32_t s_max[COL ? 8 : 1][COL ? WIDE : 8];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long c0 = (long long)blockIdx.x * WIDE, r0 = (long long)blockIdx.y * 128;
  Values<T, V> v[R][REP];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int k = 0; k < REP; ++k) {
      const long long r = r0 + i * TY + ty, c = c0 + (k * TX + tx) * V;
      if (r < rows && c < cols) {
        v[i][k] = *reinterpret_cast<const Values<T, V> *>(x + r * ldx + c);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][k].v[j] = (T)0.f;
      }
    }
  // the largest magnitudes of the block's columns (one value for a tile); finite: without NaN and infinities
  uint32_t amax[COL ? V : 1];
  auto largest = [&](bool finite) {
#pragma unroll
    for (int j = 0; j < (COL ? V : 1); ++j) amax[j] = 0;
    if (!finite && COL && sizeof(T) == 2 && V == 8) {  // two columns to an instruction, as in largest_of
      uint32_t m[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&v[i][0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) m[j] = max_pairs(m[j], w[j] & 0x7fff7fffu);
      }
#pragma unroll
      for (int j = 0; j < (COL ? V : 1); ++j) amax[j] = j & 1 ? m[(j / 2) & 3] & 0xffff0000u : m[(j / 2) & 3] << 16;
    } else {
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int k = 0; k < REP; ++k) {
          if (!finite && !COL) {
            amax[0] = max(amax[0], largest_of<T, V>(v[i][k]));
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float f = widen<T>(v[i][k].v[j]);
              uint32_t &m = amax[COL ? j : 0];
              m = max(m, finite ? finite_magnitude(f) : __float_as_uint(f) & 0x7fffffffu);
            }
          }
        }
    }
#pragma unroll
    for (int o = 16; o >= (COL ? TX : 1); o >>= 1)
#pragma unroll
      for (int j = 0; j < (COL ? V : 1); ++j) amax[j] = max(amax[j], __shfl_xor_sync(0xffffffffu, amax[j], o));
    __syncthreads();
    if (COL) {
      if (lane < TX) {
#pragma unroll
        for (int j = 0; j < V; ++j) s_max[warp][tx * V + j] = amax[COL ? j : 0];
      }
    } else if (lane == 0) {
      s_max[0][warp] = amax[0];
    }
    __syncthreads();
    if (COL) {  // a thread per column, then everybody reads what its own columns have
      if ((int)threadIdx.x < WIDE) {
        uint32_t m = s_max[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < (COL ? 8 : 1); ++w) m = max(m, s_max[w][threadIdx.x]);
        s_max[0][threadIdx.x] = m;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < (COL ? V : 1); ++j) amax[j] = s_max[0][COL ? tx * V + j : 0];
    } else {
#pragma unroll
      for (int w = 0; w < 8; ++w) amax[0] = max(amax[0], s_max[0][COL ? 0 : w]);
    }
  };
  largest(false);
  bool odd = false;
#pragma unroll
  for (int j = 0; j < (COL ? V : 1); ++j) odd |= amax[j] >= 0x7f800000u;
  const bool any_odd = __syncthreads_or(odd);
  if (any_odd) largest(true);
  float inv[COL ? V : 1];
#pragma unroll
  for (int j = 0; j < (COL ? V : 1); ++j) {
    const float scale = block_scale<E5M2>(amax[j]);
    inv[j] = inverse(scale);
    if (COL) {
      if (ty == 0 && c0 + tx * V + j < cols) scales[(long long)blockIdx.y * cols + c0 + tx * V + j] = scale;
    } else if (threadIdx.x == 0) {
      scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = scale;
    }
  }
  auto store = [&](auto any) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int k = 0; k < REP; ++k) {
        const long long r = r0 + i * TY + ty, c = c0 + (k * TX + tx) * V;
        if (r >= rows || c >= cols) continue;
        uint8_t *to = q + r * ldq + c;
        if constexpr (COL && V > 1) {
          uint32_t w[V / 4];
#pragma unroll
          for (int j = 0; j < V; j += 4)
            w[j / 4] = to_f8x4<E5M2, decltype(any)::value>(widen<T>(v[i][k].v[j]) * inv[j], widen<T>(v[i][k].v[j + 1]) * inv[j + 1],
                                     widen<T>(v[i][k].v[j + 2]) * inv[j + 2], widen<T>(v[i][k].v[j + 3]) * inv[j + 3]);
          if constexpr (V == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
          else *reinterpret_cast<uint32_t *>(to) = w[0];
        } else {
          store_f8<T, V, E5M2, decltype(any)::value>(to, v[i][k], inv[0]);
        }
      }
  };
  if (any_odd) store(std::true_type());
  else store(std::false_type());
}

template <typename T, int V, bool E5M2>
static void launch_quantize_as(b200_engine *e, int block, const T *x, long long ldx, long long rows, long long cols, uint8_t *q,
                               long long ldq, float *scales) {
  if (block == B200_BLOCK_ROW) {
    // a warp per row and piece of it; eight rows per block
    const long long step = 4 * (V == 1 ? 128 : 32 * V);
    launch_kernel(e, quantize_rows_kernel<T, V, E5M2>,
                  dim3((unsigned)((cols + step - 1) / step), (unsigned)std::min<long long>((rows + 7) / 8, 65535)), 256, 0, x, ldx, rows,
                  cols, q, ldq, scales);
    return;
  }
  const bool col = block == B200_BLOCK_COL;
  const long long wide = col ? (V == 1 ? 32 : 16 * V) : 128;
  const dim3 grid((unsigned)((cols + wide - 1) / wide), (unsigned)((rows + 127) / 128));
  if (col) launch_kernel(e, quantize_tiles_kernel<T, V, E5M2, true>, grid, 256, 0, x, ldx, rows, cols, q, ldq, scales);
  else launch_kernel(e, quantize_tiles_kernel<T, V, E5M2, false>, grid, 256, 0, x, ldx, rows, cols, q, ldq, scales);
}

template <typename T>
static int launch_quantize(b200_engine *e, int qtype, int block, const T *x, long long ldx, long long rows, long long cols,
                           uint8_t *q, long long ldq, float *scales) {
  constexpr int V = 16 / sizeof(T);
  if ((cols + 31) / 32 >= (1LL << 31))
    return set_error(e, B200_ERR_UNSUPPORTED, "b200_quantize_blocks: %lld columns are more than one launch takes", cols);
  // 16-byte loads where every row's vectors lie on their boundaries, and what is stored for them too
  const bool vec = (uintptr_t)x % 16 == 0 && ldx % V == 0 && (uintptr_t)q % V == 0 && ldq % V == 0 && cols % V == 0;
  auto launch = [&](const T *xr, long long n, uint8_t *qr, float *sr) {
    if (qtype == B200_E5M2) {
      if (vec) launch_quantize_as<T, V, true>(e, block, xr, ldx, n, cols, qr, ldq, sr);
      else launch_quantize_as<T, 1, true>(e, block, xr, ldx, n, cols, qr, ldq, sr);
    } else {
      if (vec) launch_quantize_as<T, V, false>(e, block, xr, ldx, n, cols, qr, ldq, sr);
      else launch_quantize_as<T, 1, false>(e, block, xr, ldx, n, cols, qr, ldq, sr);
    }
  };
  // Tiles and columns have a block of the grid for each 128 rows, 65535 at most: more rows take several launches. (Rows that
  // follow each other by ldx, a multiple of V where `vec` holds, keep their alignment.)
  const long long piece = block == B200_BLOCK_ROW ? rows : 65535LL * 128;
  const long long scales_of_128 = block == B200_BLOCK_COL ? cols : (cols + 127) / 128;
  for (long long r = 0; r < rows; r += piece) {
    launch(x + r * ldx, std::min(piece, rows - r), q + r * ldq, scales + r / 128 * scales_of_128);
    B200_CHECK_LAUNCH(e, "quantize_kernel");
  }
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

// b200_token_logprobs and its gradient: what a loss, and sampling, read from the logits of a row.
//
//   lse = m + ln s, m = max x, s = sum e^(x - m);  logp = (x[t] - m) - ln s;  H = ln s - (sum e^(x - m) (x - m)) / s
// (the log probability not as x[t] - lse: in a row that is masked with the type's lowest value, m + ln s is m).
// A logit of -Inf has e = 0 and no term in either sum. A row of nothing else has s = 0: lse -Inf, entropy 0.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "engine.h"
#include "ptx.cuh"

namespace b200 {

template <typename T>
struct LogitTraits;
template <>
struct LogitTraits<float> { using Stat = float; };
template <>
struct LogitTraits<double> { using Stat = double; };
template <>
struct LogitTraits<__nv_bfloat16> { using Stat = float; };

__device__ __forceinline__ float widen_logit(float v) { return v; }
__device__ __forceinline__ double widen_logit(double v) { return v; }
__device__ __forceinline__ float widen_logit(__nv_bfloat16 v) { return __bfloat162float(v); }

// Whether (v, i) stands in front of (w, j) among the alternatives: the larger value, NaN above all, the lower index.
template <typename S>
__device__ __forceinline__ bool in_front(S v, long long i, S w, long long j) {
  if (v != v) return w == w || i < j;
  return v > w || (v == w && i < j);
}

template <typename S, typename F>
__device__ S block_reduce(S v, S *buf, F f) {
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v = f(v, buf[w]);
  return v;
}

// One CTA per row: the maximum, the sums, then one search per alternative.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_kernel(const T *__restrict__ x, long long ldx, long long vocab,
                                                             const long long *__restrict__ targets,
                                                             typename LogitTraits<T>::Stat *__restrict__ logp,
                                                             typename LogitTraits<T>::Stat *__restrict__ entropy,
                                                             typename LogitTraits<T>::Stat *__restrict__ lse_out, int top,
                                                             typename LogitTraits<T>::Stat *__restrict__ top_logp,
                                                             long long *__restrict__ top_index, int *bad) {
  ptx::grid_begin();
  using S = typename LogitTraits<T>::Stat;
  __shared__ S buf[8];
  __shared__ S s_val[8];
  __shared__ long long s_idx[8];
  const long long r = blockIdx.x;
  x += r * ldx;
  const S inf = (S)INFINITY;
  S m = -inf;
  bool wild = false;
  for (long long i = threadIdx.x; i < vocab; i += blockDim.x) {
    const S v = widen_logit(x[i]);
    wild |= v != v || v == inf;
    if (v > m) m = v;
  }
  m = block_reduce(m, buf, [](S a, S b) { return a > b ? a : b; });
  wild = __syncthreads_or(wild);
  S s = 0, t = 0;
  for (long long i = threadIdx.x; i < vocab; i += blockDim.x) {
    const S v = widen_logit(x[i]);
    if (v > -inf) {
      s += exp(v - m);
      t += exp(v - m) * (v - m);
    }
  }
  s = block_reduce(s, buf, [](S a, S b) { return a + b; });
  t = block_reduce(t, buf, [](S a, S b) { return a + b; });
  const S nan = inf - inf;
  const S log_s = log(s), lse = wild ? nan : s > 0 ? m + log_s : -inf;
  auto log_prob = [&](S v) { return wild ? nan : s > 0 ? (v - m) - log_s : -inf; };
  if (threadIdx.x == 0) {
    if (lse_out) lse_out[r] = lse;
    if (entropy) entropy[r] = wild ? nan : s > 0 ? log_s - t / s : S(0);
    if (targets) {
      const long long k = targets[r];
      if (k >= 0 && k < vocab) {
        logp[r] = log_prob(widen_logit(x[k]));
      } else {
        logp[r] = k == B200_NO_TOKEN ? S(0) : nan;
        if (k != B200_NO_TOKEN) atomicExch(bad, 1);
      }
    }
  }
  S last = nan;
  long long last_i = -1;  // in front of everything
  for (int k = 0; k < top; ++k) {
    S best = -inf;
    long long best_i = LLONG_MAX;
    for (long long i = threadIdx.x; i < vocab; i += blockDim.x) {
      const S v = widen_logit(x[i]);
      if (in_front(last, last_i, v, i) && (best_i == LLONG_MAX || in_front(v, i, best, best_i))) {
        best = v;
        best_i = i;
      }
    }
    auto take = [&](S v, long long i) {
      if (i != LLONG_MAX && (best_i == LLONG_MAX || in_front(v, i, best, best_i))) {
        best = v;
        best_i = i;
      }
    };
    for (int o = 16; o > 0; o >>= 1) {
      const S v = __shfl_xor_sync(0xffffffffu, best, o);
      const long long i = __shfl_xor_sync(0xffffffffu, best_i, o);
      take(v, i);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      s_val[threadIdx.x >> 5] = best;
      s_idx[threadIdx.x >> 5] = best_i;
    }
    __syncthreads();
    for (int w = 0; w < 8; ++w) take(s_val[w], s_idx[w]);
    last = best;
    last_i = best_i;
    if (threadIdx.x == 0) {
      top_logp[r * top + k] = log_prob(best);
      top_index[r * top + k] = best_i;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_bwd_kernel(const T *x, long long ldx, long long vocab,
                                                                 const long long *__restrict__ targets,
                                                                 const typename LogitTraits<T>::Stat *__restrict__ lse,
                                                                 const typename LogitTraits<T>::Stat *__restrict__ entropy,
                                                                 const typename LogitTraits<T>::Stat *__restrict__ grad_logp,
                                                                 const typename LogitTraits<T>::Stat *__restrict__ grad_entropy,
                                                                 T *dx, long long lddx, int *bad) {
  ptx::grid_begin();
  using S = typename LogitTraits<T>::Stat;
  const long long r = blockIdx.x, k = targets[r];
  x += r * ldx;
  dx += r * lddx;
  const bool inside = k >= 0 && k < vocab;
  if (!inside && k != B200_NO_TOKEN && threadIdx.x == 0) atomicExch(bad, 1);
  const S g = inside ? grad_logp[r] : S(0), h = grad_entropy ? grad_entropy[r] : S(0);
  const bool none = g == S(0) && h == S(0);
  const S l = none ? S(0) : lse[r], ent = h != S(0) ? entropy[r] : S(0);
  const bool zero = none || l == -(S)INFINITY;
  for (long long i = threadIdx.x; i < vocab; i += blockDim.x) {
    S d = 0;
    if (!zero) {
      const S lp = widen_logit(x[i]) - l, p = exp(lp);
      d = i == k ? g : S(0);
      d -= g * p;
      if (h != S(0) && !(p == S(0))) d -= h * p * (lp + ent);
    }
    dx[i] = (T)d;
  }
}

template <typename T>
static int launch_forward(b200_engine *e, const void *x, long long ldx, long long rows, long long vocab, const int64_t *targets,
                          void *logp, void *entropy, void *lse, int top, void *top_logp, int64_t *top_index) {
  using S = typename LogitTraits<T>::Stat;
  launch_kernel(e, token_logprobs_kernel<T>, (unsigned)rows, 256, 0, (const T *)x, ldx, vocab, (const long long *)targets,
                (S *)logp, (S *)entropy, (S *)lse, top, (S *)top_logp, (long long *)top_index, e->d_flags + 4);
  B200_CHECK_LAUNCH(e, "token_logprobs_kernel");
  return B200_OK;
}

template <typename T>
static int launch_backward(b200_engine *e, const void *x, long long ldx, long long rows, long long vocab, const int64_t *targets,
                           const void *lse, const void *entropy, const void *grad_logp, const void *grad_entropy, void *dx,
                           long long lddx) {
  using S = typename LogitTraits<T>::Stat;
  launch_kernel(e, token_logprobs_bwd_kernel<T>, (unsigned)rows, 256, 0, (const T *)x, ldx, vocab, (const long long *)targets,
                (const S *)lse, (const S *)entropy, (const S *)grad_logp, (const S *)grad_entropy, (T *)dx, lddx,
                e->d_flags + 4);
  B200_CHECK_LAUNCH(e, "token_logprobs_bwd_kernel");
  return B200_OK;
}

// A launch has been made that checks its token indices.
static void note_tokens(b200_engine *e) {
  if (e->capturing) {
    e->capture_has_tokens = true;  // the check replays with the tape
  } else {
    e->flags_dirty = true;
    e->tokens_dirty = true;
  }
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_token_logprobs(b200_engine *e, int dtype, const void *x, int64_t ldx, int64_t rows, int64_t vocab,
                        const int64_t *targets, void *logp, void *entropy, void *lse, int top, void *top_logp,
                        int64_t *top_index) {
  if (!e) return B200_ERR_INVALID;
  std::lock_guard<std::recursive_mutex> lk(e->mu);
  B200_REQUIRE(e, dtype == B200_F32 || dtype == B200_F64 || dtype == B200_BF16, "b200_token_logprobs: dtype %d not supported",
               dtype);
  B200_REQUIRE(e, rows >= 0 && vocab >= 1 && rows < (1LL << 31) && vocab < (1LL << 31), "b200_token_logprobs: bad extent");
  B200_REQUIRE(e, top >= 0 && top <= B200_TOP_MAX && top <= vocab, "b200_token_logprobs: %d alternatives of %lld (at most %d)",
               top, (long long)vocab, B200_TOP_MAX);
  B200_REQUIRE(e, ldx >= vocab, "b200_token_logprobs: leading dimension too small (%lld)", (long long)ldx);
  if (rows == 0) return B200_OK;
  B200_REQUIRE(e, x != nullptr, "b200_token_logprobs: x is null");
  B200_REQUIRE(e, (targets == nullptr) == (logp == nullptr), "b200_token_logprobs: targets and logp go together");
  B200_REQUIRE(e, top == 0 ? !top_logp && !top_index : top_logp && top_index,
               "b200_token_logprobs: top_logp and top_index go together with top > 0");
  const size_t es = dtype_size(dtype), ss = dtype == B200_F64 ? 8 : 4;
  B200_REQUIRE(e, (uintptr_t)x % es == 0 && ((uintptr_t)targets | (uintptr_t)top_index) % 8 == 0 &&
                      ((uintptr_t)logp | (uintptr_t)entropy | (uintptr_t)lse | (uintptr_t)top_logp) % ss == 0,
               "b200_token_logprobs: a pointer is not aligned to its type");
  DeviceGuard g(e);
  int rc = flush_pending(e);
  if (rc != B200_OK) return rc;
  if (dtype == B200_F32) rc = launch_forward<float>(e, x, ldx, rows, vocab, targets, logp, entropy, lse, top, top_logp, top_index);
  else if (dtype == B200_F64) rc = launch_forward<double>(e, x, ldx, rows, vocab, targets, logp, entropy, lse, top, top_logp, top_index);
  else rc = launch_forward<__nv_bfloat16>(e, x, ldx, rows, vocab, targets, logp, entropy, lse, top, top_logp, top_index);
  if (rc == B200_OK && targets) note_tokens(e);
  return rc;
}

int b200_token_logprobs_bwd(b200_engine *e, int dtype, const void *x, int64_t ldx, int64_t rows, int64_t vocab,
                            const int64_t *targets, const void *lse, const void *entropy, const void *grad_logp,
                            const void *grad_entropy, void *dx, int64_t lddx) {
  if (!e) return B200_ERR_INVALID;
  std::lock_guard<std::recursive_mutex> lk(e->mu);
  B200_REQUIRE(e, dtype == B200_F32 || dtype == B200_F64 || dtype == B200_BF16,
               "b200_token_logprobs_bwd: dtype %d not supported", dtype);
  B200_REQUIRE(e, rows >= 0 && vocab >= 1 && rows < (1LL << 31) && vocab < (1LL << 31), "b200_token_logprobs_bwd: bad extent");
  B200_REQUIRE(e, ldx >= vocab && lddx >= vocab, "b200_token_logprobs_bwd: leading dimension too small (%lld %lld)",
               (long long)ldx, (long long)lddx);
  if (rows == 0) return B200_OK;
  B200_REQUIRE(e, x && targets && lse && grad_logp && dx, "b200_token_logprobs_bwd: null pointer");
  B200_REQUIRE(e, !grad_entropy || entropy, "b200_token_logprobs_bwd: grad_entropy needs the entropy");
  B200_REQUIRE(e, dx != x || lddx == ldx, "b200_token_logprobs_bwd: in place, both leading dimensions must be the same");
  const size_t es = dtype_size(dtype), ss = dtype == B200_F64 ? 8 : 4;
  B200_REQUIRE(e, ((uintptr_t)x | (uintptr_t)dx) % es == 0 && (uintptr_t)targets % 8 == 0 &&
                      ((uintptr_t)lse | (uintptr_t)entropy | (uintptr_t)grad_logp | (uintptr_t)grad_entropy) % ss == 0,
               "b200_token_logprobs_bwd: a pointer is not aligned to its type");
  DeviceGuard g(e);
  int rc = flush_pending(e);
  if (rc != B200_OK) return rc;
  if (dtype == B200_F32) rc = launch_backward<float>(e, x, ldx, rows, vocab, targets, lse, entropy, grad_logp, grad_entropy, dx, lddx);
  else if (dtype == B200_F64) rc = launch_backward<double>(e, x, ldx, rows, vocab, targets, lse, entropy, grad_logp, grad_entropy, dx, lddx);
  else rc = launch_backward<__nv_bfloat16>(e, x, ldx, rows, vocab, targets, lse, entropy, grad_logp, grad_entropy, dx, lddx);
  if (rc == B200_OK) note_tokens(e);
  return rc;
}

}  // extern "C"

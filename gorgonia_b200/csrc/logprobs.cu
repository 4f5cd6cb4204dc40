// b200_token_logprobs and its gradient: what a loss, and sampling, read from the logits of a row.
//
//   lse = m + ln s, m = max x, s = sum e^(x - m);  logp = (x[t] - m) - ln s;  H = ln s - (sum e^(x - m) (x - m)) / s
// (the log probability not as x[t] - lse: in a row that is masked with the type's lowest value, m + ln s is m).
// A logit of -Inf has e = 0 and no term in either sum. A row of nothing else has s = 0: lse -Inf, entropy 0. A NaN or
// +Inf makes s a NaN, which is how such rows are told.
//
// Forward: one pass, bound by HBM. Every thread of a row's block keeps a running maximum and both sums of its
// share, relative to that maximum, and rescales them when it grows; shares are joined at the end. Rows that are
// few and long are shared by a cluster of up to eight blocks, which join through distributed shared memory.
// float32 sums are of powers of two: a term is 2^d, d = (x - m) log2 e. (d as one fma from x log2 e would save an
// instruction; it has no value where m is the type's lowest, as in a row that a mask leaves nothing of.)
//
// Alternatives, without a second pass: the threads' maxima are of different logits, so the k-th largest of them
// bounds the k-th largest logit from below, and close: few logits lie above it, all of them in the shares of
// threads whose maximum does. Only these shares are read again (from L2; k of up to 512), and what is not below the
// bound is put in order. Rows of many equal logits (a mask that leaves fewer tokens than are asked for) overflow the
// list: then only what lies above the bound is taken, and the first equals from the row's start on. What overflows
// all the same (the best logits side by side in one share), and rows with a NaN, are searched once per alternative.
//
// Measured: 4096 x 32000 float32 85 us (94 % of the copy rate), with 5 alternatives 100; 8 x 131072 bf16 with 20 alternatives
// 10.5 us, without any 4.7; gradient of 4096 x 32000 bf16 81 us (99 % of the copy rate), float32 153. Not bound by HBM: bf16, 54 and 67
// us (75 and 60 %: 74 % of the issue slots with 20 alternatives), and float64, 4096 x 16000 211 and 221 us (38 %), its
// gradient 231 (70 %): the exponentials of 64 bits. Rows of a few classes have a warp each: 2^20 x 10 float32 608 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "engine.h"
#include "ptx.cuh"

namespace b200 {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float widen_logit(float v) { return v; }
__device__ __forceinline__ double widen_logit(double v) { return v; }
__device__ __forceinline__ float widen_logit(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T narrow_logit(float v);
template <>
__device__ __forceinline__ float narrow_logit<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow_logit<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// What differs between sums in float32 and in float64. Key: an unsigned number in the order of the values (zeros
// of both signs are equal, a NaN is above all).
template <typename S>
struct Num;
template <>
struct Num<float> {
  using Key = uint32_t;
  static __device__ __forceinline__ float power(float d) { return ex2(d); }
  static __device__ __forceinline__ float distance(float x, float o) { return (x - o) * LOG2E; }
  static __device__ __forceinline__ float entropy(float s, float t) { return logf(s) - t / s * LN2; }
  static __device__ __forceinline__ float far() { return -1e4f; }
  static __device__ __forceinline__ Key key(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(Key k) {
    return k == 0xffffffffu ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
  }
};
template <>
struct Num<double> {
  using Key = unsigned long long;
  static __device__ __forceinline__ double power(double d) { return exp(d); }
  static __device__ __forceinline__ double distance(double x, double o) { return x - o; }
  static __device__ __forceinline__ double entropy(double s, double t) { return log(s) - t / s; }
  static __device__ __forceinline__ double far() { return -1e4; }
  static __device__ __forceinline__ Key key(double v) {
    if (v != v) return ~0ull;
    const Key b = (Key)__double_as_longlong(v + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
  }
  static __device__ __forceinline__ double value(Key k) {
    return k == ~0ull ? (double)NAN : __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k));
  }
};

// A share's maximum m, the offset o that its sums are relative to (m, or 0 where m is -Inf), and the sums of 2^d (e^d),
// d the distance from o in powers of two (of e), and of that times d.
template <typename S>
struct Share {
  S m = -(S)INFINITY, o = 0, s = 0, t = 0;
  __device__ __forceinline__ void raise(S top) {  // the maximum becomes top > m
    if (s > S(0)) {
      const S by = fmax(Num<S>::distance(o, top), Num<S>::far()), f = Num<S>::power(by);
      t = f * (t + by * s);
      s = f * s;
    }
    m = o = top;
  }
  __device__ __forceinline__ void add(S x) {
    const S d = Num<S>::distance(x, o), e = Num<S>::power(d);
    s += e;
    t = fma(e, fmax(d, Num<S>::far()), t);  // e = 0 for anything as far down, -Inf among it
  }
  __device__ __forceinline__ void join_lanes();
  __device__ __forceinline__ void join(S m2, S o2, S s2, S t2) {
    if (m2 > m) {
      const S a = m, b = o, c = s, d = t;
      m = m2; o = o2; s = s2; t = t2;
      m2 = a; o2 = b; s2 = c; t2 = d;
    }
    const S by = fmax(Num<S>::distance(o2, o), Num<S>::far()), f = Num<S>::power(by);
    if (s2 != S(0)) {
      s += f * s2;
      t += f * (t2 + by * s2);
    }
  }
};

// Every lane's share becomes that of the warp.
template <typename S>
__device__ __forceinline__ void Share<S>::join_lanes() {
  S top = m;
#pragma unroll
  for (int o2 = 16; o2 > 0; o2 >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o2));
  if (top > m) raise(top);
#pragma unroll
  for (int o2 = 16; o2 > 0; o2 >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o2);
    t += __shfl_xor_sync(0xffffffffu, t, o2);
  }
}

template <typename T>
struct LogitTraits { using Stat = float; };
template <>
struct LogitTraits<double> { using Stat = double; };

template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
};

constexpr int LP_LIST = 1024;  // candidates that are put in order

// The kernel's arguments, for the row's type T and Stat S.
template <typename T>
struct LogprobArgs {
  using S = typename LogitTraits<T>::Stat;
  const T *x;
  long long ldx, vocab;
  const long long *targets;
  S *logp, *entropy, *lse;
  int top;
  S *top_logp;
  long long *top_index;
  int *bad;
};

// One block, or a cluster of CL, per row. V: values per load; a row's head up to the first 16-byte boundary, and its
// tail, are read one by one.
template <typename T, int V, int CL>
__global__ void __launch_bounds__(CL > 1 ? 512 : 256, CL > 1 ? 2 : 5) token_logprobs_kernel(const LogprobArgs<T> a) {
  ptx::grid_begin();
  using S = typename LogitTraits<T>::Stat;
  using N = Num<S>;
  using Key = typename N::Key;
  __shared__ Key s_key[LP_LIST];
  __shared__ uint32_t s_at[LP_LIST];
  __shared__ Key b_key[CL > 1 ? B200_TOP_MAX : 1];  // the block's alternatives, in order
  __shared__ uint32_t b_at[CL > 1 ? B200_TOP_MAX : 1];
  __shared__ Share<S> s_share[16], b_share;
  __shared__ Key b_bound;
  __shared__ uint32_t s_warp[16];
  __shared__ uint32_t s_count, s_parts;
  __shared__ uint16_t s_who[512];
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const long long row = blockIdx.x / CL;
  const int part = CL > 1 ? (int)(blockIdx.x % CL) : 0;
  const T *x = a.x + row * a.ldx;
  // the row: `head` values, nvec vectors, `rest` values; the block's part of the vectors is [v0, v1), the first part
  // has the head and the last one the rest
  const int vocab = (int)a.vocab;
  const int head = V > 1 ? min(vocab, (int)(((V * sizeof(T) - (uintptr_t)x % (V * sizeof(T))) % (V * sizeof(T))) / sizeof(T))) : 0;
  const int nvec = (vocab - head) / V, rest = vocab - head - nvec * V;
  const int v0 = (int)((long long)nvec * part / CL), v1 = (int)((long long)nvec * (part + 1) / CL);
  const bool has_head = part == 0 && tid < head, has_rest = part == CL - 1 && tid < rest;
  const Pack<T, V> *xv = reinterpret_cast<const Pack<T, V> *>(x + head);
  if (tid == 0) s_count = s_parts = 0;

  S target = 0;
  long long token = B200_NO_TOKEN;
  if (tid == 0 && part == 0 && a.targets) {
    token = a.targets[row];
    if (token >= 0 && token < vocab) target = widen_logit(x[token]);
  }

  Share<S> sh;
  auto take = [&](S v) {
    if (v > sh.m) sh.raise(v);
    sh.add(v);
  };
  if (has_head) take(widen_logit(x[tid]));
  if (has_rest) take(widen_logit(x[vocab - rest + tid]));
  constexpr int U = sizeof(T) * V >= 16 ? 4 : 8;
  int i = v0 + tid;
  for (; i + (U - 1) * nt < v1; i += U * nt) {
    Pack<T, V> b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) b[u] = xv[i + u * nt];
    S top = -(S)INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmax(top, widen_logit(b[u].v[j]));
    if (top > sh.m) sh.raise(top);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) sh.add(widen_logit(b[u].v[j]));
  }
  for (; i < v1; i += nt) {
    const Pack<T, V> b = xv[i];
    S top = widen_logit(b.v[0]);
#pragma unroll
    for (int j = 1; j < V; ++j) top = fmax(top, widen_logit(b.v[j]));
    if (top > sh.m) sh.raise(top);
#pragma unroll
    for (int j = 0; j < V; ++j) sh.add(widen_logit(b.v[j]));
  }
  const S own_max = sh.m;

  // ---- join the sums: lanes, then warps (by the first one, which finds the bound of the alternatives too) ----
  const int n = min(a.top, (v1 - v0) * V + (part == 0 ? head : 0) + (part == CL - 1 ? rest : 0));
  sh.join_lanes();
  if (lane == 0) s_share[warp] = sh;
  if (n > 0) s_key[tid] = N::key(own_max);
  __syncthreads();
  if (warp == 0) {
    sh = lane < warps ? s_share[lane] : Share<S>();
    sh.join_lanes();
    if (lane == 0) b_share = sh;
    if (n > 0) {
      // towards the n-th largest of the threads' maxima, bit by bit from the first that they differ in, until a bound
      // is found that n threads reach, and not many more
      Key k[16], most = 0, least = ~(Key)0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        k[j] = j < warps ? s_key[j * 32 + lane] : 0;
        most = max(most, k[j]);
        if (j < warps) least = min(least, k[j]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      }
      constexpr int BITS = (int)sizeof(Key) * 8;
      const int same = most == least ? BITS : (BITS == 64 ? __clzll((long long)(most ^ least)) : __clz((int)(most ^ least)));
      Key bound = same == BITS ? most : most & ~(~(Key)0 >> same);
      for (int bit = BITS - 1 - same; bit >= 0; --bit) {
        const Key trial = bound | ((Key)1 << bit);
        int reach = 0;
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          reach += ((k[j] >= trial) + (k[j + 1] >= trial)) + ((k[j + 2] >= trial) + (k[j + 3] >= trial));
        reach = __reduce_add_sync(0xffffffffu, reach);
        if (reach >= n) bound = trial;
        if (reach >= n && reach <= 2 * n + 8) break;
      }
      if (lane == 0) b_bound = bound;
    }
  }
  __syncthreads();
  sh = b_share;
  const bool wild = sh.s != sh.s;  // of the block's part

  // ---- the block's alternatives ----
  // f(value, index) over the shares of the threads whose maximum is above the bound (or at it), by the whole block: one
  // vector of one share per thread and step. Every thread of the block calls it.
  const int per = (v1 - v0 + nt - 1) / nt;
  auto scan_shares = [&](bool takes_part, auto f) {
    if (takes_part) s_who[atomicAdd(&s_parts, 1u)] = (uint16_t)tid;
    __syncthreads();
    const int all = (int)s_parts;
    for (int c = tid; c < all * per; c += nt) {
      const int k = v0 + s_who[c / per] + c % per * nt;
      if (k >= v1) continue;
      const Pack<T, V> b = xv[k];
#pragma unroll
      for (int j = 0; j < V; ++j) f(widen_logit(b.v[j]), (uint32_t)(head + k * V + j));
    }
    if (takes_part && has_head) f(widen_logit(x[tid]), (uint32_t)tid);
    if (takes_part && has_rest) f(widen_logit(x[vocab - rest + tid]), (uint32_t)(vocab - rest + tid));
    __syncthreads();
  };
  auto push = [&](Key key, uint32_t at) {
    const uint32_t p = atomicAdd(&s_count, 1u);
    if (p < LP_LIST) {
      s_key[p] = key;
      s_at[p] = at;
    }
  };
  auto in_front = [](Key k, uint32_t i2, Key l, uint32_t j2) { return k > l || (k == l && i2 < j2); };
  // g(rank, key, index) for the first n of `count` listed candidates
  auto ranked = [&](int count, int first, auto g) {
    for (int c = tid; c < count; c += nt) {
      const Key k = s_key[c];
      const uint32_t at = s_at[c];
      int before = 0;
      for (int d = 0; d < count; ++d) before += in_front(s_key[d], s_at[d], k, at) ? 1 : 0;
      if (before < first) g(before, k, at);
    }
  };
  int listed = 0;
  if (n > 0) {
    bool search = wild;
    if (!wild) {
      const Key mine = N::key(own_max), bound = b_bound;
      scan_shares(mine >= bound, [&](S v, uint32_t at) {
        const Key k = N::key(v);
        if (k >= bound) push(k, at);
      });
      listed = (int)s_count;
      if (listed > LP_LIST) {
        // many equals: what lies above the bound, then the first equals in the order of the row
        __syncthreads();
        if (tid == 0) s_count = s_parts = 0;
        __syncthreads();
        scan_shares(mine > bound, [&](S v, uint32_t at) {
          const Key k = N::key(v);
          if (k > bound) push(k, at);
        });
        listed = (int)s_count;
        search = listed > LP_LIST;
        int missing = search ? 0 : n - listed;  // the same in every thread, as is what follows
        const int last = vocab - (part == CL - 1 ? 0 : rest + (nvec - v1) * V), first = part == 0 ? 0 : head + v0 * V;
        for (int at0 = first; at0 < last && missing > 0; at0 += nt) {
          const int at = at0 + tid;
          const bool eq = at < last && N::key(widen_logit(x[at])) == bound;
          const uint32_t votes = __ballot_sync(0xffffffffu, eq);
          __syncthreads();
          if (lane == 0) s_warp[warp] = __popc(votes);
          __syncthreads();
          int before = __popc(votes & ((1u << lane) - 1u)), all = 0;
          for (int w = 0; w < warps; ++w) {
            if (w < warp) before += s_warp[w];
            all += s_warp[w];
          }
          if (eq && before < missing && listed + before < LP_LIST) {
            s_key[listed + before] = bound;
            s_at[listed + before] = (uint32_t)at;
          }
          listed += min(all, missing);
          missing -= min(all, missing);
        }
        __syncthreads();
      }
    }
    if (search) {
      // one search per alternative for what comes behind the last one
      Key last_k = 0;
      uint32_t last_at = 0;
      for (int r = 0; r < n; ++r) {
        Key best = 0;
        uint32_t best_at = UINT_MAX;
        auto see = [&](Key k, uint32_t at) {
          if ((r == 0 || in_front(last_k, last_at, k, at)) && (best_at == UINT_MAX || in_front(k, at, best, best_at))) {
            best = k;
            best_at = at;
          }
        };
        if (has_head) see(N::key(widen_logit(x[tid])), (uint32_t)tid);
        if (has_rest) see(N::key(widen_logit(x[vocab - rest + tid])), (uint32_t)(vocab - rest + tid));
        for (int k = v0 + tid; k < v1; k += nt) {
          const Pack<T, V> b = xv[k];
#pragma unroll
          for (int j = 0; j < V; ++j) see(N::key(widen_logit(b.v[j])), (uint32_t)(head + k * V + j));
        }
        __syncthreads();
        s_key[tid] = best;
        s_at[tid] = best_at;
        __syncthreads();
        best_at = UINT_MAX;
        for (int c = 0; c < nt; ++c)
          if (s_at[c] != UINT_MAX) see(s_key[c], s_at[c]);
        last_k = best;
        last_at = best_at;
        __syncthreads();
        if (tid == 0) {
          s_key[LP_LIST - B200_TOP_MAX + r] = best;
          s_at[LP_LIST - B200_TOP_MAX + r] = best_at;
        }
        __syncthreads();
      }
      if (tid < n) {
        s_key[tid] = s_key[LP_LIST - B200_TOP_MAX + tid];
        s_at[tid] = s_at[LP_LIST - B200_TOP_MAX + tid];
      }
      __syncthreads();
      listed = n;
    }
  }

  // ---- the cluster's parts ----
  if constexpr (CL > 1) {
    ranked(listed, n, [&](int r, Key k, uint32_t at) {
      b_key[r] = k;
      b_at[r] = at;
    });
    __syncthreads();
    ptx::cluster_sync();
    if (part == 0) {
      auto cluster = cooperative_groups::this_cluster();
      for (int c = 1; c < CL; ++c) {
        const Share<S> *o = cluster.map_shared_rank(&b_share, c);
        sh.join(o->m, o->o, o->s, o->t);
      }
      // every part has at least `top` values (the launch sees to it)
      for (int c = tid; c < CL * n; c += nt) {
        s_key[c] = *cluster.map_shared_rank(&b_key[c % n], c / n);
        s_at[c] = *cluster.map_shared_rank(&b_at[c % n], c / n);
      }
      listed = CL * n;
      __syncthreads();
    }
    ptx::cluster_sync();  // no block leaves while another may read it
    if (part != 0) return;
  }

  const S nan = (S)NAN, inf = (S)INFINITY;
  const bool odd = sh.s != sh.s;
  const S log_s = sh.s > S(0) ? log(sh.s) : S(0);
  auto log_prob = [&](S v) { return odd ? nan : sh.s > S(0) ? (v - sh.m) - log_s : -inf; };
  if (tid == 0) {
    if (a.lse) a.lse[row] = odd ? nan : sh.s > S(0) ? sh.m + log_s : -inf;
    if (a.entropy) a.entropy[row] = odd ? nan : sh.s > S(0) ? N::entropy(sh.s, sh.t) : S(0);
    if (a.targets) {
      if (token >= 0 && token < vocab) {
        a.logp[row] = log_prob(target);
      } else {
        a.logp[row] = token == B200_NO_TOKEN ? S(0) : nan;
        if (token != B200_NO_TOKEN) atomicExch(a.bad, 1);
      }
    }
  }
  ranked(listed, a.top, [&](int r, Key k, uint32_t at) {
    a.top_logp[row * a.top + r] = log_prob(N::value(k));
    a.top_index[row * a.top + r] = at;
  });
}

// dx = -p (g + h (ln p + H)) + g delta, p = e^(x - lse): elementwise, bound by HBM (a row read, a row written).
template <typename T>
struct LogprobBwdArgs {
  using S = typename LogitTraits<T>::Stat;
  const T *x;
  long long ldx, vocab;
  const long long *targets;
  const S *lse, *entropy, *grad_logp, *grad_entropy;
  T *dx;
  long long lddx;
  int *bad;
};
__device__ __forceinline__ float gradient_of(float x, float lse, float ent, float g, float h) {
  const float lp = x - lse;
  return -(ex2(lp * LOG2E) * fmaf(h, fmaxf(lp, -1e4f) + ent, g));
}
__device__ __forceinline__ double gradient_of(double x, double lse, double ent, double g, double h) {
  const double lp = x - lse;
  return -(exp(lp) * fma(h, fmax(lp, -1e4) + ent, g));
}

// `parts` blocks per row, each with a share of its vectors (V values: 16 bytes where x and dx lie alike, else one).
template <typename T, int V>
__global__ void __launch_bounds__(512) token_logprobs_bwd_kernel(const LogprobBwdArgs<T> a, int parts) {
  ptx::grid_begin();
  using S = typename LogitTraits<T>::Stat;
  const int tid = threadIdx.x, nt = blockDim.x, vocab = (int)a.vocab;
  const long long row = blockIdx.x / parts, token = a.targets[row];
  const int part = (int)(blockIdx.x % parts);
  const T *x = a.x + row * a.ldx;
  T *dx = a.dx + row * a.lddx;
  const int head = V > 1 ? min(vocab, (int)(((V * sizeof(T) - (uintptr_t)x % (V * sizeof(T))) % (V * sizeof(T))) / sizeof(T))) : 0;
  const int nvec = (vocab - head) / V, rest = vocab - head - nvec * V;
  const int v0 = (int)((long long)nvec * part / parts), v1 = (int)((long long)nvec * (part + 1) / parts);
  const bool inside = token >= 0 && token < vocab;
  if (!inside && token != B200_NO_TOKEN && tid == 0 && part == 0) atomicExch(a.bad, 1);
  const S g = inside ? a.grad_logp[row] : S(0), h = a.grad_entropy ? a.grad_entropy[row] : S(0);
  const bool none = g == S(0) && h == S(0);
  const S lse = none ? S(0) : a.lse[row], ent = h != S(0) ? a.entropy[row] : S(0);
  const int at = inside ? (int)token : -1;
  const Pack<T, V> *xv = reinterpret_cast<const Pack<T, V> *>(x + head);
  Pack<T, V> *dv = reinterpret_cast<Pack<T, V> *>(dx + head);
  auto store = [](S v) -> T {
    if constexpr (sizeof(T) == 8) return v;
    else return narrow_logit<T>((float)v);
  };
  if (none || lse == -(S)INFINITY) {
    if (part == 0 && tid < head) dx[tid] = store(S(0));
    if (part == parts - 1 && tid < rest) dx[vocab - rest + tid] = store(S(0));
    Pack<T, V> zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = store(S(0));
    for (int i = v0 + tid; i < v1; i += nt) dv[i] = zero;
    return;
  }
  auto one = [&](int i) { dx[i] = store(gradient_of(widen_logit(x[i]), lse, ent, g, h) + (i == at ? g : S(0))); };
  if (part == 0 && tid < head) one(tid);
  if (part == parts - 1 && tid < rest) one(vocab - rest + tid);
  auto many = [&](int i, const Pack<T, V> &b) {
    S d[V];
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = gradient_of(widen_logit(b.v[j]), lse, ent, g, h);
    const unsigned hit = (unsigned)(at - head - i * V);
    if (hit < (unsigned)V) {
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] += j == (int)hit ? g : S(0);
    }
    Pack<T, V> out;
#pragma unroll
    for (int j = 0; j < V; ++j) out.v[j] = store(d[j]);
    dv[i] = out;
  };
  constexpr int U = 4;
  int i = v0 + tid;
  for (; i + (U - 1) * nt < v1; i += U * nt) {
    Pack<T, V> b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) b[u] = xv[i + u * nt];
#pragma unroll
    for (int u = 0; u < U; ++u) many(i + u * nt, b[u]);
  }
  for (; i < v1; i += nt) many(i, xv[i]);
}

// Threads per row: sixteen vectors each, one warp at least.
static int row_threads(long long nvec, int most) {
  int nt = 32;
  while (nt < most && nt * 16 < nvec) nt *= 2;
  return nt;
}

template <typename T, int V, int CL>
static void launch_forward_as(b200_engine *e, const LogprobArgs<T> &a, long long rows, int nt) {
  auto kern = token_logprobs_kernel<T, V, CL>;
  if (CL == 1) {
    launch_kernel(e, kern, (unsigned)rows, nt, 0, a);
    return;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // as launch_kernel does
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * CL));
  cfg.blockDim = dim3((unsigned)nt);
  cfg.stream = e->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T>
static int launch_forward(b200_engine *e, const void *x, long long ldx, long long rows, long long vocab, const int64_t *targets,
                          void *logp, void *entropy, void *lse, int top, void *top_logp, int64_t *top_index) {
  using S = typename LogitTraits<T>::Stat;
  constexpr int V = 16 / sizeof(T);
  const LogprobArgs<T> a{(const T *)x, ldx, vocab, (const long long *)targets, (S *)logp, (S *)entropy, (S *)lse, top,
                         (S *)top_logp, (long long *)top_index, e->d_flags + 4};
  if (vocab < 256) {  // a few values per thread: not worth the heads and tails of vectors
    launch_forward_as<T, 1, 1>(e, a, rows, 32);
  } else {
    const long long nvec = vocab / V;
    // Few rows are shared by clusters, as long as a block keeps two vectors for each of its threads; with as many threads
    // as a block can have, since nothing else runs on their SMs. Many rows have blocks of 256, five to an SM: what
    // one of them waits for (its sums' joining, its alternatives) passes behind the others' loads. 4096 x 32000 with
    // 5 alternatives: blocks of 512 111 us (bf16 83), 256 100 (72), 128 109 (64).
    int cl = 1, nt = row_threads(nvec, 512);
    while (cl < 8 && rows * cl < e->sm_count && nvec / (2 * cl) >= 2 * nt) cl *= 2;
    if (cl == 1) nt = row_threads(nvec, 256);
    if (cl == 8) launch_forward_as<T, V, 8>(e, a, rows, nt);
    else if (cl == 4) launch_forward_as<T, V, 4>(e, a, rows, nt);
    else if (cl == 2) launch_forward_as<T, V, 2>(e, a, rows, nt);
    else launch_forward_as<T, V, 1>(e, a, rows, nt);
  }
  B200_CHECK_LAUNCH(e, "token_logprobs_kernel");
  return B200_OK;
}

template <typename T>
static int launch_backward(b200_engine *e, const void *x, long long ldx, long long rows, long long vocab, const int64_t *targets,
                           const void *lse, const void *entropy, const void *grad_logp, const void *grad_entropy, void *dx,
                           long long lddx) {
  using S = typename LogitTraits<T>::Stat;
  constexpr int V = 16 / sizeof(T);
  const LogprobBwdArgs<T> a{(const T *)x, ldx, vocab, (const long long *)targets, (const S *)lse, (const S *)entropy,
                            (const S *)grad_logp, (const S *)grad_entropy, (T *)dx, lddx, e->d_flags + 4};
  // vectors where the rows of x and dx lie alike to 16-byte boundaries
  const bool alike = ((uintptr_t)x - (uintptr_t)dx) % 16 == 0 && (ldx - lddx) * (long long)sizeof(T) % 16 == 0;
  const long long nvec = alike && vocab >= 256 ? vocab / V : vocab;
  const int nt = row_threads(nvec, 512);
  const long long parts = std::max<long long>(1, std::min<long long>((2LL * e->sm_count + rows - 1) / rows, nvec / (4 * nt)));
  if (rows * parts >= (1LL << 31))
    return set_error(e, B200_ERR_UNSUPPORTED, "b200_token_logprobs_bwd: %lld rows are more than one launch takes", rows);
  if (alike && vocab >= 256) launch_kernel(e, token_logprobs_bwd_kernel<T, V>, (unsigned)(rows * parts), nt, 0, a, (int)parts);
  else launch_kernel(e, token_logprobs_bwd_kernel<T, 1>, (unsigned)(rows * parts), nt, 0, a, (int)parts);
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
  B200_REQUIRE(e, rows >= 0 && vocab >= 1 && rows < (1LL << 31) && vocab <= (1LL << 30), "b200_token_logprobs: bad extent");
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
  B200_REQUIRE(e, rows >= 0 && vocab >= 1 && rows < (1LL << 31) && vocab <= (1LL << 30), "b200_token_logprobs_bwd: bad extent");
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

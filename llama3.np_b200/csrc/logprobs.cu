// Log probabilities of given tokens, with the distribution's entropy and its most likely tokens (L3TokenLogprobs).  With m = max x, d = x - m:
//   S = sum e^d,  log p_t = d_t - log S,  H = - sum p log p = log S - (sum d e^d) / S
// (both terms of H are 0 or more: no difference of near equals where one token has nearly all).
//
// Bound by the logits, read once.  A row is a CTA's, or of few rows a cluster's, whose CTAs meet over shared memory.  A thread streams
// 16-byte pieces with a running maximum and sums of its own.  The n most likely: the n-th largest of the threads' maxima - found bit by bit, a
// count over the CTA a time - bounds the n-th largest logit from below, so only the few threads whose maximum passes it look at their logits
// again (a warp together at one thread's, 32 pieces at a time), and what passes is ranked by counting.  Where more values pass than there is room
// for (many equal ones), the n are drawn one after the other.
#include <float.h>
#include <math.h>

#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "packed.h"

namespace {
constexpr int LT = 512, LW = LT / 32;
constexpr int ROOM = 512;  // values that pass a CTA's bound

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t order_key(float v) {  // larger values, larger keys; both zeros alike
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr uint32_t NO_KEY = 0x007fffffu;  // that of -infinity
// a value with its place: the larger value first, then the lower place
__device__ __forceinline__ unsigned long long entry(uint32_t key, int v) { return (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)v); }

template <typename T> __device__ __forceinline__ float value(const T* p) { return to_f32(*p); }
template <> __device__ __forceinline__ float value<__half>(const __half* p) { return __half2float(*p); }
template <typename T> struct Piece {  // 16 bytes of a row
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void again(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void values(float (&x)[N]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 4) x[i] = __uint_as_float(u[i]);
      else if constexpr (std::is_same<T, bf16>::value) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};
struct Sums { float m, s, t; };  // largest logit, sum e^(x - m), sum (x - m) e^(x - m)
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m), from = m == -INFINITY ? 0.f : m;
  const float da = a.m == -INFINITY ? 0.f : a.m - from, db = b.m == -INFINITY ? 0.f : b.m - from;
  const float fa = ex2(da * 1.4426950408889634f), fb = ex2(db * 1.4426950408889634f);
  // a side at -infinity has sums 0, or NaN of a NaN; one too far down for its factor may have s d = -infinity
  return Sums{m, a.s * fa + b.s * fb, (fa > 0.f ? (a.t + a.s * da) * fa : 0.f) + (fb > 0.f ? (b.t + b.s * db) * fb : 0.f)};
}
template <bool ENTROPY, int N> __device__ __forceinline__ void take(Sums& a, const float (&x)[N]) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > a.m) {
    const float d = a.m == -INFINITY ? 0.f : a.m - top, f = ex2(d * 1.4426950408889634f);
    if (ENTROPY) a.t = f > 0.f ? (a.t + a.s * d) * f : 0.f;
    a.s *= f;
    a.m = top;
  }
  const float from = a.m == -INFINITY ? 0.f : a.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the difference first and by itself: a logit's own multiple of log2 e would be off by more than the difference's
    const float d = x[i] - from, e = ex2(d * 1.4426950408889634f);
    a.s += e;
    if (ENTROPY) a.t += e * fmaxf(d, -FLT_MAX);  // 0 for a logit of -infinity
  }
}

// A cluster of S CTAs (gridDim.x = S) has a row; its CTA c the pieces c, c + S, ... of LT threads' pieces each.
template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(LT, TOP ? 2 : 3) logprobs_kernel(const LogprobsArgs a) {
  constexpr int N = Piece<T>::N;
  __shared__ Sums parts[LW];
  __shared__ Sums cta_sums;
  __shared__ unsigned long long hits[TOP ? ROOM : 1], best[TOP ? LOGPROBS_MAX_TOP : 1];
  __shared__ int count;
  __shared__ unsigned long long draw[LW];
  pdl_launch();
  pdl_wait();
  const int S = gridDim.x, c = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x0 = (const T*)a.logits + row * a.stride;
  const int token = a.tokens[row];
  // logits ahead of the first whole piece, pieces, logits behind the last; those at the ends are the first threads' of CTA 0
  const int ahead = min((int)((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)), a.V), pieces = (a.V - ahead) / N, behind = a.V - ahead - pieces * N;
  const T* xp = x0 + ahead;
  const int ends = c == 0 && (int)threadIdx.x < ahead + behind ? (int)threadIdx.x + ((int)threadIdx.x < ahead ? 0 : pieces * N) : -1;
  Sums my{-INFINITY, 0.f, 0.f};
  const int first = c * LT + threadIdx.x, step = S * LT;
  {
    constexpr int AHEAD = 4;
    Piece<T> p[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (first + i * step < pieces) p[i].load(xp + (size_t)(first + i * step) * N);
    for (int at = first; at < pieces; at += AHEAD * step) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (at + i * step < pieces) {
          float x[N];
          p[i].values(x);
          if (at + (i + AHEAD) * step < pieces) p[i].load(xp + (size_t)(at + (i + AHEAD) * step) * N);
          take<ENTROPY>(my, x);
        }
      }
    }
    if (ends >= 0) {
      const float x[1] = {value(x0 + ends)};
      take<ENTROPY>(my, x);
    }
  }
  const float most = my.m;  // of this thread
#pragma unroll
  for (int o = 16; o; o >>= 1)
    my = joined(my, Sums{__shfl_xor_sync(L3_FULL, my.m, o), __shfl_xor_sync(L3_FULL, my.s, o), __shfl_xor_sync(L3_FULL, my.t, o)});
  if (lane == 0) parts[warp] = my;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  if (warp == 0) {
    my = parts[lane & (LW - 1)];
#pragma unroll
    for (int o = LW / 2; o; o >>= 1)
      my = joined(my, Sums{__shfl_xor_sync(L3_FULL, my.m, o), __shfl_xor_sync(L3_FULL, my.s, o), __shfl_xor_sync(L3_FULL, my.t, o)});
    if (lane == 0) cta_sums = my;
  }
  if constexpr (TOP) {
    const int n = a.n;
    // the largest key that at least n threads' maxima reach (of the first 20 bits: it is a bound only); none: every finite logit passes
    const uint32_t mine = order_key(most);
    uint32_t bound = 0;
    for (int bit = 31; bit >= 12; --bit) {
      const uint32_t with = bound | 1u << bit;
      if (__syncthreads_count(most > -INFINITY && mine >= with) >= n) bound = with;
    }
    bound = max(bound, NO_KEY + 1);
    auto offer = [&](float x, int v) {
      const uint32_t key = order_key(x);
      if (x > -INFINITY && key >= bound) {  // NaN is none
        const int at = atomicAdd(&count, 1);
        if (at < ROOM) hits[at] = entry(key, v);
      }
    };
    for (uint32_t who = __ballot_sync(L3_FULL, most > -INFINITY && mine >= bound); who; who &= who - 1) {
      const int of = __ffs(who) - 1, its_first = c * LT + warp * 32 + of, its_ends = __shfl_sync(L3_FULL, ends, of);
      for (int at = its_first + lane * step; at < pieces; at += 32 * step) {
        Piece<T> p;
        p.again(xp + (size_t)at * N);
        float x[N];
        p.values(x);
#pragma unroll
        for (int e = 0; e < N; ++e) offer(x[e], ahead + at * N + e);
      }
      if (lane == 0 && its_ends >= 0) offer(value(x0 + its_ends), its_ends);
    }
    __syncthreads();
    const int found = count;
    if (found <= ROOM) {
      for (int i = threadIdx.x; i < n; i += LT) best[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < found; i += LT) {
        const unsigned long long me = hits[i];
        int rank = 0;
        for (int j = 0; j < found; ++j) rank += hits[j] > me;
        if (rank < n) best[rank] = me;
      }
    } else {
      unsigned long long last = ~0ull;  // the one drawn before
      for (int i = 0; i < n; ++i) {
        unsigned long long top = 0;
        auto look = [&](float x, int v) {
          const unsigned long long e = entry(order_key(x), v);
          if (x > -INFINITY && e < last && e > top) top = e;
        };
        for (int at = first; at < pieces; at += step) {
          Piece<T> p;
          p.again(xp + (size_t)at * N);
          float x[N];
          p.values(x);
#pragma unroll
          for (int e = 0; e < N; ++e) look(x[e], ahead + at * N + e);
        }
        if (ends >= 0) look(value(x0 + ends), ends);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(L3_FULL, top, o);
          top = other > top ? other : top;
        }
        __syncthreads();
        if (lane == 0) draw[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < LW; ++w) top = draw[w] > top ? draw[w] : top;
        if (threadIdx.x == 0) best[i] = top;
        last = top;
      }
    }
  }
  // the cluster's CTAs meet in the first one
  Sums all;
  if (S > 1) {
    cluster_sync_all();
    if (c == 0) {
      all = cta_sums;
      for (int o = 1; o < S; ++o) {
        const uint32_t at = cluster_at((uint32_t)__cvta_generic_to_shared(&cta_sums), o);
        Sums other;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.m) : "r"(at) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.s) : "r"(at + 4) : "memory");
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other.t) : "r"(at + 8) : "memory");
        all = joined(all, other);
      }
      if constexpr (TOP) {
        for (int i = threadIdx.x; i < S * a.n; i += LT) {
          const uint32_t at = cluster_at((uint32_t)__cvta_generic_to_shared(&best[i % a.n]), i / a.n);
          asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(hits[i]) : "r"(at) : "memory");
        }
      }
    }
    cluster_sync_all();
    if (c) return;
    if constexpr (TOP) {
      for (int i = threadIdx.x; i < a.n; i += LT) best[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < S * a.n; i += LT) {
        const unsigned long long me = hits[i];
        int rank = 0;
        for (int j = 0; j < S * a.n; ++j) rank += hits[j] > me;
        if (me && rank < a.n) best[rank] = me;
      }
    }
    __syncthreads();
  } else {
    __syncthreads();
    all = cta_sums;
  }
  const float log_s = logf(all.s);
  const bool none = all.m == -INFINITY && !(all.s != all.s);  // no token has a probability
  if (threadIdx.x == 0) {
    float lp = 0.f;
    if (token >= a.V) lp = NAN;
    else if (token >= 0) lp = none ? -INFINITY : value(x0 + token) - all.m - log_s;
    a.out_logprobs[row] = lp;
    if (ENTROPY && a.out_entropy) a.out_entropy[row] = none ? 0.f : log_s - all.t / all.s;
  }
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < a.n; i += LT) {
      const unsigned long long e = best[i];
      a.out_top[(size_t)row * a.n + i] = e ? key_value((uint32_t)(e >> 32)) - all.m - log_s : -INFINITY;
      a.out_top_tokens[(size_t)row * a.n + i] = e ? (int)(0xffffffffu - (uint32_t)e) : -1;
    }
  }
}
template <typename T, bool ENTROPY, bool TOP> cudaError_t launch_tt(const LogprobsArgs& a, int n_sm, cudaStream_t s) {
  // a cluster's CTAs: as many as fill the SMs, if each has a piece for every thread
  int S = 1;
  while (S < 8 && (long long)a.R * S * 2 <= 2LL * n_sm && (long long)a.V >= (long long)S * 2 * LT * Piece<T>::N) S *= 2;
  for (int row = 0; row < a.R; row += 65535) {
    LogprobsArgs b = a;
    b.R = min(a.R - row, 65535);
    b.logits = (const T*)a.logits + row * a.stride;
    b.tokens += row; b.out_logprobs += row;
    if (b.out_entropy) b.out_entropy += row;
    if (TOP) { b.out_top += (size_t)row * a.n; b.out_top_tokens += (size_t)row * a.n; }
    const cudaError_t e = launch_kc(logprobs_kernel<T, ENTROPY, TOP>, dim3(S, b.R), dim3(LT), 0, s, S, b);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
template <typename T> cudaError_t launch_t(const LogprobsArgs& a, int n_sm, cudaStream_t s) {
  if (a.n) return a.out_entropy ? launch_tt<T, true, true>(a, n_sm, s) : launch_tt<T, false, true>(a, n_sm, s);
  return a.out_entropy ? launch_tt<T, true, false>(a, n_sm, s) : launch_tt<T, false, false>(a, n_sm, s);
}
}  // namespace

cudaError_t launch_token_logprobs(const LogprobsArgs& a, int n_sm, cudaStream_t s) {
  if (a.dtype == L3_DTYPE_F32) return launch_t<float>(a, n_sm, s);
  if (a.dtype == L3_DTYPE_BF16) return launch_t<bf16>(a, n_sm, s);
  return launch_t<__half>(a, n_sm, s);
}

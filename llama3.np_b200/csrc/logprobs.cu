// Log probabilities of given tokens, with the distribution's entropy and its most likely tokens (L3TokenLogprobs).  With d = x - m, for any m:
//   S = sum e^d,  log p_t = d_t - log S,  H = - sum p log p = log S - (sum d e^d) / S
// m lies at most 1 below the largest logit (LAG): where one token has nearly all, what is subtracted from log S is no larger than 1, and the
// result as good as fp32 has 1, not m's distance.
//
// Bound by the logits, read once.  A row is a CTA's, or of few rows a cluster's, whose CTAs meet over shared memory.  A thread streams
// 16-byte pieces with a running maximum and sums of its own.  The n most likely: the threads' maxima
// bound the n-th largest logit from below, so only the few threads whose maximum passes the bound look at their logits
// again (a warp together at one thread's, 32 pieces at a time), and what passes is ranked by counting.  Where more values pass than there is room
// for, a better bound is found; where that does not help (many equal ones), the n are drawn one after the other.
//
// 2047 rows of 128256 in bf16 with entropy: 99.8 us, 5.3 TB/s (81 % of a copy's rate) at 74 % of the issue slots: an exponential and five other
// instructions a logit.  48 rows in fp32 with entropy and 20 tokens: 16.5 us, 7.3 without the tokens, whose ranking is a chain of barriers.
#include <float.h>
#include <math.h>

#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "packed.h"

namespace {
constexpr int LT = 512, LW = LT / 32;
// How far a logit may pass m before the sums move to it.  us, 2047 rows of 128256 in bf16 with entropy, 1 : 2 : 8: 99.8 : 99.6 : 98.9; but with 8 a
// token of probability 0.997 had its log p, -0.003, off by 4e-7, with 1 by 6e-8, the rounding of 1.
constexpr float LAG = 1.f;
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
  __device__ __forceinline__ float most() const {  // 16-bit values two at a time; NaN is none
    if constexpr (N == 4) return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
    else {
      using T2 = typename std::conditional<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>::type;
      const T2 *a = reinterpret_cast<const T2*>(&w.x), *b = reinterpret_cast<const T2*>(&w.y), *c = reinterpret_cast<const T2*>(&w.z),
               *d = reinterpret_cast<const T2*>(&w.w);
      const T2 m = __hmax2(__hmax2(*a, *b), __hmax2(*c, *d));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
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
struct Sums { float m, s, t; };  // a logit, sum e^(x - m), sum (x - m) e^(x - m)
// sums against another logit, none of the row's beyond it by much
__device__ __forceinline__ Sums moved(const Sums& a, float m) {
  const float from = m == -INFINITY ? 0.f : m, d = a.m == -INFINITY ? 0.f : a.m - from, f = ex2(d * 1.4426950408889634f);
  // a side at -infinity has sums 0, or NaN of a NaN; one too far down for its factor may have s d = -infinity
  return Sums{m, a.s * f, f > 0.f ? (a.t + a.s * d) * f : 0.f};
}
// of the N neighbouring lanes (the least of them the whole one's)
template <int N> __device__ __forceinline__ Sums joined(Sums a) {
  const uint32_t key = __reduce_max_sync(L3_FULL, order_key(a.m));
  a = moved(a, key > NO_KEY ? key_value(key) : -INFINITY);
#pragma unroll
  for (int o = N / 2; o; o >>= 1) {
    a.s += __shfl_xor_sync(L3_FULL, a.s, o);
    a.t += __shfl_xor_sync(L3_FULL, a.t, o);
  }
  return a;
}
// how many of the n entries at `list` (shared memory, 16-byte aligned, one of 0 behind an odd number) are larger
__device__ __forceinline__ int larger(const unsigned long long* list, int n, unsigned long long me) {
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < n; j += 2) {
    const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(list + j);
    rank += (x.x > me) + (x.y > me);
  }
  return rank;
}
__device__ __forceinline__ float2 pair(float x, float y) { return make_float2(x, y); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(d) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
// More values, the largest of them `top`.  m follows the largest lazily: some lane of a warp has a new largest value in nearly every piece, and would
// move its sums each time.
template <bool ENTROPY, int N> __device__ __forceinline__ void take(Sums& a, const float (&x)[N], float top) {
  if (top > a.m + LAG) {
    const float d = a.m == -INFINITY ? 0.f : a.m - top, f = ex2(d * 1.4426950408889634f);
    if (ENTROPY) a.t = f > 0.f ? (a.t + a.s * d) * f : 0.f;
    a.s *= f;
    a.m = top;
  }
  const float from = a.m == -INFINITY ? 0.f : a.m;
  // the difference first and by itself: a logit's own multiple of log2 e would be off by more than the difference's
  if constexpr (N == 1) {
    const float d = x[0] - from, e = ex2(d * 1.4426950408889634f);
    a.s += e;
    if (ENTROPY) a.t += e * fmaxf(d, -FLT_MAX);  // 0 for a logit of -infinity
  } else {
    const float2 one = pair(1.f, 1.f), down = pair(-from, -from), log2e = pair(1.4426950408889634f, 1.4426950408889634f);
    float2 s = pair(0.f, 0.f), t = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 d = fma2(pair(x[i], x[i + 1]), one, down), y = mul2(d, log2e), e = pair(ex2(y.x), ex2(y.y));
      s = fma2(e, one, s);
      if (ENTROPY) t = fma2(e, pair(fmaxf(d.x, -FLT_MAX), fmaxf(d.y, -FLT_MAX)), t);
    }
    a.s += s.x + s.y;
    if (ENTROPY) a.t += t.x + t.y;
  }
}

// A cluster of S CTAs (gridDim.x = S) has a row; its CTA c the pieces c, c + S, ... of LT threads' pieces each.
template <typename T, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(LT, 2) logprobs_kernel(const LogprobsArgs a) {
  constexpr int N = Piece<T>::N;
  __shared__ Sums parts[LW];
  __shared__ Sums gathered[8];  // of the cluster's CTAs, in the first one's; its own ones in the others'
  __shared__ __align__(16) unsigned long long hits[TOP ? ROOM : 1], best[TOP ? 8 * LOGPROBS_MAX_TOP : 1], chosen[TOP ? LOGPROBS_MAX_TOP : 1];  // best: likewise
  __shared__ int count;
  __shared__ unsigned long long draw[LW];
  __shared__ uint32_t kths[LW];
  const int S = gridDim.x;
  if (S > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // has begun
  pdl_launch();
  pdl_wait();
  const int  c = blockIdx.x, row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x0 = (const T*)a.logits + row * a.stride;
  const int token = a.tokens[row];
  // logits ahead of the first whole piece, pieces, logits behind the last; those at the ends are the first threads' of CTA 0
  const int ahead = min((int)((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)), a.V), pieces = (a.V - ahead) / N, behind = a.V - ahead - pieces * N;
  const T* xp = x0 + ahead;
  const int ends = c == 0 && (int)threadIdx.x < ahead + behind ? (int)threadIdx.x + ((int)threadIdx.x < ahead ? 0 : pieces * N) : -1;
  Sums my{-INFINITY, 0.f, 0.f};
  const int first = c * LT + threadIdx.x, step = S * LT;
  float most = -INFINITY;  // of this thread
  {
    constexpr int AHEAD = 4;
    const int mine = first < pieces ? (pieces - first + step - 1) / step : 0;  // pieces of this thread
    const T* at = xp + (size_t)first * N;
    const size_t apart = (size_t)step * N;
    Piece<T> p[AHEAD];
    auto use = [&](Piece<T>& q, const T* next) {  // and ask for another
      float x[N];
      q.values(x);
      const float top = q.most();
      if (next) q.load(next);
      if (TOP) most = fmaxf(most, top);
      take<ENTROPY>(my, x, top);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < mine) p[i].load(at + i * apart);
    int k = 0;
    for (; k + 2 * AHEAD <= mine; k += AHEAD) {
      at += AHEAD * apart;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) use(p[i], at + i * apart);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (k + i < mine) use(p[i], k + AHEAD + i < mine ? at + (AHEAD + i) * apart : nullptr);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (k + AHEAD + i < mine) use(p[i], nullptr);
    if (ends >= 0) {
      const float x[1] = {value(x0 + ends)};
      most = fmaxf(most, x[0]);
      take<ENTROPY>(my, x, fmaxf(x[0], -INFINITY));
    }
  }
  my = joined<32>(my);
  if (lane == 0) parts[warp] = my;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  if (warp == 0) {
    my = joined<LW>(parts[lane & (LW - 1)]);
    if (lane == 0) gathered[0] = my;
  }
  if constexpr (TOP) {
    const int n = a.n;
    const uint32_t mine = order_key(most);
    // n values reach the least of the warps' k-th largest maxima, k = n over the warps
    uint32_t bound = most > -INFINITY ? mine : 0;
    {
      uint32_t left = bound, kth = 0;
      for (int k = 0; k < (n + LW - 1) / LW; ++k) {
        kth = __reduce_max_sync(L3_FULL, left);
        if (__ffs(__ballot_sync(L3_FULL, left == kth)) - 1 == lane) left = 0;
      }
      if (lane == 0) kths[warp] = kth;
    }
    __syncthreads();
    bound = kths[lane & (LW - 1)];
    bound = max(__reduce_min_sync(L3_FULL, bound), NO_KEY + 1);  // where a warp has too few, every finite logit passes
    auto offer = [&](float x, int v) {
      const uint32_t key = order_key(x);
      if (x > -INFINITY && key >= bound) {  // NaN is none
        const int at = atomicAdd(&count, 1);
        if (at < ROOM) hits[at] = entry(key, v);
      }
    };
    const int most_pieces = (pieces + step - 1) / step;  // of a thread
    auto collect = [&]() {
      uint32_t who = __ballot_sync(L3_FULL, most > -INFINITY && mine >= bound);
      while (who) {
        constexpr int TOGETHER = 4;  // threads whose pieces are on their way at once
        int of[TOGETHER];
#pragma unroll
        for (int i = 0; i < TOGETHER; ++i) {
          of[i] = who ? __ffs(who) - 1 : -1;
          who &= who - 1;
        }
        for (int at = lane; at < most_pieces; at += 32) {
          Piece<T> p[TOGETHER];
#pragma unroll
          for (int i = 0; i < TOGETHER; ++i) {
            const int piece = c * LT + warp * 32 + of[i] + at * step;
            if (of[i] >= 0 && piece < pieces) p[i].again(xp + (size_t)piece * N);
          }
#pragma unroll
          for (int i = 0; i < TOGETHER; ++i) {
            const int piece = c * LT + warp * 32 + of[i] + at * step;
            if (of[i] < 0 || piece >= pieces) continue;
            float x[N];
            p[i].values(x);
            if (order_key(p[i].most()) < bound) continue;
#pragma unroll
            for (int e = 0; e < N; ++e) offer(x[e], ahead + piece * N + e);
          }
        }
      }
      if (ends >= 0) offer(value(x0 + ends), ends);
    };
    auto refine = [&]() {  // the best bound that the threads' maxima give: the largest key that n of them reach (its first 20 bits)
      bound = 0;
      for (int bit = 31; bit >= 12; --bit) {
        const uint32_t with = bound | 1u << bit;
        if (__syncthreads_count(most > -INFINITY && mine >= with) >= n) bound = with;
      }
      bound = max(bound, NO_KEY + 1);
    };
    // a warp with too few bounds nothing: rows shorter than the threads' pieces, or banned tokens (2 rows of 3277 in bf16, 33 tokens: 7.3 us, 34 without this)
    const bool weak = bound == NO_KEY + 1;
    if (weak) refine();
    collect();
    __syncthreads();
    if (!weak && count > ROOM) {
      __syncthreads();
      if (threadIdx.x == 0) count = 0;
      refine();
      collect();
    }
    __syncthreads();
    const int found = count;
    if (found <= ROOM) {
      for (int i = threadIdx.x; i < n; i += LT) best[i] = 0;
      if (threadIdx.x == 0 && found < ROOM) hits[found] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < found; i += LT) {
        const unsigned long long me = hits[i];
        const int rank = larger(hits, found, me);
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
  __syncthreads();
  Sums all = gathered[0];
  if (S > 1) {  // the others hand theirs to the first CTA, and are done
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (c) {
      if (threadIdx.x == 0) {
        const uint32_t to = cluster_at((uint32_t)__cvta_generic_to_shared(&gathered[c]), 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(all.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(all.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(all.t) : "memory");
      }
      if constexpr (TOP) {
        if ((int)threadIdx.x < a.n)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_at((uint32_t)__cvta_generic_to_shared(&best[c * a.n + threadIdx.x]), 0)), "l"(best[threadIdx.x]) : "memory");
      }
      __syncwarp();
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (c) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int o = 1; o < S; ++o) {
      const float top = fmaxf(all.m, gathered[o].m);
      const Sums other = moved(gathered[o], top);
      all = moved(all, top);
      all.s += other.s;
      all.t += other.t;
    }
    if constexpr (TOP) {
      const int each = S * a.n;  // an even number
      for (int i = threadIdx.x; i < a.n; i += LT) chosen[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < each; i += LT) {
        const unsigned long long me = best[i];
        const int rank = larger(best, each, me);
        if (me && rank < a.n) chosen[rank] = me;
      }
      __syncthreads();
    }
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
      const unsigned long long e = (S > 1 ? chosen : best)[i];
      a.out_top[(size_t)row * a.n + i] = e ? key_value((uint32_t)(e >> 32)) - all.m - log_s : -INFINITY;
      a.out_top_tokens[(size_t)row * a.n + i] = e ? (int)(0xffffffffu - (uint32_t)e) : -1;
    }
  }
}
template <typename T, bool ENTROPY, bool TOP> cudaError_t launch_tt(const LogprobsArgs& a, int n_sm, cudaStream_t s) {
  // a cluster's CTAs: as many as fill the SMs, if each has a piece for every thread.  us, rows of 128256 in fp32 with entropy and 20 tokens, by 1 : as chosen : by 8:
  // 1 row 14.7 : 12.7 : 12.7 (8 chosen; calls differ by 0.5), 48 rows 19.3 : 16.5 : 24.5 (4), 148 rows 23.7 : 21.6 : 57.7 (2), 600 rows 100 : 100 : 225 (1)
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

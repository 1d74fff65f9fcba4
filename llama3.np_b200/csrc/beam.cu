// Beam search's selection (L3BeamSelect): the n best of
//   score(k, v) = scores[k] + logits[k, v] - log sum_u e^logits[k, u]
// over the beams k of a sequence and the vocabulary v; equal scores go to the lowest k V + v.
//
// Bound by the logits, read once.  A row is cut into slices, one CTA each, whose values stay in registers: maximum and sum of
// exponentials, and the slice's n largest logits (within a row the order of the logits is the order of the scores).  A second, dependent
// launch, one CTA per sequence, joins the sums of a row's slices in 64 bits, turns its candidates into scores - in 64 bits too, so that
// two that are close keep the order of the formula - and picks the n best.
// Both find the n largest the same way: the n-th largest of the lanes' own maxima bounds the n-th largest value from below, few values
// pass that bound, and each of those counts how many precede it.  Where more pass than there is room for (many equal values), the n
// largest are drawn one after the other.
#include <math.h>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "paged.h"

namespace {
constexpr int BT = 256, BW = BT / 32;
constexpr int ROOM = 512;  // values that pass the bound

__device__ __forceinline__ uint32_t order_key(float v) {  // larger values, larger keys; both zeros alike
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
constexpr uint32_t NO_KEY = 0x007fffffu;  // that of -infinity

// A lower bound of the warp's n-th largest key, from two values a lane (the largest of each half of what the lane has).
__device__ __forceinline__ uint32_t nth_of_warp(uint32_t a, uint32_t b, int n) {
  uint32_t t = 0;
  for (int i = 0; i < n; ++i) {
    t = __reduce_max_sync(L3_FULL, a > b ? a : b);
    if (a == t) a = 0;
    else if (b == t) b = 0;
  }
  return t;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = __reduce_max_sync(L3_FULL, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < BW; ++i) m = red[i] > m ? red[i] : m;
  return m;
}

struct RowPart { float m, s; };  // of a slice: the largest logit and the sum of e^(logit - m)

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

// part [R, S], cand_v / cand_i [R, S, n]
template <typename T, int EPT>
__global__ void __launch_bounds__(BT) beam_rows_kernel(const BeamSelectArgs a, int S, RowPart* part, float* cand_v, int* cand_i) {
  __shared__ uint32_t red[BW];
  __shared__ float sums[BW];
  __shared__ unsigned long long room[ROOM];
  __shared__ int count;
  pdl_launch();
  pdl_wait();
  const int row = blockIdx.y, slice = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = row / a.K, k = row % a.K;
  if (a.done && a.done[row]) return;  // a finished beam has one continuation, whatever its logits
  const T* x0 = (const T*)a.logits + b * a.sb + k * a.sk;
  const int base = slice * BT * EPT + tid;
  if (tid == 0) count = 0;
  float x[EPT];
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    const int v = base + i * BT;
    x[i] = v < a.V ? as_float(__ldcs(x0 + v)) : -INFINITY;
  }
  float ma = -INFINITY, mb = -INFINITY;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    if (i < EPT / 2) ma = fmaxf(ma, x[i]);
    else mb = fmaxf(mb, x[i]);
  }
  const uint32_t ka = order_key(ma), kb = order_key(mb);
  const float top = key_value(block_max(ka > kb ? ka : kb, red)), from = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < EPT; ++i) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((x[i] - from) * 1.4426950408889634f));
    sum += e;
  }
  sum = warp_sum(sum);
  if (lane == 0) sums[warp] = sum;
  const uint32_t nth = nth_of_warp(ka, kb, a.n);
  __syncthreads();  // red has been read
  uint32_t bound = block_max(nth, red);
  bound = bound > NO_KEY ? bound : NO_KEY + 1;  // -infinity is no candidate
  if (tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < BW; ++i) s += sums[i];
    part[(long long)row * S + slice] = RowPart{top, s};
  }
  // what passes the bound: key and, the lower the better, index
  if (ka >= bound || kb >= bound) {
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint32_t key = order_key(x[i]);
      if (key >= bound && x[i] == x[i]) {
        const int at = atomicAdd(&count, 1);
        if (at < ROOM) room[at] = (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)(base + i * BT));
      }
    }
  }
  __syncthreads();
  const int c = count;
  const long long out = ((long long)row * S + slice) * a.n;
  if (c <= ROOM) {
    for (int i = tid; i < c; i += BT) {
      const unsigned long long me = room[i];
      int rank = 0;
      for (int j = 0; j < c; ++j) rank += room[j] > me;
      if (rank < a.n) {
        cand_v[out + rank] = key_value((uint32_t)(me >> 32));
        cand_i[out + rank] = (int)(0xffffffffu - (uint32_t)me);
      }
    }
    for (int i = c + tid; i < a.n; i += BT) cand_i[out + i] = -1;
    return;
  }
  unsigned long long last = ~0ull;
  for (int it = 0; it < a.n; ++it) {
    unsigned long long best = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const uint32_t key = order_key(x[i]);
      const unsigned long long me = (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)(base + i * BT));
      if (key > NO_KEY && x[i] == x[i] && me < last && me > best) best = me;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long y = __shfl_xor_sync(L3_FULL, best, o);
      best = y > best ? y : best;
    }
    __syncthreads();
    if (lane == 0) room[warp] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BW; ++i) best = room[i] > best ? room[i] : best;
    last = best;
    if (tid == 0) {
      cand_v[out + it] = key_value((uint32_t)(best >> 32));
      cand_i[out + it] = best ? (int)(0xffffffffu - (uint32_t)best) : -1;
    }
  }
}

struct Scored {
  double s;
  unsigned at;  // k V + v
};
__device__ __forceinline__ bool ahead(const Scored& x, const Scored& y) { return x.s > y.s || (x.s == y.s && x.at < y.at); }

__global__ void __launch_bounds__(BT) beam_pick_kernel(const BeamSelectArgs a, int S, const RowPart* part, const float* cand_v, const int* cand_i) {
  // a beam's largest logit m and scores[k] - log sum_u e^(logit - m): apart, since logits may all be the type's lowest value
  __shared__ double add[BEAM_MAX_K];
  __shared__ float off[BEAM_MAX_K];
  __shared__ uint32_t red[BW];
  __shared__ Scored room[ROOM];
  __shared__ Scored win[BW];
  __shared__ int count;
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = S * a.n, all = a.K * per;
  if (tid == 0) count = 0;
  for (int k = warp; k < a.K; k += BW) {
    const long long row = (long long)b * a.K + k;
    const float s0 = a.scores[row];
    if (a.done && a.done[row]) {
      if (lane == 0) add[k] = s0;
      continue;
    }
    float mx = -INFINITY;
    for (int i = lane; i < S; i += 32) mx = fmaxf(mx, part[row * S + i].m);
    mx = warp_max(mx);
    const float from = mx == -INFINITY ? 0.f : mx;
    double s = 0.;
    for (int i = lane; i < S; i += 32) {
      const RowPart p = part[row * S + i];
      if (p.m > -INFINITY || p.s != p.s) s += (double)p.s * exp((double)p.m - (double)from);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(L3_FULL, s, o);
    if (lane == 0) {
      add[k] = (double)s0 - log(s);
      off[k] = from;
    }
  }
  __syncthreads();
  // candidate i: beam i / per, its slice's list; a finished beam has the end token, at its own score
  auto scored = [&](int i) {
    const int k = i / per, in = i % per;
    const long long row = (long long)b * a.K + k;
    Scored c{-INFINITY, 0};
    if (a.done && a.done[row]) {
      if (in == 0) c = Scored{add[k], (unsigned)(k * a.V + a.eos)};
    } else {
      const int v = cand_i[row * per + in];
      if (v >= 0) c = Scored{((double)cand_v[row * per + in] - (double)off[k]) + add[k], (unsigned)(k * a.V + v)};
    }
    if (!(c.s > -INFINITY) || c.s == INFINITY) c.s = -INFINITY;  // NaN, too
    return c;
  };
  // the bound on scores rounded to fp32, which keeps their order up to ties
  uint32_t ka = 0, kb = 0;
  for (int i = tid; i < all; i += BT) {
    const uint32_t key = order_key((float)scored(i).s);
    if ((i / BT) & 1) ka = key > ka ? key : ka;
    else kb = key > kb ? key : kb;
  }
  uint32_t bound = block_max(nth_of_warp(ka, kb, a.n), red);
  bound = bound > NO_KEY ? bound : NO_KEY + 1;
  for (int i = tid; i < all; i += BT) {
    const Scored c = scored(i);
    if (c.s > -INFINITY && order_key((float)c.s) >= bound) {
      const int at = atomicAdd(&count, 1);
      if (at < ROOM) room[at] = c;
    }
  }
  __syncthreads();
  auto put = [&](int place, const Scored& c) {
    const long long o = (long long)b * a.n + place;
    const int k = c.at / a.V, v = c.at % a.V;
    a.out_scores[o] = (float)c.s;
    a.out_tokens[o] = v;
    a.out_parents[o] = k;
    a.out_done[o] = (a.done && a.done[(long long)b * a.K + k]) || v == a.eos;
  };
  auto leave = [&](int place) {  // no candidate is left
    const long long o = (long long)b * a.n + place;
    a.out_scores[o] = -INFINITY;
    a.out_tokens[o] = a.eos >= 0 ? a.eos : 0;
    a.out_parents[o] = 0;
    a.out_done[o] = 1;
  };
  const int c = count;
  if (c <= ROOM) {
    for (int i = tid; i < c; i += BT) {
      const Scored me = room[i];
      int rank = 0;
      for (int j = 0; j < c; ++j) rank += ahead(room[j], me);
      if (rank < a.n) put(rank, me);
    }
    for (int i = c + tid; i < a.n; i += BT) leave(i);
    return;
  }
  Scored last{INFINITY, 0};
  for (int it = 0; it < a.n; ++it) {
    Scored best{-INFINITY, 0xffffffffu};
    for (int i = tid; i < all; i += BT) {
      const Scored x = scored(i);
      if (x.s > -INFINITY && ahead(last, x) && ahead(x, best)) best = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Scored y{__shfl_xor_sync(L3_FULL, best.s, o), __shfl_xor_sync(L3_FULL, best.at, o)};
      if (ahead(y, best)) best = y;
    }
    __syncthreads();
    if (lane == 0) win[warp] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < BW; ++i)
      if (ahead(win[i], best)) best = win[i];
    last = best;
    if (tid == 0) {
      if (best.s > -INFINITY) put(it, best);
      else leave(it);
    }
  }
}

// values of a thread: as few as still give every SM two CTAs, so that a small call ends early, and at most 32
int values_of(int rows, int V, int n_sm) {
  int ept = 32;
  while (ept > 4 && (long long)rows * ((V + BT * ept - 1) / (BT * ept)) < 2 * n_sm) ept /= 2;
  return ept;
}
template <typename T>
cudaError_t rows_of(const BeamSelectArgs& a, int ept, int S, RowPart* part, float* cv, int* ci, cudaStream_t s) {
  const dim3 g(S, a.B * a.K);
  switch (ept) {
    case 4: return launch_k(beam_rows_kernel<T, 4>, g, dim3(BT), 0, s, a, S, part, cv, ci);
    case 8: return launch_k(beam_rows_kernel<T, 8>, g, dim3(BT), 0, s, a, S, part, cv, ci);
    case 16: return launch_k(beam_rows_kernel<T, 16>, g, dim3(BT), 0, s, a, S, part, cv, ci);
    default: return launch_k(beam_rows_kernel<T, 32>, g, dim3(BT), 0, s, a, S, part, cv, ci);
  }
}
}  // namespace

size_t beam_select_workspace(int B, int K, int V, int n, int n_sm) {
  const int ept = values_of(B * K, V, n_sm);
  const size_t lists = (size_t)B * K * ((V + BT * ept - 1) / (BT * ept));
  return lists * (sizeof(RowPart) + (size_t)n * 8);
}
cudaError_t launch_beam_select(const BeamSelectArgs& a, int n_sm, cudaStream_t s) {
  const int ept = values_of(a.B * a.K, a.V, n_sm), S = (a.V + BT * ept - 1) / (BT * ept);
  const size_t lists = (size_t)a.B * a.K * S;
  RowPart* part = (RowPart*)a.ws;
  float* cv = (float*)(part + lists);
  int* ci = (int*)(cv + lists * a.n);
  cudaError_t e = a.dtype == L3_DTYPE_F32    ? rows_of<float>(a, ept, S, part, cv, ci, s)
                  : a.dtype == L3_DTYPE_BF16 ? rows_of<bf16>(a, ept, S, part, cv, ci, s)
                                             : rows_of<__half>(a, ept, S, part, cv, ci, s);
  if (e != cudaSuccess) return e;
  g_l3_pdl_next = true;
  return launch_k(beam_pick_kernel, dim3(a.B), dim3(BT), 0, s, a, S, (const RowPart*)part, (const float*)cv, (const int*)ci);
}

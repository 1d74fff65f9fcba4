// Beam search's selection (L3BeamSelect): the n best of
//   score(k, v) = scores[k] + logits[k, v] - log sum_u e^logits[k, u]
// over the beams k of a sequence and the vocabulary v; equal scores go to the lowest k V + v.
//
// Bound by the logits.  A row is cut into segments, a warp each, which the warp streams through with the next 4 KB on their way: a lane
// keeps a running maximum and sum of exponentials, and the three largest of its portions' maxima.  The n-th largest of the lanes' largest
// bounds the segment's n-th logit from below, so the few portions whose maxima pass it are looked at once more, what passes is counted off
// against the rest, and the n largest are left, in order (within a row the order of the logits is the order of the scores).  A second,
// dependent launch, one CTA per sequence, joins the sums of a row's segments in 64 bits, turns the candidates into scores - in 64 bits too, so
// that two of a row that are close keep the order of the formula - and picks the n best in the same way,
// its bound the n-th best of the segments' first candidates.  Between beams scores are as exact as their rows' sums, whose terms are fp32
// exponentials: two that are closer than 2^-19 may come in either order.
// Where more values pass a bound than there is room for, the n best are drawn one after the other: many equal ones, but also n near 64, since the
// n-th of 64 maxima bounds little then (shares of segments that do, of random logits: none up to n = 40, most at 60, all at 64).
// Measured (B200, both launches): 32 sequences of 8 beams (37 of the 256 finished), 128256 fp32 logits, 8 best: 30.9 us = 3.6 TB/s, 55 % of what a
// copy reaches (the first launch alone 27 us, 64 %: its warps end together, each with 3 us of looking again); one sequence of 4 beams, 32000
// logits: 8 us, of which the two launches' own latency is most; 8 sequences of 8 beams, 32 best 49 us, 64 best 210.  Before: a CTA per slice of 8192 logits with the n-th largest found per slice
// 70 us; lists kept sorted while streaming 44 us; a lane's third portion looked at one portion at a time, by the lane alone, 44 us.
#include <float.h>
#include <math.h>

#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "paged.h"

namespace {
constexpr int BT = 256, BW = BT / 32;  // of the second launch
constexpr int ROOM = 512;               // candidates that pass its bound
constexpr int RW = 4, HITS = 96;        // warps of a CTA of the first, values that pass a warp's bound

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
constexpr int warps_of_sm(bool f32) { return f32 ? 24 : 16; }  // two portions of a lane are 32 registers, their values 16 (32) more
struct RowPart { float m, s; };  // of a segment: the largest logit and the sum of e^(logit - m)

// 32 bits of a row: one fp32 logit or two of 16 bits
template <typename T> struct Word {
  static constexpr int N = sizeof(T) == 4 ? 1 : 2;
  static constexpr uint32_t NONE = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, bf16>::value ? 0xff80u : 0xfc00u;  // -infinity
  __device__ static __forceinline__ uint32_t bits(const T* p) {
    if constexpr (N == 1) return __float_as_uint(__ldcs(p));
    else return __ldcs(reinterpret_cast<const unsigned short*>(p));
  }
  __device__ static __forceinline__ float value(uint32_t w, int e) {
    if constexpr (N == 1) return __uint_as_float(w);
    else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float(e ? w & 0xffff0000u : w << 16);
    else return e ? __high2float(*reinterpret_cast<const __half2*>(&w)) : __low2float(*reinterpret_cast<const __half2*>(&w));
  }
};
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The n largest values of a warp so far, by value and then index: place r is lane r % 32 of v[r / 32].
template <int NL> struct Best {
  float v[NL];
  int at[NL];
  float least;   // the n-th, and its index (none: -infinity, -1)
  int least_at;
  __device__ __forceinline__ void none() {
#pragma unroll
    for (int i = 0; i < NL; ++i) { v[i] = -INFINITY; at[i] = -1; }
    least = -INFINITY;
    least_at = -1;
  }
  __device__ __forceinline__ bool passes(float x, int i) const { return x > least || (x == least && x > -INFINITY && i < least_at); }
  __device__ __forceinline__ void insert(float x, int i, int n, int lane) {
    if constexpr (NL == 2) {
      const int first = __popc(__ballot_sync(L3_FULL, v[0] > x || (v[0] == x && at[0] < i)));
      const float carry = __shfl_sync(L3_FULL, v[0], 31);
      const int carry_at = __shfl_sync(L3_FULL, at[0], 31);
      if (first < 32) {
        put(0, first, x, i, lane);
        put(1, 0, carry, carry_at, lane);
      } else put(1, __popc(__ballot_sync(L3_FULL, v[1] > x || (v[1] == x && at[1] < i))), x, i, lane);
    } else put(0, __popc(__ballot_sync(L3_FULL, v[0] > x || (v[0] == x && at[0] < i))), x, i, lane);
    const int last = (n - 1) & 31;
    least = __shfl_sync(L3_FULL, NL == 2 && n > 32 ? v[NL - 1] : v[0], last);
    least_at = __shfl_sync(L3_FULL, NL == 2 && n > 32 ? at[NL - 1] : at[0], last);
  }
  __device__ __forceinline__ void put(int part, int place, float x, int i, int lane) {
    const float up = __shfl_up_sync(L3_FULL, v[part], 1);
    const int up_at = __shfl_up_sync(L3_FULL, at[part], 1);
    if (lane >= place) {
      v[part] = lane == place ? x : up;
      at[part] = lane == place ? i : up_at;
    }
  }
};

// the row that has `nth` unfinished ones ahead of it, or -1; all lanes of a warp
__device__ __forceinline__ int unfinished(const unsigned char* done, int rows, int nth, int lane) {
  for (int base = 0; base < rows; base += 128) {  // four rows a lane
    uint32_t live = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) live |= (base + 4 * lane + i < rows && !done[base + 4 * lane + i] ? 1u : 0u) << i;
    int run = __popc(live);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(L3_FULL, run, o);
      if (lane >= o) run += x;
    }
    const int all = __shfl_sync(L3_FULL, run, 31);
    if (nth < all) {
      const int src = __ffs(__ballot_sync(L3_FULL, run > nth)) - 1;
      uint32_t left = __shfl_sync(L3_FULL, live, src);
      for (int i = __shfl_sync(L3_FULL, run, src) - __popc(left); i < nth; ++i) left &= left - 1;
      return base + 4 * src + __ffs(left) - 1;
    }
    nth -= all;
  }
  return -1;
}

// A portion that was read from multiples of 16 bytes on, `bytes` of them ahead of its logits, becomes the portion itself: every lane's values move
// up, and the last ones come from the next lane - lane 31's from lane 0's next four words, at the portion's end from `behind` (word i in lane i).
__device__ __forceinline__ void move_up(uint32_t (&w)[16], uint32_t behind, int bytes, int lane) {
  int used = 0;  // words of `behind` so far
  auto next = [&](int j, int i) {
    const uint32_t x = __shfl_sync(L3_FULL, lane == 0 && j < 3 ? w[4 * (j < 3 ? j + 1 : 3) + i] : w[4 * j + i], (lane + 1) & 31);
    if (j < 3) return x;
    const uint32_t end = __shfl_sync(L3_FULL, behind, used + i);
    return lane == 31 ? end : x;
  };
  if (bytes & 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = next(j, 0), b = next(j, 1);
      w[4 * j] = w[4 * j + 2]; w[4 * j + 1] = w[4 * j + 3]; w[4 * j + 2] = a; w[4 * j + 3] = b;
    }
    used = 2;
  }
  if (bytes & 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = next(j, 0);
      w[4 * j] = w[4 * j + 1]; w[4 * j + 1] = w[4 * j + 2]; w[4 * j + 2] = w[4 * j + 3]; w[4 * j + 3] = a;
    }
    ++used;
  }
  if (bytes & 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = next(j, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * j + i] = __funnelshift_r(w[4 * j + i], i < 3 ? w[4 * j + (i < 3 ? i + 1 : 3)] : a, 16);
    }
  }
}

// part [R, S], cand_v / cand_i [R, S, n].  A portion is 16 words a lane.  Which logits a lane has of which portion hangs on their index alone,
// and not on where a row begins: beams with the same logits have the same sum to the last bit, so that equal candidates stay equal.
// Moving up costs rows that begin between multiples of 16 bytes a tenth: 256 rows of 128257 logits 35.8 us in fp32 and 34.3 in bf16, by places of 16
// bytes (sums that hang on the address) 33.0 and 31.5; rows of 128256 30.9 and 29.9 with either.
template <typename T, int NL>
__global__ void __launch_bounds__(RW * 32, warps_of_sm(sizeof(T) == 4) / RW) beam_rows_kernel(const BeamSelectArgs a, int S, int portions, RowPart* part, float* cand_v, int* cand_i) {
  constexpr int N = Word<T>::N, PIECE = 4 * N, PORTION = 128 * PIECE;  // logits of 16 bytes, of a portion
  __shared__ unsigned long long hits[RW][HITS];
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long id = (long long)blockIdx.x * RW + (threadIdx.x >> 5);
  if (id >= (long long)a.B * a.K * S) return;
  int row = (int)(id / S);
  const int seg = (int)(id - (long long)row * S);
  // A finished beam has one continuation, whatever its logits.  The warps count the others only: left where their rows are, the finished ones'
  // would idle on some SMs more than on others.
  if (a.done && (row = unfinished(a.done, a.B * a.K, row, lane)) < 0) return;
  const int b = row / a.K, k = row - b * a.K;
  const long long list = (long long)row * S + seg;
  const T* x0 = (const T*)a.logits + b * a.sb + k * a.sk;
  const int skip = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));  // logits from the last multiple of 16 bytes to the row's first
  const int first = seg * portions, stop = min(first + portions, (a.V + PORTION - 1) / PORTION);
  // whole portions, which are loaded 16 bytes at a time, two ahead; the last of a row may be a part.  Where skip is not 0, the 16 bytes ahead of a
  // portion and behind it are touched, too, and have to lie within the row.
  const int lo = skip ? 1 : 0, hi = min(stop, skip ? max(a.V + skip - PIECE, 0) / PORTION : a.V / PORTION);
  uint32_t wa[16], wb[16], behind_a = 0, behind_b = 0;
  auto load_whole = [&](uint32_t (&w)[16], uint32_t& behind, int p, int of) {  // of: the lane whose values; to be moved up by skip
    const T* x = x0 - skip + (p * PORTION + of * PIECE);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 r = __ldcs(reinterpret_cast<const uint4*>(x + j * 32 * PIECE));
      w[4 * j] = r.x; w[4 * j + 1] = r.y; w[4 * j + 2] = r.z; w[4 * j + 3] = r.w;
    }
    if (skip) behind = __ldcs(reinterpret_cast<const uint32_t*>(x0 - skip + (p + 1) * PORTION) + (lane & 3));
  };
  auto load = [&](uint32_t (&w)[16], int p, int of) {
    if (!skip && p < hi) return load_whole(w, behind_a, p, of);
    const int base = p * PORTION + of * PIECE;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      w[i] = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int v = base + (i / 4) * 32 * PIECE + (i & 3) * N + e;
        w[i] |= (v < a.V ? Word<T>::bits(x0 + v) : Word<T>::NONE) << (16 * e);
      }
    }
  };
  float m = -INFINITY, s = 0.f;                             // of this lane
  float v1 = -INFINITY, v2 = -INFINITY, v3 = -INFINITY;     // its portions' largest maxima (NaN is none), and where the first two are
  int p1 = first, p2 = first;
  auto take = [&](uint32_t (&w)[16], uint32_t& behind, int p, bool whole, bool more) {
    if (whole && skip) move_up(w, behind, skip * (int)sizeof(T), lane);
    float x[16 * N];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) x[i * N + e] = Word<T>::value(w[i], e);
    if (more) load_whole(w, behind, p + 2, lane);
    float half[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 8 * N; ++i) {
      half[0] = fmaxf(half[0], x[i]);
      half[1] = fmaxf(half[1], x[i + 8 * N]);
    }
    const float top = fmaxf(half[0], half[1]), mn = fmaxf(m, top), from = mn == -INFINITY ? 0.f : mn;
    s *= ex2((m - from) * 1.4426950408889634f);
    m = mn;
    float2 sum = make_float2(0.f, 0.f);
    const float2 one = make_float2(1.f, 1.f), down = make_float2(-from, -from), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
    for (int i = 0; i < 16 * N; i += 2) {
      // the difference first and by itself: a logit's own multiple of log2 e would be off by more than the difference's
      const float2 d = fma2(fma2(make_float2(x[i], x[i + 1]), one, down), log2e, make_float2(0.f, 0.f));
      sum = fma2(make_float2(ex2(d.x), ex2(d.y)), one, sum);
    }
    s += sum.x + sum.y;
    if (stop - first == 1) {  // one portion: its halves, which lie in the same one
      v1 = top;
      v2 = fminf(half[0], half[1]);
    } else if (top > v1) {
      v3 = v2; v2 = v1; v1 = top;
      p2 = p1; p1 = p;
    } else if (top > v2) {
      v3 = v2; v2 = top;
      p2 = p;
    } else v3 = fmaxf(v3, top);
  };
  if (first < hi) {
    if (first >= lo) load_whole(wa, behind_a, first, lane);
    else load(wa, first, lane);
  }
  if (first + 1 < hi) load_whole(wb, behind_b, first + 1, lane);
  for (int p = first; p < hi; p += 2) {
    take(wa, behind_a, p, p >= lo, p + 2 < hi);
    if (p + 1 < hi) take(wb, behind_b, p + 1, true, p + 3 < hi);
  }
  for (int p = max(first, hi); p < stop; ++p) {
    load(wa, p, lane);
    take(wa, behind_a, p, false, false);
  }
  const float mw = warp_max(m), from = mw == -INFINITY ? 0.f : mw;
  s = warp_sum(s * ex2((m - from) * 1.4426950408889634f));
  if (lane == 0) part[list] = RowPart{mw, s};

  const uint32_t nth = nth_of_warp(order_key(v1), order_key(v2), a.n);
  const float bound = nth > NO_KEY ? key_value(nth) : -FLT_MAX;
  unsigned long long* hit = hits[threadIdx.x >> 5];
  int count = 0;
  auto collect = [&](const uint32_t (&w)[16], int p, int of, bool mine) {  // the values of lane `of` of portion p, if this lane has any
    const int base = p * PORTION + of * PIECE;
#pragma unroll
    for (int i = 0; i < 16 * N; ++i) {
      const float x = Word<T>::value(w[i / N], i % N);
      const bool in = mine && x >= bound;
      const uint32_t ones = __ballot_sync(L3_FULL, in);
      if (in) {
        const int at = count + __popc(ones & ((1u << lane) - 1));
        if (at < HITS) hit[at] = (unsigned long long)order_key(x) << 32 | (0xffffffffu - (uint32_t)(base + (i / PIECE) * 32 * PIECE + i % PIECE));
      }
      count += __popc(ones);
    }
  };
  const bool one = first < stop && v1 >= bound, two = stop - first > 1 && v2 >= bound && p2 != p1;
  if (one) load(wa, p1, lane);
  if (two) load(wb, p2, lane);
  collect(wa, p1, lane, one);
  if (__any_sync(L3_FULL, two)) collect(wb, p2, lane, two);
  // a lane with three such portions may have more: all of its values, a portion of them each lane
  for (uint32_t many = __ballot_sync(L3_FULL, v3 >= bound); many; many &= many - 1) {
    const int of = __ffs(many) - 1, q1 = __shfl_sync(L3_FULL, p1, of), q2 = __shfl_sync(L3_FULL, p2, of);
    for (int p0 = first; p0 < stop; p0 += 32) {
      const int p = p0 + lane;
      const bool mine = p < stop && p != q1 && p != q2;
      if (mine) load(wa, p, of);
      collect(wa, p, of, mine);
    }
  }
  __syncwarp();
  if (count <= HITS) {
    for (int i = lane; i < count; i += 32) {
      const unsigned long long me = hit[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) rank += hit[j] > me;
      if (rank < a.n) {
        cand_v[list * a.n + rank] = key_value((uint32_t)(me >> 32));
        cand_i[list * a.n + rank] = (int)(0xffffffffu - (uint32_t)me);
      }
    }
    for (int i = count + lane; i < a.n; i += 32) cand_i[list * a.n + i] = -1;
    return;
  }
  // many equal values: a list of the n largest so far, sorted
  Best<NL> best;
  best.none();
  for (int p = first; p < stop; ++p) {
    load(wa, p, lane);
    const int base = p * PORTION + lane * PIECE;
    for (int i = 0; i < 16 * N; ++i) {
      float x = 0.f;
#pragma unroll
      for (int j = 0; j < 16 * N; ++j) x = i == j ? Word<T>::value(wa[j / N], j % N) : x;
      const int v = base + (i / PIECE) * 32 * PIECE + i % PIECE;
      uint32_t ones = __ballot_sync(L3_FULL, best.passes(x, v));
      while (ones) {
        const int src = __ffs(ones) - 1;
        ones &= ones - 1;
        const float nx = __shfl_sync(L3_FULL, x, src);
        const int nv = __shfl_sync(L3_FULL, v, src);
        if (best.passes(nx, nv)) best.insert(nx, nv, a.n, lane);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NL; ++i)
    if (i * 32 + lane < a.n) {
      cand_v[list * a.n + i * 32 + lane] = best.v[i];
      cand_i[list * a.n + i * 32 + lane] = best.at[i];
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
  __shared__ uint32_t keys[2 * BT], least;
  __shared__ int kept;
  __shared__ Scored room[ROOM];
  __shared__ Scored win[BW];
  __shared__ int open[ROOM], passed, count;
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = S * a.n, lists = a.K * S;
  if (tid == 0) {
    count = passed = kept = 0;
    least = NO_KEY + 1;
  }
  const float* cv = cand_v + (long long)b * lists * a.n;
  const int* ci = cand_i + (long long)b * lists * a.n;
  constexpr int HOLD = 4;  // lists whose first candidates a thread keeps; asked for ahead of the rows' sums
  float x[HOLD];
  int v[HOLD];
#pragma unroll
  for (int u = 0; u < HOLD; ++u) {
    const int i = (tid + u * BT) * a.n;
    x[u] = tid + u * BT < lists ? cv[i] : 0.f;
    v[u] = tid + u * BT < lists ? ci[i] : -1;
  }
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
      if (p.m > -INFINITY || p.s != p.s) s += (double)p.s * (double)expf(p.m - from);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(L3_FULL, s, o);
    if (lane == 0) {
      add[k] = (double)s0 - log(s);
      off[k] = from;
    }
  }
  __syncthreads();
  // candidate i: beam i / per, its segment's list; a finished beam has the end token, at its own score
  auto scored = [&](int i, float x, int v) {
    const int k = i / per, in = i - k * per;
    Scored c{-INFINITY, 0};
    if (a.done && a.done[(long long)b * a.K + k]) {
      if (in == 0) c = Scored{add[k], (unsigned)(k * a.V + a.eos)};
    } else if (v >= 0) c = Scored{((double)x - (double)off[k]) + add[k], (unsigned)(k * a.V + v)};
    if (!(c.s > -INFINITY) || c.s == INFINITY) c.s = -INFINITY;  // NaN, too
    return c;
  };
  auto read = [&](int i) { return scored(i, cv[i], ci[i]); };
  // Every list begins with its best, so the n-th best of the lists' firsts bounds the n-th of all from below, and only lists whose first
  // passes it hold any that do.  The bound is on scores rounded to fp32, which keeps their order up to ties.
  auto key_of = [&](const Scored& c) { return order_key((float)c.s); };
  uint32_t held[HOLD], ka = 0, kb = 0;
#pragma unroll
  for (int u = 0; u < HOLD; ++u) {
    held[u] = tid + u * BT < lists ? key_of(scored((tid + u * BT) * a.n, x[u], v[u])) : 0;
    if (u & 1) ka = held[u] > ka ? held[u] : ka;
    else kb = held[u] > kb ? held[u] : kb;
  }
  for (int i = tid + HOLD * BT; i < lists; i += BT) {
    const uint32_t key = key_of(read(i * a.n));
    if ((i / BT) & 1) ka = key > ka ? key : ka;
    else kb = key > kb ? key : kb;
  }
  // ... of which each warp finds its own n-th; the largest of those leaves few that are counted off against one another
  const uint32_t floor_key = nth_of_warp(ka, kb, a.n);
  if (lane == 0) atomicMax(&least, floor_key);
  __syncthreads();
  const uint32_t rough = least;
  for (uint32_t key : {ka, kb})
    if (key >= rough) keys[atomicAdd(&kept, 1)] = key;
  __syncthreads();
  const int m = kept;
  for (int i = tid; i < m; i += BT) {
    const uint32_t me = keys[i];
    int more = 0, same = 0;
    for (int j = 0; j < m; ++j) {
      more += keys[j] > me;
      same += keys[j] == me;
    }
    if (more < a.n && more + same >= a.n) least = me;  // all that write write the same; fewer than n: what is there stays
  }
  __syncthreads();
  const uint32_t bound = least;
  auto pass = [&](int i, uint32_t key) {
    if (key < bound) return;
    const int at = atomicAdd(&passed, 1);
    if (at < ROOM) open[at] = i;
  };
#pragma unroll
  for (int u = 0; u < HOLD; ++u) pass(tid + u * BT, held[u]);
  for (int i = tid + HOLD * BT; i < lists; i += BT) pass(i, key_of(read(i * a.n)));
  __syncthreads();
  const int some = passed;
  for (int i = tid; i < min(some, ROOM) * a.n; i += BT) {
    const Scored c = read(open[i / a.n] * a.n + i % a.n);
    if (c.s > -INFINITY && key_of(c) >= bound) {
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
  if (c <= ROOM && some <= ROOM) {
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
    for (int i = tid; i < lists * a.n; i += BT) {
      const Scored x = read(i);
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

struct Cut { int S, portions; };
// Segments of a row: as many as the machine has room for at once (219 rows of 128256 fp32 logits 30.5 us; two segments for every place 34.7, three
// 37.4), of one portion (2 KB of a row) at least.
Cut cut_of(int rows, int V, int dtype, int n_sm) {
  const bool f32 = dtype == L3_DTYPE_F32;
  const int portion = f32 ? 512 : 1024, all = (V + portion - 1) / portion;
  const int want = warps_of_sm(f32) * n_sm / rows;
  const int portions = want >= all ? 1 : want <= 1 ? all : (all + want - 1) / want;
  return Cut{(all + portions - 1) / portions, portions};
}
template <typename T> cudaError_t launch_rows(const BeamSelectArgs& a, const Cut& c, RowPart* part, float* cv, int* ci, cudaStream_t s) {
  const dim3 g((unsigned)(((long long)a.B * a.K * c.S + RW - 1) / RW));
  if (a.n > 32) return launch_k(beam_rows_kernel<T, 2>, g, dim3(RW * 32), 0, s, a, c.S, c.portions, part, cv, ci);
  return launch_k(beam_rows_kernel<T, 1>, g, dim3(RW * 32), 0, s, a, c.S, c.portions, part, cv, ci);
}
}  // namespace

size_t beam_select_workspace(int B, int K, int V, int n, int n_sm) {
  const int wide = cut_of(B * K, V, L3_DTYPE_F32, n_sm).S, half = cut_of(B * K, V, L3_DTYPE_BF16, n_sm).S;  // any type's
  const size_t lists = (size_t)B * K * (wide > half ? wide : half);
  return lists * (sizeof(RowPart) + (size_t)n * 8);
}
cudaError_t launch_beam_select(const BeamSelectArgs& a, int n_sm, cudaStream_t s) {
  const Cut c = cut_of(a.B * a.K, a.V, a.dtype, n_sm);
  const size_t lists = (size_t)a.B * a.K * c.S;
  RowPart* part = (RowPart*)a.ws;
  float* cv = (float*)(part + lists);
  int* ci = (int*)(cv + lists * a.n);
  cudaError_t e = a.dtype == L3_DTYPE_F32    ? launch_rows<float>(a, c, part, cv, ci, s)
                  : a.dtype == L3_DTYPE_BF16 ? launch_rows<bf16>(a, c, part, cv, ci, s)
                                             : launch_rows<__half>(a, c, part, cv, ci, s);
  if (e != cudaSuccess) return e;
  g_l3_pdl_next = true;
  return launch_k(beam_pick_kernel, dim3(a.B), dim3(BT), 0, s, a, c.S, (const RowPart*)part, (const float*)cv, (const int*)ci);
}

// ------------------------------------------------------------------------------------------------ beam search over a model's own caches
namespace {
__global__ void beam_prompts_kernel(const BeamState b, int L) {
  pdl_launch();
  pdl_wait();
  const int r = blockIdx.x;
  for (int t = threadIdx.x; t < L; t += blockDim.x) b.table[(long long)r * b.M + t] = r / b.K * b.stride + t;
  if (threadIdx.x == 0) {
    b.scores[r] = 0.f;
    b.done[r] = 0;
  }
}
__global__ void beam_begin_kernel(const BeamState b) {
  pdl_launch();
  pdl_wait();
  const int step = b.scal[1] + 1, pos = b.scal[2] + step;
  for (int r = threadIdx.x; r < b.rows; r += blockDim.x) b.table[(long long)r * b.M + pos] = r * b.stride + pos;
  __syncthreads();
  if (threadIdx.x == 0) {
    b.scal[1] = step;
    b.scal[0] = pos;
  }
}
__global__ void beam_commit_kernel(const BeamState b) {
  pdl_launch();
  pdl_wait();
  const long long step = b.scal[1];
  for (int r = blockIdx.x * blockDim.x + threadIdx.x; r < b.rows; r += gridDim.x * blockDim.x) {
    b.scores[r] = b.new_scores[r];
    b.done[r] = b.new_done[r];
    b.hist_tokens[step * b.rows + r] = b.tokens[r];
    b.hist_parents[step * b.rows + r] = b.parents[r];
  }
}
}  // namespace

cudaError_t launch_beam_prompts(const BeamState& b, int L, cudaStream_t s) {
  return launch_k(beam_prompts_kernel, dim3(b.rows), dim3(128), 0, s, b, L);
}
cudaError_t launch_beam_begin(const BeamState& b, cudaStream_t s) { return launch_k(beam_begin_kernel, dim3(1), dim3(256), 0, s, b); }
cudaError_t launch_beam_commit(const BeamState& b, cudaStream_t s) {
  return launch_k(beam_commit_kernel, dim3((b.rows + 127) / 128), dim3(128), 0, s, b);
}

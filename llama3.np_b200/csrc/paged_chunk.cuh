// What the kernels of attention of a packed step share (paged_chunk.cu: fp32 caches, paged_chunk_tc.cu: 16-bit ones): how the work is cut, and the slow path of rows
// that a value without a number has reached.
//
// The R query heads of a kv head and the n rows of a request are n R flat rows that see (nearly) the same keys; row f is token f / R, head f % R of
// the group.  An item is tile_rows of them (a tile) against the blocks of BK keys that its last row sees.  The items of all requests, tiles and kv heads, in
// that order, are one long line, weighed by their blocks, that the CTAs share out evenly: prompts, portions and single tokens of any mixture leave no
// SM idle.  An item of few blocks goes to the CTA that has its middle; longer ones are cut where the shares end, leave partials (m, l, o) that a
// second, dependent launch joins in the order of the keys, so that results do not change from run to run.
#pragma once
#include <math.h>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "packed.h"
#include "paged_chunk_tc.h"

namespace chunk {
template <typename T> __device__ __forceinline__ float up(T x) { return to_f32(x); }
template <> __device__ __forceinline__ float up<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T down(float x) { return from_f32<T>(x); }
template <> __device__ __forceinline__ __half down<__half>(float x) { return __float2half_rn(x); }

struct Request {
  int s0, n;      // its rows
  int len;        // its tokens, those of the rows among them
  int keys;       // tokens that the table has columns for
  __device__ __forceinline__ int seen(int t) const { return min(max(len - n + t + 1, 0), keys); }  // by its row t: [0, seen)
};
__device__ __forceinline__ Request request(const ChunkArgs& a, int b) {
  Request r;
  r.s0 = min(max(a.starts[b], 0), a.T);
  r.n = min(max(a.starts[b + 1], r.s0), a.T) - r.s0;
  r.len = max(a.lengths[b], 0);
  r.keys = a.max_pages << a.log_page;
  return r;
}
__device__ __forceinline__ int tiles(const ChunkArgs& a, int n) { return (int)((unsigned)(n * a.R + a.tile_rows - 1) / (unsigned)a.tile_rows); }
template <int BK> __device__ __forceinline__ int blocks(const ChunkArgs& a, const Request& r, int tile) {
  const int last = min(r.n * a.R, (tile + 1) * a.tile_rows) - 1;
  return (int)((unsigned)(r.seen(last / a.R) + BK - 1) / BK);
}
// An item's weight: 8 a block, or from `few` on of a tile of up to 128 rows, and `ends` for what begins and ends it.  Items of `whole` blocks or
// fewer are not cut; `least`: the least weight of a share.
struct Split { int block, whole, least, few, ends; };
// paged_chunk_tc.cu: one tile of rows has two blocks at a time, which takes half the time as long as the tiles' copies keep up: not in heads of 128, and in
// smaller ones the sooner, the larger the copies.  us, few 4 : 5 : 6 of heads of 64, 48 requests of up to 3001 tokens in pages of 32 98.5 : 100.2 : 104.5, of
// 16 113.5 : - : 106.9, of 8 142 : - : 120; six prompts of up to 4096 in pages of 32 374 : - : 356, of 16 447 : 414 : 381; heads of 128, pages of 16, 6 : 7 : 8
// 508 : 467 : 458
__host__ __device__ constexpr Split tc_split(int HD) { return Split{TC_BK, 4, 8, HD <= 64 ? 5 : 8, 12}; }
__device__ __forceinline__ int per_block(const ChunkArgs& a, const Split& sp, const Request& r, int tile) {
  return min(r.n * a.R - tile * a.tile_rows, a.tile_rows) > 128 ? 8 : min(sp.few + (a.log_page >= 5 ? 0 : a.log_page == 4 ? 1 : 3), 8);
}
// The blocks of an item of nb that lie ahead of weight x.
__device__ __forceinline__ int ahead(long long x, int nb, int per, const Split& sp) {
  const int w = per * nb + sp.ends;
  if (x <= 0) return 0;
  if (x >= w) return nb;
  if (nb <= sp.whole) return 2 * x >= w ? nb : 0;
  return min((int)x / per, nb);
}

struct Place { int b, tile, g, pad; long long off, rest; };  // an item, the weight of it that others have, and what this CTA has from there on

// all * i / n, in 32 bits where that will do
__device__ __forceinline__ long long share_of(long long all, int i, int n) {
  return all < (1 << 21) && i < (1 << 11) ? (long long)((uint32_t)all * (uint32_t)i / (uint32_t)n) : all * i / n;
}
// This CTA's share, by all NT threads (`room`: NT / 32 + 1 words of shared memory).
template <int BK, int NT>
__device__ __forceinline__ void find_share(const ChunkArgs& a, const Split& sp, long long* room, Place* place) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // a thread takes `each` requests, or one of `parts` parts of a request's tiles
  const int parts = max(NT / max(a.B, 1), 1), each = (a.B + NT - 1) / NT;
  auto walk = [&](auto f) {
    const int b0 = parts > 1 ? threadIdx.x / parts : threadIdx.x * each, b1 = min(parts > 1 ? b0 + 1 : b0 + each, a.B);
    for (int b = b0; b < b1; ++b) {
      const Request r = request(a, b);
      const int nt = tiles(a, r.n), part = parts > 1 ? threadIdx.x % parts : 0;
      const int t0 = share_of(nt, part, parts), t1 = share_of(nt, part + 1, parts);
      for (int t = t0; t < t1; ++t)
        if (f(b, t, per_block(a, sp, r, t) * blocks<BK>(a, r, t) + sp.ends)) return;
    }
  };
  long long sum = 0;
  walk([&](int, int, int w) {
    sum += (long long)w * a.G;
    return false;
  });
  long long run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(L3_FULL, run, o);
    if (lane >= o) run += y;
  }
  if (lane == 31) room[warp] = run;
  if (threadIdx.x == 0) *place = Place{-1, 0, 0, 0, 0, 0};
  __syncthreads();
  long long before = run - sum, all = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += room[w];
    all += room[w];
  }
  const int ctas = (int)min((long long)a.n_cta, max(all / sp.least, 1LL));
  if (blockIdx.x < ctas) {
    const long long w0 = share_of(all, blockIdx.x, ctas), w1 = share_of(all, blockIdx.x + 1, ctas);
    if (before <= w0 && w0 < before + sum) {
      long long at = before;
      walk([&](int b, int t, int w) {
        const long long whole = (long long)w * a.G;
        if (w0 >= at + whole) {
          at += whole;
          return false;
        }
        const int g = (int)((w0 - at) / w);
        *place = Place{b, t, g, 0, w0 - at - (long long)g * w, w1 - w0};
        return true;
      });
    }
  }
  __syncthreads();
}

// One stretch of blocks after the other.
template <int BK> struct Cursor {
  int b, tile, g, nt, nb, per;
  Request r;
  long long off, rest;
  int j0, j1;               // blocks of this stretch
  __device__ __forceinline__ void at_tile(const ChunkArgs& a, const Split& sp) {
    nb = blocks<BK>(a, r, tile);
    per = per_block(a, sp, r, tile);
  }
  __device__ __forceinline__ bool start(const ChunkArgs& a, const Split& sp, const Place& p) {
    b = p.b; tile = p.tile; g = p.g; off = p.off; rest = p.rest;
    if (b < 0) return false;
    r = request(a, b);
    nt = tiles(a, r.n);
    at_tile(a, sp);
    return settle(sp) ? true : next(a, sp);
  }
  // the stretch of this item, if there is one
  __device__ __forceinline__ bool settle(const Split& sp) {
    if (rest <= 0) return false;
    j0 = ahead(off, nb, per, sp);
    j1 = ahead(off + rest, nb, per, sp);
    return j1 > j0 || (nb == 0 && off == 0);
  }
  __device__ __forceinline__ bool next(const ChunkArgs& a, const Split& sp) {
    for (;;) {
      rest -= per * nb + sp.ends - off;
      off = 0;
      if (rest <= 0) return false;
      if (++g == a.G) {
        g = 0;
        if (++tile == nt) {
          tile = 0;
          do {
            if (++b >= a.B) return false;
            r = request(a, b);
            nt = tiles(a, r.n);
          } while (nt == 0);
        }
        at_tile(a, sp);
      }
      if (settle(sp)) return true;
    }
  }
  __device__ __forceinline__ bool whole() const { return j0 == 0 && j1 == nb; }
  __device__ __forceinline__ int slot() const { return j0 > 0 ? 0 : 1; }  // of a partial: of the item that this CTA goes on with, or begins
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The values of a key that a row sees may be infinite or NaN, those of keys that it does not see have to be kept out even so, and tiles
// multiply them by a weight of 0.  A row whose result is not finite is therefore taken once more, behind the join, by the formula alone, by a warp:
// scores with a lane a key, then the values a key at a time, four on their way; only what the row sees enters.  A weight is 0 for a score of
// -infinity only, however small, as its value may be infinite.
template <typename T, int HD> __device__ __forceinline__ void by_formula(const ChunkArgs& a, int b, int g, int row, int head, int seen) {
  constexpr int N = (HD + 31) / 32, E = 16 / sizeof(T);
  struct alignas(16) Piece { T x[E]; };
  const int lane = threadIdx.x & 31;
  const int* table = a.table + b * a.table_stride;
  const T* q = (const T*)a.q + row * a.q_st + head * a.q_sh;
  const float sc = a.scale * 1.4426950408889634f;
  auto row_of = [&](const PagedPool& p, int j, int page) { return (const T*)p.p + page * p.sp + g * p.sh + (j & ((1 << a.log_page) - 1)) * p.st; };
  auto score = [&](int j, int& page) {  // of this lane's key; page -1: there is none
    page = j < seen ? table[j >> a.log_page] : -1;
    if ((unsigned)page >= (unsigned)a.n_pages) page = -1;
    if (page < 0) return -INFINITY;
    const T* k = row_of(a.k, j, page);
    float s = 0.f;
#pragma unroll 4
    for (int i = 0; i < HD; i += E) {
      const Piece x = *reinterpret_cast<const Piece*>(q + i), y = *reinterpret_cast<const Piece*>(k + i);
#pragma unroll
      for (int e = 0; e < E; ++e) s += up(x.x[e]) * up(y.x[e]);
    }
    return s * sc;
  };
  float o[N], m = -INFINITY, l = 0.f;
  int page;
  for (int j = 0; j < seen; j += 32) m = fmaxf(m, score(j + lane, page));
  m = warp_max(m);
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  const float from = m == -INFINITY ? 0.f : m;
  for (int j = 0; j < seen; j += 32) {
    const float s = score(j + lane, page), x = s - from;
    const float w = page < 0 ? 0.f : x < -149.f && s > -INFINITY ? 1.4e-45f : exp2f(x);
    l += w;
    unsigned list = __ballot_sync(L3_FULL, page >= 0);
    while (list) {
      float wk[4], v[4][N];
      int of[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        of[k] = __ffs(list) - 1;
        list &= list - 1;
        const int from_lane = max(of[k], 0), its = __shfl_sync(L3_FULL, page, from_lane);
        wk[k] = __shfl_sync(L3_FULL, w, from_lane);
#pragma unroll
        for (int i = 0; i < N; ++i) v[k][i] = of[k] >= 0 && lane + 32 * i < HD ? up(row_of(a.v, j + from_lane, its)[lane + 32 * i]) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (of[k] >= 0) o[i] += wk[k] * v[k][i];
    }
  }
  l = warp_sum(l);
  const long long at = (long long)row * a.H + head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 32 * i < HD) ((T*)a.out)[at * HD + lane + 32 * i] = down<T>(o[i] * inv);
  if (lane == 0 && a.lse) a.lse[at] = (m + log2f(l)) * 0.6931471805599453f;
}

// rows of no request, ahead of the first and behind the last
template <typename T> __device__ __forceinline__ void clear_rest(const ChunkArgs& a, int thread, int threads) {  // by some of a CTA's threads
  if (!a.clear_rest) return;
  const int from = a.B ? min(max(a.starts[a.B], 0), a.T) : 0, ahead = a.B ? min(max(a.starts[0], 0), from) : 0;
  const long long first = (long long)ahead * a.H, gap = (long long)(from - ahead) * a.H, n = (long long)a.T * a.H - gap;  // heads' rows; i-th: behind the gap from `first` on
  const long long begin = (long long)blockIdx.x * threads + thread, step = (long long)gridDim.x * threads;
  if (a.lse)
    for (long long i = begin; i < n; i += step) a.lse[i < first ? i : i + gap] = -INFINITY;
  if (a.clear_rest == 1)
    for (long long i = begin; i < n * a.HD; i += step) ((T*)a.out)[i < first * a.HD ? i : i + gap * a.HD] = down<T>(0.f);
}

// What a CTA leaves for the join: its share, whether a result of an item that it has whole is not finite, and of its two partials - of the
// item that it goes on with, and of the one that it begins - (request, tile, kv head, 1 if the item ends with it), request -1: none.
struct Left {
  Place place;
  int4 part[2];
  int odd, pad[3];
};
static_assert(sizeof(Left) % 16 == 0, "");
// the partials begin on 32 bytes, as they are stored; a workspace need not
constexpr size_t PART_ALIGN = 32;
inline float* part_begin(void* ws) { return reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ws) + PART_ALIGN - 1) & ~(uintptr_t)(PART_ALIGN - 1)); }
__device__ __forceinline__ Left& left_of(const ChunkArgs& a, int cta) { return reinterpret_cast<Left*>(a.left)[cta]; }
__device__ __forceinline__ void leave_nothing(const ChunkArgs& a, const Place& place) {  // by one thread, ahead of all others' words
  Left& left = left_of(a, blockIdx.x);
  left.place = place;
  left.part[0] = left.part[1] = make_int4(-1, 0, 0, 0);
  left.odd = 0;
}
}  // namespace chunk

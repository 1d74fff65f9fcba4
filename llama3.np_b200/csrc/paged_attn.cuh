// Attention of one new token per sequence over a key / value cache in pages (L3PagedAttn):
//   s_j = scale q_h . k_j,  o_h = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse_h = m + log sum_j e^(s_j - m),  m = max_j s_j
// over the tokens j < length of the sequence; token j lies in page table[j / P] at place j % P.
//
// Bound by the cache's bytes: every key and value is read once for all query heads of its kv head (2 HD values for 4 HD flops per
// query head).  The keys of all (sequence, kv head) items, in tiles of 8 - 32, are one long row that the warps of the machine share
// out evenly - lengths of any mixture leave no SM idle, and a single long sequence fills the machine.  A warp works through its
// stretch alone, without a block barrier, its next tiles on their way into two buffers of its own in shared memory by
// asynchronous copies, across items; one pass with running maximum and sum.  An item that lies within one warp's stretch
// is written at once; one that several warps share leaves a partial (m, l, o) per warp, and a second, dependent launch joins those
// in the order of the keys, so that results do not change from run to run.  Where items have few keys, an item is one to four
// warps' of a block (paged_whole_kernel) or, of few items, a cluster's (paged_item_kernel) instead, which join their partials themselves.
//
// Measured (B200, both launches, replayed from a graph over inputs larger than L2): 64 sequences of 4096 tokens, 32 query heads over 8 kv heads of
// 128 in bf16, 182 us = 5.9 TB/s, 90 % of what a copy reaches; one sequence of 131072 tokens 99 us (83 %); 48 of up to 4001 tokens, heads of 64
// in fp16, 43 us (70 %); 256 of up to 256 tokens, 6 heads of 48 in fp32, 21 us (57 %); one of 701 tokens 8.6 us.  What the smaller ones pay is
// fixed: the lengths, then the table, then the rows are three round trips to memory, and the join is three more behind a launch.  Steps on the way, in us for the 131072 / 4001 / 256 tokens: four tiles a warp of 8 warps an SM, pointers passed between lanes
// 105 / 70 / 37; rows straight into registers in the order that the products read them 111 / 43 / 30 (too few bytes on their way at head size
// 128); two tiles a warp of 12 warps, offsets of 32 bits, next item's query ahead of time 98 / 45 / 29; items weighed by half a tile 98 / 44 / 26.
//
// STEP: the rows are a packed step's (PagedAttnArgs::starts), several of a sequence perhaps, and a row's sequence is searched for.  A kernel that can do
// both takes 9.0 us for 8.5 over one sequence of 1000 tokens, 5.3 for 5.0 over one of 100 (rows of a step: five over 1500 tokens 14.4 for 13.9), so the two
// are apart (paged.cu, paged_packed.cu).
#pragma once
#include <math.h>

#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "attn_decode.cuh"
#include "paged.h"

namespace {
constexpr int MOST_WARPS = 16;  // of an SM (Core::CTAS of Core::NW warps)
constexpr int HEADS = 8;        // most query heads of an item

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, bf16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two values as the nearest 16-bit ones, and what those leave (again as 16-bit values)
template <typename T> __device__ __forceinline__ void two_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, bf16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 r = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    const __half2 r = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
}
// The same where a factor that is not 0 must not become 0, since the other one may be infinite: what fp16 has no number for enters as its smallest
// one, 2^-24, and the rest takes that back.  Weights are 0 or more, and what multiplies one of 0 is 0, too (a key that is not there).
template <typename T> __device__ __forceinline__ void weight_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, bf16>::value) two_parts<T>(x, y, hi, lo);  // fp32's exponents
  else {
    const __half2 h = __hmax2_nan(__floats2half2_rn(x, y), __half2_raw{0x0001, 0x0001});
    const __half2 r = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <typename T> __device__ __forceinline__ void query_parts(float x, float y, uint32_t& hi, uint32_t& lo) {
  two_parts<T>(x, y, hi, lo);
  if constexpr (!std::is_same<T, bf16>::value) {
    const bool low = x != 0.f && !(hi & 0x7fffu), high = y != 0.f && !(hi & 0x7fff0000u);
    if (!low && !high) return;
    if (low) hi |= 0x0001u;   // the sign is there already
    if (high) hi |= 0x00010000u;
    const __half2 h = *reinterpret_cast<const __half2*>(&hi), r = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
}
// What two parts' products add up to.  Times an infinite value the rest gives an infinity of either sign, or NaN; then the first part alone has the
// product's sign, and is NaN where the sum is.  (Scores of an fp32 query take up to 2 % more for it.)
__device__ __forceinline__ float of_parts(float first, float rest) { return fabsf(rest) < INFINITY ? first + rest : first; }
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes into shared memory, zeros where !take (the address is not read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float load_q(const PagedAttnArgs& a, long long i) {
  if (a.q_dtype == L3_DTYPE_F32) return __ldg((const float*)a.q + i);
  if (a.q_dtype == L3_DTYPE_BF16) return __bfloat162float(((const bf16*)a.q)[i]);
  return __half2float(((const __half*)a.q)[i]);
}
// N (2, 4 or 8) neighbouring outputs, i a multiple of N
template <int N> __device__ __forceinline__ void store_out(const PagedAttnArgs& a, long long i, const float (&v)[N]) {
  if (a.out_dtype == L3_DTYPE_F32) {
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float2 x = make_float2(v[e], v[e + 1]);
      if (a.out_lo) {
        float2 lo;
        split_tf32(v[e], x.x, lo.x);
        split_tf32(v[e + 1], x.y, lo.y);
        *reinterpret_cast<float2*>(a.out_lo + i + e) = lo;
      }
      *reinterpret_cast<float2*>((float*)a.out + i + e) = x;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; e += 2) {
    uint32_t x, rest;
    if (a.out_dtype == L3_DTYPE_BF16) two_parts<bf16>(v[e], v[e + 1], x, rest);
    else two_parts<__half>(v[e], v[e + 1], x, rest);
    *reinterpret_cast<uint32_t*>((bf16*)a.out + i + e) = x;
  }
}
// the sequence that row b belongs to (a packed step's rows), or -1
__device__ __forceinline__ int sequence_of(const PagedAttnArgs& a, int b) {
  int lo = -1, hi = a.requests;  // starts[lo] <= b < starts[hi], as far as they rise
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo >= 0 && b < a.starts[lo + 1] ? lo : -1;
}
template <bool STEP> __device__ __forceinline__ int asked_length(const PagedAttnArgs& a, int b) {
  if constexpr (STEP) {
    const int r = sequence_of(a, b);
    return r < 0 ? 0 : max(a.lengths[r], 0) - min(a.starts[r + 1], a.B) + b + 1;
  } else return a.lengths ? a.lengths[b] : *a.pos_ptr + 1;
}
template <bool STEP> __device__ __forceinline__ const int* table_of(const PagedAttnArgs& a, int b) {
  if constexpr (STEP) return a.table + sequence_of(a, b) * a.table_stride;
  else return a.table + b * a.table_stride;
}
template <bool STEP> __device__ __forceinline__ int length_of(const PagedAttnArgs& a, int b) { return min(max(asked_length<STEP>(a, b), 0), a.max_pages << a.log_page); }

// where a warp is in the long row of tiles: tile t of the nt tiles of item (sequence b, kv head g, block of its query heads)
struct Cursor {
  int b, g, blk, t, nt, len;
  __device__ __forceinline__ int head0(const PagedAttnArgs& a) const { return g * a.nrep + blk * a.heads_blk; }
  __device__ __forceinline__ int heads(const PagedAttnArgs& a) const { return min(a.heads_blk, a.nrep - blk * a.heads_blk); }
  __device__ __forceinline__ int item(const PagedAttnArgs& a) const { return (b * a.G + g) * a.blocks + blk; }
};
template <int TK> __device__ __forceinline__ int tiles_of(int len) { return (int)((unsigned)(len + TK - 1) / TK); }
template <int TK, bool STEP> __device__ __forceinline__ void advance(const PagedAttnArgs& a, Cursor& c) {
  if (++c.t < c.nt) return;
  c.t = 0;
  if (++c.blk < a.blocks) return;
  c.blk = 0;
  if (++c.g < a.G) return;
  c.g = 0;
  do {
    ++c.b;
    c.len = c.b < a.B ? length_of<STEP>(a, c.b) : 0;
    c.nt = tiles_of<TK>(c.len);
  } while (c.b < a.B && c.nt == 0);
}
__device__ __forceinline__ long long weight_of(int nt) { return nt ? 2LL * nt + 1 : 0; }
// 64-bit division that is a 32-bit one wherever that will do
__device__ __forceinline__ long long quotient(long long x, int d) { return (unsigned long long)x >> 32 ? x / d : (long long)((uint32_t)x / (uint32_t)d); }

// The rows of a tile: lane j (of TK; the others repeat them) has the places of key j's rows, in units of the pools.
struct Rows {
  uint32_t k, v;               // offsets in units of a.unit bytes
  uint32_t mask;               // keys that there are
  int fresh, writes;           // the key that comes from k_new / v_new, or -1; the same if this item writes it to its page
};
struct Fresh { const char *k, *v; };  // its rows
struct Home { uint32_t k, v; };       // the offsets of their places in the pools
__device__ __forceinline__ const char* row_at(const void* pool, uint32_t off, int unit) { return (const char*)pool + (unsigned long long)off * (uint32_t)unit; }

// A tile's rows in shared memory: TK rows of NCH pieces of 16 bytes.  TURN: a row's pieces lie in an order that keeps the eight rows of a
// matrix that ldmatrix reads on different banks.
template <int TK, int NCH, bool TURN> struct Tile {
  static_assert(NCH <= 32, "a lane writes a piece of a row");
  static constexpr uint32_t ALL = TK == 32 ? 0xffffffffu : (1u << (TK & 31)) - 1;
  __device__ static __forceinline__ int turn(int row) { return !TURN ? 0 : NCH % 8 == 0 ? row & 7 : NCH % 4 == 0 ? (row >> 1) & 3 : (row >> 2) & 1; }
  __device__ static __forceinline__ uint32_t place(int row, int piece) { return (row * NCH + (piece ^ turn(row))) * 16; }
  // writes a row that has arrived to its page
  __device__ static __forceinline__ void write(uint32_t tile, int row, char* to, int lane) {
    if (lane >= NCH) return;
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(tile + place(row, lane)) : "memory");
    reinterpret_cast<uint4*>(to)[lane] = x;
  }
  // copies the rows, asynchronously; rows that are not there become zeros (0 times whatever would lie there has to be 0)
  __device__ static __forceinline__ void copy(const void* pool, int unit, uint32_t off, uint32_t step, bool one_page, const Rows& r, const char* fresh,
                                              uint32_t dst, int lane) {
    constexpr bool EVEN = 32 % NCH == 0;           // every copy of a lane is of the same column of pieces
    constexpr int RS = EVEN ? 32 / NCH : 0;        // and RS rows behind the last
    const int row0 = lane / NCH, c0 = lane % NCH;
    const uint32_t to = dst + row0 * NCH * 16, x = (c0 ^ turn(row0)) * 16;  // turn() of a sum of disjoint bits is the parts' exclusive or
    if (one_page && r.mask == ALL && r.fresh < 0) {  // rows at equal distances from the first lane's
      const uint32_t first = __shfl_sync(L3_FULL, off, 0);
      if constexpr (EVEN) {
        const char* base = (const char*)pool + c0 * 16;
        const uint32_t at = first + row0 * step;
#pragma unroll
        for (int i = 0; i < TK * NCH / 32; ++i) cp16(to + (x ^ (turn(i * RS) * 16)) + i * 512, row_at(base, at + i * RS * step, unit), true);
      } else {
#pragma unroll
        for (int i = 0; i < TK * NCH / 32; ++i) {
          const int at = i * 32 + lane, row = at / NCH, c = at % NCH;
          cp16(dst + place(row, c), row_at(pool, first + row * step, unit) + c * 16, true);
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < TK * NCH / 32; ++i) {
      const int at = i * 32 + lane, row = EVEN ? i * RS + row0 : at / NCH, c = EVEN ? c0 : at % NCH;
      const char* p = row_at(pool, __shfl_sync(L3_FULL, off, row), unit);
      if (row == r.fresh) p = fresh;
      cp16(EVEN ? to + (x ^ (turn(i * RS) * 16)) + i * 512 : dst + place(row, c), p + c * 16, r.mask >> row & 1);
    }
  }
};

// ------------------------------------------------------------------------------------------ 16-bit caches: tensor cores
// The item's (up to 8) query heads are rows 0 - 7 of an m16n8k16 tile.  Rows 8 - 15, which a tile has anyway, carry what rounding to 16
// bits leaves of the same heads: the rest of an fp32 query in S = Q K^T, the rest of the weights in O += P V, so that the weights
// enter with 16 (bf16) or 22 (fp16) significant bits at no further instruction.  fp16 weights (at most 1) are scaled by 2^12 ahead of the
// rounding: those from 2^-15 of the largest on enter with 22 bits; below, what counts is that the rest is off by up to half of fp16's smallest
// number, 2^-37 of the largest weight (weights down to 2^-26 of it are normal numbers themselves, down to 2^-36 more than 0).
// Keys and values are copied apart, so that a tile's keys make room for those of the tile after next while its values are still in use.
template <typename T, int HD_, bool QLO> struct MmaCore {
  static constexpr int HD = HD_, TK = HD > 64 ? 16 : 32;
  static constexpr int NW = 4, CTAS = HD > 96 && QLO ? 2 : HD > 32 ? 3 : 4;  // as many warps as registers and shared memory leave room for
  static constexpr int KS = HD / 16, NT = HD / 8, NCH = HD / 8, HALF = TK * HD * 2, AHEAD = 2;
  using Half = Tile<TK, NCH, true>;
  static constexpr int QW = (QLO ? 4 : 2) * KS;     // words of a lane's share of Q, which waits in shared memory
  static constexpr size_t SMEM = (size_t)NW * (AHEAD * 2 * HALF + (QW + 3) / 4 * 512);
  static constexpr float BIAS = std::is_same<T, bf16>::value ? 0.f : 12.f;
  uint32_t* q;
  uint32_t ring;   // [AHEAD][keys | values] of the warp
  float o[NT][4];
  float m, l;  // of row lane / 4, in units of log 2; l: this lane's share
  float sc, down;  // what turns products into scores in units of log 2; the query's share of it
  float s[TK / 8][4];

  __device__ __forceinline__ void memory(uint8_t* smem, int warp) {
    ring = smem_u32(smem) + warp * AHEAD * 2 * HALF;
    q = reinterpret_cast<uint32_t*>(smem + NW * AHEAD * 2 * HALF) + warp * ((QW + 3) / 4 * 128);
  }
  // words of step ks: its two registers' high parts, then (QLO) what they leave; 16 bytes of every lane side by side
  __device__ __forceinline__ uint32_t& q_word(int i, int lane) { return q[(i / 4 * 32 + lane) * 4 + i % 4]; }
  // The next item's query: asked for (ask_query) ahead of the last tile of the one before, laid into shared memory (load_query) behind it.
  uint32_t asked[QLO ? 1 : KS][2];
  __device__ __forceinline__ void ask_query(const PagedAttnArgs& a, const Cursor& c, int lane) {
    if (QLO || !a.q_vec) return;
    const int g = lane >> 2, t = lane & 3;
    const char* p = (const char*)a.q + (c.b * a.q_sb + (long long)(c.head0(a) + min(g, c.heads(a) - 1)) * a.q_sh) * 2 + t * 4;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      asked[QLO ? 0 : ks][0] = __ldg(reinterpret_cast<const uint32_t*>(p + ks * 32));
      asked[QLO ? 0 : ks][1] = __ldg(reinterpret_cast<const uint32_t*>(p + ks * 32 + 16));
    }
  }
  __device__ __forceinline__ void load_query(const PagedAttnArgs& a, const Cursor& c, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const long long qp = c.b * a.q_sb + (long long)(c.head0(a) + min(g, c.heads(a) - 1)) * a.q_sh;
    if (!QLO && a.q_vec) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) *reinterpret_cast<uint2*>(&q_word(2 * ks, lane)) = make_uint2(asked[QLO ? 0 : ks][0], asked[QLO ? 0 : ks][1]);
      return;
    }
    float x[2 * KS][2], up = 1.f;  // read together: fp32 queries, 48 sequences of up to 4001 tokens in fp16 46.1 us, by pairs 54.7; 64 of 4096 in bf16 180.7 : 193.5
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) x[i][e] = load_q(a, qp + i * 8 + 2 * t + e);
    if constexpr (QLO) {
      // Times a power of two, which the scores' scale takes back.  fp16: the one that takes the row's largest value to [2^14, 2^15), so that two
      // parts hold a query of any size, values down to 2^-17 of the largest with 22 bits (smaller ones to 2^-39 of the largest).  bf16, which has
      // fp32's exponents: one that takes a largest value of 4 or more to [2, 4), so that none rounds to infinity; never up, since keys may be as large.
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) most = fmaxf(most, fmaxf(fabsf(x[i][0]), fabsf(x[i][1])));
      most = fmaxf(most, __shfl_xor_sync(L3_FULL, most, 1));
      most = fmaxf(most, __shfl_xor_sync(L3_FULL, most, 2));
      constexpr bool WIDE = std::is_same<T, bf16>::value;
      const int by = max(min(127 + (WIDE ? 1 : 14) - (int)(__float_as_uint(most) >> 23), WIDE ? 0 : 126), -126);
      up = __uint_as_float((uint32_t)(127 + by) << 23);
      down = __uint_as_float((uint32_t)(127 - by) << 23);
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t high, rest;
        query_parts<T>(x[2 * ks + h][0] * up, x[2 * ks + h][1] * up, high, rest);
        q_word((QLO ? 4 : 2) * ks + h, lane) = high;
        if (QLO) q_word(4 * ks + 2 + h, lane) = rest;
      }
  }
  __device__ __forceinline__ void reset(const PagedAttnArgs& a) {
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m = -INFINITY;
    l = 0.f;
    sc = a.scale * 1.4426950408889634f * (QLO ? down : 1.f);
  }
  // address of the pieces 2 step + second of a matrix row, ks steps on
  __device__ static __forceinline__ uint32_t matrix_row(uint32_t half, int row, int second, int step) {
    if constexpr (NCH % 8 == 0 || NCH == 4) return (half + row * NCH * 16 + (second ^ Half::turn(row)) * 16) ^ (step * 32);  // halves begin on whole rows
    else return half + Half::place(row, step * 2 + second);
  }
  __device__ __forceinline__ void load_keys(const PagedAttnArgs& a, const Rows& r, const Fresh& f, int buf, int lane) {
    Half::copy(a.k.p, a.unit, r.k, a.ku_token, (1 << a.log_page) >= TK, r, f.k, ring + buf * 2 * HALF, lane);
  }
  __device__ __forceinline__ void load_values(const PagedAttnArgs& a, const Rows& r, const Fresh& f, int buf, int lane) {
    Half::copy(a.v.p, a.unit, r.v, a.vu_token, (1 << a.log_page) >= TK, r, f.v, ring + buf * 2 * HALF + HALF, lane);
  }
  __device__ __forceinline__ void scores(int buf, int lane) {
    const int mi = lane >> 3, row = (mi >> 1) * 8 + (lane & 7);
#pragma unroll
    for (int n = 0; n < TK / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t h0, h1, l0 = 0u, l1 = 0u;
      if constexpr (QLO) {
        const uint4 x = *reinterpret_cast<const uint4*>(&q_word(4 * ks, lane));
        h0 = x.x; h1 = x.y; l0 = x.z; l1 = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(&q_word(2 * ks, lane));
        h0 = x.x; h1 = x.y;
      }
#pragma unroll
      for (int u = 0; u < TK / 16; ++u) {
        uint32_t kb[4];
        ldsm_x4(matrix_row(ring + buf * 2 * HALF, row, mi & 1, ks) + u * 16 * NCH * 16, kb);
        mma16816<T>(s[2 * u], h0, l0, h1, l1, kb[0], kb[1]);
        mma16816<T>(s[2 * u + 1], h0, l0, h1, l1, kb[2], kb[3]);
      }
    }
  }
  // weights from the scores (first), then the tile's values (second)
  uint32_t p[TK / 16][4];
  __device__ __forceinline__ void weigh(uint32_t mask, int lane) {
    constexpr uint32_t ALL = TK == 32 ? 0xffffffffu : (1u << (TK & 31)) - 1;
    const int t = lane & 3;
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < TK / 8; ++n) {
      s[n][0] = (QLO ? of_parts(s[n][0], s[n][2]) : s[n][0]) * sc;
      s[n][1] = (QLO ? of_parts(s[n][1], s[n][3]) : s[n][1]) * sc;
      if (mask != ALL) {
        if (!(mask >> (n * 8 + 2 * t) & 1)) s[n][0] = -INFINITY;
        if (!(mask >> (n * 8 + 2 * t + 1) & 1)) s[n][1] = -INFINITY;
      }
      mx = fmaxf(mx, fmaxf(s[n][0], s[n][1]));
    }
    mx = fmaxf(mx, __shfl_xor_sync(L3_FULL, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(L3_FULL, mx, 2));
    const float mn = fmaxf(m, mx), from = mn == -INFINITY ? 0.f : mn;  // no key so far: every weight is 0
    if (__any_sync(L3_FULL, mn > m)) {
      const float alpha = ex2(m - from);
      l *= alpha;
#pragma unroll
      for (int n = 0; n < NT; ++n) { o[n][0] *= alpha; o[n][1] *= alpha; o[n][2] *= alpha; o[n][3] *= alpha; }
      m = mn;
    }
#pragma unroll
    for (int n = 0; n < TK / 8; ++n) {
      s[n][0] = ex2(s[n][0] - from + BIAS);
      s[n][1] = ex2(s[n][1] - from + BIAS);
      l += s[n][0] + s[n][1];
    }
#pragma unroll
    for (int u = 0; u < TK / 16; ++u) {
      weight_parts<T>(s[2 * u][0], s[2 * u][1], p[u][0], p[u][1]);
      weight_parts<T>(s[2 * u + 1][0], s[2 * u + 1][1], p[u][2], p[u][3]);
    }
  }
  __device__ __forceinline__ void add_values(int buf, int lane) {
    const int mi = lane >> 3, row = (mi & 1) * 8 + (lane & 7);
#pragma unroll
    for (int u = 0; u < TK / 16; ++u)
#pragma unroll
      for (int np = 0; np < KS; ++np) {
        uint32_t vb[4];
        ldsm_x4_trans(matrix_row(ring + buf * 2 * HALF + HALF, row, mi >> 1, np) + u * 16 * NCH * 16, vb);
        mma16816<T>(o[2 * np], p[u][0], p[u][1], p[u][2], p[u][3], vb[0], vb[1]);
        mma16816<T>(o[2 * np + 1], p[u][0], p[u][1], p[u][2], p[u][3], vb[2], vb[3]);
      }
  }
  // whole: the result; else the partial: o [heads][HD] and (m, l) [heads]
  __device__ __forceinline__ void end(const PagedAttnArgs& a, bool whole, const Cursor& c, float* part_o, float2* part_ml, int lane) {
    const int b = c.b, head0 = c.head0(a), heads = c.heads(a);
    const int g = lane >> 2, t = lane & 3;
    l += __shfl_xor_sync(L3_FULL, l, 1);
    l += __shfl_xor_sync(L3_FULL, l, 2);
    if (g >= heads) return;
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const long long oi = ((long long)b * a.H + head0 + g) * HD;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float x[2] = {of_parts(o[n][0], o[n][2]) * inv, of_parts(o[n][1], o[n][3]) * inv};
        store_out(a, oi + n * 8 + 2 * t, x);
      }
      if (a.lse && t == 0) a.lse[(long long)b * a.H + head0 + g] = (m - BIAS + log2f(l)) * 0.6931471805599453f;
    } else {
      float* po = part_o + g * HD;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        *reinterpret_cast<float2*>(po + n * 8 + 2 * t) = make_float2(of_parts(o[n][0], o[n][2]), of_parts(o[n][1], o[n][3]));
      if (t == 0) part_ml[g] = make_float2((m - BIAS) * 0.6931471805599453f, l);
    }
  }
};

// --------------------------------------------------------------------------------------------------- fp32 caches: FFMA
// LPK lanes share a key (DecodeCfg), KPW keys side by side; NREP query heads of an item (a.heads_blk of them real).  m, l and o are
// kept per lane group and merged over the warp at the end of an item.
template <int HD_, int NREP> struct F32Core {
  using C = DecodeCfg<HD_, float>;
  static constexpr int HD = HD_, NW = 4, AHEAD = 2;
  static constexpr int EPL = C::EPL, LPK = C::LPK, KPW = C::KPW;
  static constexpr int TK = HD > 64 ? 8 : HD > 32 ? 16 : 32, U = TK / KPW, NCH = HD / 4, HALF = TK * HD * 4;  // keys of a tile, of a lane
  using Half = Tile<TK, NCH, false>;   // eight lanes read one row or two neighbouring ones: no turns
  static constexpr size_t SMEM = (size_t)NW * AHEAD * 2 * HALF;
  static constexpr int NEED = (NREP * EPL <= 16 ? 3 : 2) * NREP * EPL + U * NREP + 2 * EPL + 2 * NREP + 56;  // registers
  static constexpr int BY_REGS = NEED <= 124 ? 4 : NEED <= 164 ? 3 : 2, BY_SMEM = (int)(222 * 1024 / SMEM);
  static constexpr int CTAS = BY_REGS < BY_SMEM ? BY_REGS : BY_SMEM;
  float q[NREP][EPL], o[NREP][EPL], m[NREP], l[NREP];
  float s[U][NREP];
  uint32_t ring;   // as MmaCore's
  __device__ __forceinline__ void memory(uint8_t* smem, int warp) { ring = smem_u32(smem) + warp * AHEAD * 2 * HALF; }

  static constexpr bool ASK = NREP * EPL <= 16;  // as MmaCore's, where the registers are there
  float asked[ASK ? NREP : 1][EPL];
  __device__ __forceinline__ void read_query(const PagedAttnArgs& a, const Cursor& c, int lane, float (&to)[NREP][EPL]) {
    const int sl = lane % LPK;
#pragma unroll
    for (int r = 0; r < NREP; ++r) {
      const float* p = (const float*)a.q + c.b * a.q_sb + (long long)(c.head0(a) + min(r, c.heads(a) - 1)) * a.q_sh;
      if (a.q_vec) {
#pragma unroll
        for (int e = 0; e < EPL; e += 4) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(p + C::dim(sl, e)));
          to[r][e] = x.x; to[r][e + 1] = x.y; to[r][e + 2] = x.z; to[r][e + 3] = x.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < EPL; ++e) to[r][e] = __ldg(p + C::dim(sl, e));
      }
    }
  }
  __device__ __forceinline__ void ask_query(const PagedAttnArgs& a, const Cursor& c, int lane) {
    if constexpr (ASK) read_query(a, c, lane, asked);
  }
  __device__ __forceinline__ void load_query(const PagedAttnArgs& a, const Cursor& c, int lane) {
    if constexpr (!ASK) read_query(a, c, lane, q);
#pragma unroll
    for (int r = 0; r < NREP; ++r)
#pragma unroll
      for (int e = 0; e < EPL; ++e) q[r][e] = (ASK ? asked[ASK ? r : 0][e] : q[r][e]) * a.scale;
  }
  __device__ __forceinline__ void reset(const PagedAttnArgs&) {
#pragma unroll
    for (int r = 0; r < NREP; ++r) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] = 0.f;
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
  }
  __device__ __forceinline__ void load_keys(const PagedAttnArgs& a, const Rows& r, const Fresh& f, int buf, int lane) {
    Half::copy(a.k.p, a.unit, r.k, a.ku_token, (1 << a.log_page) >= TK, r, f.k, ring + buf * 2 * HALF, lane);
  }
  __device__ __forceinline__ void load_values(const PagedAttnArgs& a, const Rows& r, const Fresh& f, int buf, int lane) {
    Half::copy(a.v.p, a.unit, r.v, a.vu_token, (1 << a.log_page) >= TK, r, f.v, ring + buf * 2 * HALF + HALF, lane);
  }
  __device__ __forceinline__ void read_row(uint32_t row, int sl, float (&x)[EPL]) {
#pragma unroll
    for (int c = 0; c < C::CPL; ++c)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(x[4 * c]), "=f"(x[4 * c + 1]), "=f"(x[4 * c + 2]), "=f"(x[4 * c + 3]) : "r"(row + (c * LPK + sl) * 16) : "memory");
  }
  __device__ __forceinline__ void scores(int buf, int lane) {
    const int sub = lane / LPK, sl = lane % LPK;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float k[EPL];
      read_row(ring + buf * 2 * HALF + (u * KPW + sub) * HD * 4, sl, k);
#pragma unroll
      for (int r = 0; r < NREP; ++r) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < EPL; ++e) d = fmaf(q[r][e], k[e], d);
#pragma unroll
        for (int off = LPK / 2; off > 0; off >>= 1) d += __shfl_xor_sync(L3_FULL, d, off);
        s[u][r] = d;
      }
    }
  }
  __device__ __forceinline__ void weigh(uint32_t mask, int lane) {
    const int sub = lane / LPK;
    if (mask != Half::ALL) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!(mask >> (u * KPW + sub) & 1)) {
#pragma unroll
          for (int r = 0; r < NREP; ++r) s[u][r] = -INFINITY;
        }
    }
#pragma unroll
    for (int r = 0; r < NREP; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
      const float from = mx == -INFINITY ? 0.f : mx;
      if (__any_sync(L3_FULL, mx > m[r])) {
        const float alpha = expf(m[r] - from);
        l[r] *= alpha;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] *= alpha;
        m[r] = mx;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][r] = expf(s[u][r] - from);
        l[r] += s[u][r];
      }
    }
  }
  __device__ __forceinline__ void add_values(int buf, int lane) {
    const int sub = lane / LPK, sl = lane % LPK;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[EPL];
      read_row(ring + buf * 2 * HALF + HALF + (u * KPW + sub) * HD * 4, sl, v);
#pragma unroll
      for (int r = 0; r < NREP; ++r)
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] = fmaf(s[u][r], v[e], o[r][e]);
    }
  }
  __device__ __forceinline__ void end(const PagedAttnArgs& a, bool whole, const Cursor& c, float* part_o, float2* part_ml, int lane) {
    const int b = c.b, head0 = c.head0(a), heads = c.heads(a);
    const int sub = lane / LPK, sl = lane % LPK;
#pragma unroll
    for (int off = LPK; off < 32; off <<= 1) {
#pragma unroll
      for (int r = 0; r < NREP; ++r) {
        const float mo = __shfl_xor_sync(L3_FULL, m[r], off), lo = __shfl_xor_sync(L3_FULL, l[r], off);
        const float mn = fmaxf(m[r], mo), from = mn == -INFINITY ? 0.f : mn;
        const float wa = expf(m[r] - from), wb = expf(mo - from);
        l[r] = l[r] * wa + lo * wb;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] = o[r][e] * wa + __shfl_xor_sync(L3_FULL, o[r][e], off) * wb;
        m[r] = mn;
      }
    }
    if (sub) return;
#pragma unroll
    for (int r = 0; r < NREP; ++r) {
      if (r >= heads) break;
      const float inv = l[r] == 0.f ? 0.f : 1.0f / l[r];
      const long long oi = ((long long)b * a.H + head0 + r) * HD;
      float* po = part_o + r * HD;
#pragma unroll
      for (int e = 0; e < EPL; e += 4) {
        if (whole) {
          const float x[4] = {o[r][e] * inv, o[r][e + 1] * inv, o[r][e + 2] * inv, o[r][e + 3] * inv};
          store_out(a, oi + C::dim(sl, e), x);
        } else *reinterpret_cast<float4*>(po + C::dim(sl, e)) = make_float4(o[r][e], o[r][e + 1], o[r][e + 2], o[r][e + 3]);
      }
      if (sl == 0) {
        if (!whole) part_ml[r] = make_float2(m[r], l[r]);
        else if (a.lse) a.lse[(long long)b * a.H + head0 + r] = m[r] + logf(l[r]);
      }
    }
  }
};

// what a warp's lanes tell one another
template <int AHEAD> struct Mail {
  Fresh fresh;
  Home home[AHEAD];
};

// A warp's stretch of the row of tiles: from tile C on, which begins at unit pos, as far as tiles begin ahead of unit `stop`.  At the end of
// every item's part: end(core, its last tile, its first tile here, whether that is the item's end, whether it is the stretch's first, the unit
// behind it).
template <typename Core, typename T, bool STEP, typename End>
__device__ __forceinline__ void stretch(const PagedAttnArgs& a, Cursor C, int pos, int stop, uint8_t* core_smem, Mail<Core::AHEAD>& mail, int warp, int lane,
                                        End end) {
  constexpr int TK = Core::TK;
  Cursor L = C;      // the tile whose rows are looked up next
  int load_pos = pos;
  int entry = 0;     // the page of this lane's key there
  auto look = [&] {
    const int pos = L.t * TK + (lane & (TK - 1));
    entry = L.b < a.B && pos < L.len ? __ldg(table_of<STEP>(a, L.b) + (pos >> a.log_page)) : -1;
  };
  auto rows = [&](Rows& r, int buf) {
    const int pos = L.t * TK + (lane & (TK - 1)), g = L.g;
    const bool ok = pos < L.len && (unsigned)entry < (unsigned)a.n_pages;
    const uint32_t in = pos & ((1 << a.log_page) - 1);
    r.k = ok ? (uint32_t)entry * a.ku_page + in * a.ku_token + g * a.ku_head : 0u;
    r.v = ok ? (uint32_t)entry * a.vu_page + in * a.vu_token + g * a.vu_head : 0u;
    r.mask = __ballot_sync(L3_FULL, ok) & (uint32_t)((1ull << TK) - 1);
    r.fresh = r.writes = -1;
    // the tile of the new token, unless that lies behind the table: its row comes from k_new / v_new, and goes to its page
    if (!STEP && a.k_new && L.t == L.nt - 1 && asked_length<STEP>(a, L.b) == L.len) {
      const int row = (L.len - 1) & (TK - 1);
      r.fresh = row;
      const char* kn = (const char*)((const T*)a.k_new + L.b * a.kn_sb + g * a.kn_sh);
      const char* vn = (const char*)((const T*)a.v_new + L.b * a.vn_sb + g * a.vn_sh);
      __syncwarp();
      if (lane == 0) mail.fresh = Fresh{kn, vn};
      __syncwarp();
      // its page gets them from the tile, where they have arrived by then
      r.writes = r.mask >> row & 1 && L.blk == 0 ? row : -1;
      if (lane == row) mail.home[buf] = Home{r.k, r.v};
    }
    load_pos += L.t + 1 < L.nt ? 2 : 3;
    advance<TK, STEP>(a, L);
    look();
  };
  Core core;
  core.memory(core_smem, warp);
  Rows r;
  if (pos < stop) {
    look();
    core.ask_query(a, C, lane);
  }
  uint32_t masks[Core::AHEAD];
  int writes[Core::AHEAD];
#pragma unroll
  for (int j = 0; j < Core::AHEAD; ++j) {
    masks[j] = 0;
    writes[j] = -1;
    const bool some = load_pos < stop;
    if (some) {
      rows(r, j);
      masks[j] = r.mask;
      writes[j] = r.writes;
      core.load_keys(a, r, mail.fresh, j, lane);
    }
    cp_commit();
    if (some) core.load_values(a, r, mail.fresh, j, lane);
    cp_commit();
  }
  if (pos < stop) core.load_query(a, C, lane);
  core.reset(a);
  __syncwarp();
  int t0 = C.t;          // first tile of the present item here
  bool first = true;
  for (int buf = 0; pos < stop; buf = (buf + 1) % Core::AHEAD) {
    const uint32_t mask = masks[0];
    const int write = writes[0];
    Home to{};
    if (write >= 0) {  // ahead of rows(), which may put another tile's there
      to = mail.home[buf];
      __syncwarp();
    }
    const bool more = load_pos < stop, ends = C.t == C.nt - 1;
    pos += ends ? 3 : 2;
    const bool goes_on = pos < stop;
    if (more) rows(r, buf);
    Cursor next = C;
    if (goes_on) advance<TK, STEP>(a, next);
    if (ends && goes_on) core.ask_query(a, next, lane);
#pragma unroll
    for (int j = 0; j + 1 < Core::AHEAD; ++j) {
      masks[j] = masks[j + 1];
      writes[j] = writes[j + 1];
    }
    masks[Core::AHEAD - 1] = r.mask;
    writes[Core::AHEAD - 1] = more ? r.writes : -1;
    cp_wait<2 * Core::AHEAD - 1>();
    __syncwarp();
    core.scores(buf, lane);
    if (write >= 0) Core::Half::write(core.ring + buf * 2 * Core::HALF, write, (char*)row_at(a.k.p, to.k, a.unit), lane);
    __syncwarp();
    if (more) core.load_keys(a, r, mail.fresh, buf, lane);
    cp_commit();
    core.weigh(mask, lane);
    cp_wait<2 * Core::AHEAD - 1>();
    __syncwarp();
    core.add_values(buf, lane);
    if (write >= 0) Core::Half::write(core.ring + buf * 2 * Core::HALF + Core::HALF, write, (char*)row_at(a.v.p, to.v, a.unit), lane);
    __syncwarp();
    if (more) core.load_values(a, r, mail.fresh, buf, lane);
    cp_commit();
    if (ends || !goes_on) {
      end(core, C, t0, ends, first, pos);
      first = false;
      if (goes_on) {
        core.load_query(a, next, lane);
        core.reset(a);
        t0 = 0;
      }
    }
    C = next;
  }
}

template <typename Core, typename T, bool STEP>
__global__ void __launch_bounds__(Core::NW * 32, Core::CTAS) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int HD = Core::HD, TK = Core::TK, NW = Core::NW;
  extern __shared__ __align__(256) uint8_t core_smem[];
  __shared__ Mail<Core::AHEAD> mail[NW];
  __shared__ long long before[NW * 32], of_warp[NW];
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = gridDim.x * NW, w = warp * gridDim.x + blockIdx.x;  // neighbours in the row of tiles on different SMs
  const int items = a.G * a.blocks;

  // The row of tiles in units of half a tile, with one more ahead of every item for its query and its result: items * weight_of of a
  // sequence.  A thread sums a few neighbouring sequences, `before` holds the sums ahead of it.
  const int share = (a.B + NW * 32 - 1) / (NW * 32);
  long long sum = 0;
  for (int b = threadIdx.x * share; b < min(a.B, ((int)threadIdx.x + 1) * share); ++b) sum += weight_of(tiles_of<TK>(length_of<STEP>(a, b)));
  long long run = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(L3_FULL, run, o);
    if (lane >= o) run += x;
  }
  before[threadIdx.x] = run - sum;
  if (lane == 31) of_warp[warp] = run;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) total += of_warp[i];
  total *= items;
  const int per = max(2, (int)quotient(total + W - 1, W));  // 2: no warp between two of an item's has none of its tiles
  // sequences without tokens
  for (int b = w; b < a.B; b += W) {
    if (length_of<STEP>(a, b) > 0) continue;
    const float zero[2] = {0.f, 0.f};
    for (int i = lane; i < a.H * (HD / 2); i += 32) store_out(a, (long long)b * a.H * HD + 2 * i, zero);
    if (a.lse)
      for (int h = lane; h < a.H; h += 32) a.lse[(long long)b * a.H + h] = -INFINITY;
    if (a.by_item)
      for (int i = lane; i < items; i += 32) a.info[(long long)b * items + i] = make_int4(0, 0, 0, 0);
  }
  int4 tail = make_int4(0, 0, 0, 0);  // the item that begins here and goes on in the next warps: first slot, warp, partials, item
  const long long u0 = (long long)per * w;
  if (u0 < total) {
    const int stop = (int)(u0 + per < total ? per : total - u0);
    // the first tile that begins at unit u0 or behind it
    Cursor C{};
    int pos;  // where it begins, from u0 on
    {
      long long ahead = 0;
      int i = 0;
      while (i < NW - 1 && (ahead + of_warp[i]) * items <= u0) ahead += of_warp[i++];
      const uint32_t past = __ballot_sync(L3_FULL, (ahead + before[i * 32 + lane]) * items > u0);
      const int own = i * 32 + (past ? __ffs(past) - 2 : 31);  // the thread in whose sum tile u0 lies (lane 0's own never lies past it)
      long long at = u0 - (ahead + before[own]) * items;
      C.b = own * share;
      long long weight;
      for (;;) {
        C.len = length_of<STEP>(a, C.b);
        C.nt = tiles_of<TK>(C.len);
        weight = weight_of(C.nt);
        if (at < weight * items) break;
        at -= weight * items;
        ++C.b;
      }
      const int gb = (int)quotient(at, (int)weight);
      const int in = (int)(at - gb * weight);
      C.g = gb / a.blocks;
      C.blk = gb - C.g * a.blocks;
      C.t = in / 2 - 1;   // tile t begins at unit 1 + 2 t of its item
      pos = 1 + 2 * (in / 2) - in;
      if (in / 2 == C.nt) ++pos;  // none of this item's tiles: the next one's first
      advance<TK, STEP>(a, C);
    }
    stretch<Core, T, STEP>(a, C, pos, stop, core_smem, mail[warp], warp, lane, [&](Core& core, const Cursor& c, int t0, bool ends, bool first, int behind) {
      const int slot = 2 * w + (first ? 0 : 1);
      core.end(a, t0 == 0 && ends, c, a.part_o + (long long)slot * a.heads_blk * HD, reinterpret_cast<float2*>(a.part_ml) + (long long)slot * a.heads_blk,
               lane);
      if (t0 == 0) {
        // the item's last tile is 2 (nt - 1 - t) units behind this one's beginning: the warp that it begins in
        const int parts = ends ? 0 : 1 + (int)quotient(behind - 2 + 2LL * (c.nt - 1 - c.t), per);
        const int4 in = make_int4(slot, w, parts, c.item(a));
        if (!a.by_item) tail = in;
        else if (lane == 0) a.info[c.item(a)] = in;
      }
    });
  }
  if (!a.by_item && lane == 0) a.info[w] = tail;
}

// Joins the partials of one item and query head.  HD / 4 threads have a partial, with running maximum and sum as in the main loop, so that
// nothing waits for the weights of all; the groups of threads meet in shared memory.
template <int JOIN_T>
__global__ void __launch_bounds__(JOIN_T) paged_join_kernel(const __grid_constant__ PagedAttnArgs a) {
  __shared__ float4 acc[JOIN_T];
  __shared__ float2 ml[JOIN_T];
  pdl_launch();
  pdl_wait();
  const int4 in = a.info[blockIdx.x];
  const int parts = in.z, r = blockIdx.y, tid = threadIdx.x;
  if (parts == 0) return;
  const int items = a.G * a.blocks, b = in.w / items, gb = in.w - b * items, g = gb / a.blocks, blk = gb - g * a.blocks;
  if (r >= min(a.heads_blk, a.nrep - blk * a.heads_blk)) return;
  const int q4 = a.HD / 4, d = tid % q4, grp = tid / q4, ngrp = JOIN_T / q4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  if (grp < ngrp) {
    constexpr int U = 4;
    for (int p0 = grp; p0 < parts; p0 += U * ngrp) {
      float4 x[U];
      float2 y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int p = p0 + u * ngrp;
        const long long row = (long long)(p == 0 ? in.x : 2 * (in.y + p)) * a.heads_blk + r;
        y[u] = p < parts ? *reinterpret_cast<const float2*>(a.part_ml + row * 2) : make_float2(-INFINITY, 0.f);
        x[u] = p < parts ? *reinterpret_cast<const float4*>(a.part_o + row * a.HD + 4 * d) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float mx = m;
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, y[u].x);
      const float from = mx == -INFINITY ? 0.f : mx, keep = expf(m - from);
      m = mx;
      l *= keep;
      o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = expf(y[u].x - from);
        l = fmaf(w, y[u].y, l);
        o.x = fmaf(w, x[u].x, o.x); o.y = fmaf(w, x[u].y, o.y); o.z = fmaf(w, x[u].z, o.z); o.w = fmaf(w, x[u].w, o.w);
      }
    }
    acc[tid] = o;
    if (d == 0) ml[grp] = make_float2(m, l);
  }
  __syncthreads();
  if (grp) return;
  const int used = min(parts, ngrp);
  float mx = m;
  for (int i = 1; i < used; ++i) mx = fmaxf(mx, ml[i].x);
  const float from = mx == -INFINITY ? 0.f : mx;
  float w = expf(m - from);
  l *= w;
  o.x *= w; o.y *= w; o.z *= w; o.w *= w;
  for (int i = 1; i < used; ++i) {
    const float4 x = acc[i * q4 + d];
    w = expf(ml[i].x - from);
    l = fmaf(w, ml[i].y, l);
    o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int head = g * a.nrep + blk * a.heads_blk + r;
  const float out[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  store_out(a, ((long long)b * a.H + head) * a.HD + 4 * d, out);
  if (a.lse && d == 0) a.lse[(long long)b * a.H + head] = mx + logf(l);
}

// Few items: the warps of a cluster of S blocks share an item's tiles and join their partials through one another's shared memory, in the order
// of the keys.  No second launch, no workspace, and no search for where a warp begins.
template <typename Core, typename T, bool STEP>
__global__ void __launch_bounds__(Core::NW * 32, Core::CTAS) paged_item_kernel(const __grid_constant__ PagedAttnArgs a, int S) {
  constexpr int HD = Core::HD, NW = Core::NW, NT = NW * 32, Q4 = HD / 4;
  static_assert(HEADS * HD * 4 <= Core::AHEAD * 2 * Core::HALF, "a warp's partial takes the place of its tiles");
  extern __shared__ __align__(256) uint8_t core_smem[];
  __shared__ Mail<Core::AHEAD> mail[NW];
  __shared__ float2 ml[NW][HEADS];
  __shared__ float4 acc[NT];
  __shared__ float2 acc_ml[NT];
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = blockIdx.x % S, items = a.G * a.blocks;
  Cursor C{};
  C.b = blockIdx.x / S / items;
  const int gb = blockIdx.x / S - C.b * items;
  C.g = gb / a.blocks;
  C.blk = gb - C.g * a.blocks;
  C.len = length_of<STEP>(a, C.b);
  C.nt = tiles_of<Core::TK>(C.len);
  const int parts = S * NW, way = rank * NW + warp, from = (int)((long long)C.nt * way / parts), to = (int)((long long)C.nt * (way + 1) / parts);
  const int heads = C.heads(a), head0 = C.head0(a);
  float* part = reinterpret_cast<float*>(core_smem + warp * Core::AHEAD * 2 * Core::HALF);
  if (lane < HEADS) ml[warp][lane] = make_float2(-INFINITY, 0.f);  // a warp without tiles
  __syncwarp();
  const Cursor item = C;
  C.t = from;
  if (from < to)
    stretch<Core, T, STEP>(a, C, 1 + 2 * from, 1 + 2 * to, core_smem, mail[warp], warp, lane,
                     [&](Core& core, const Cursor& c, int, bool, bool, int) { core.end(a, false, c, part, ml[warp], lane); });
  cluster_sync_all();
  // this block's outputs, groups of four of them each (head, four dimensions): rank, rank + S, ...; a few threads each, which share the partials
  const int mine = (heads * Q4 - rank + S - 1) / S, wide = mine < NT ? mine : NT, groups = wide > 0 ? min(NT / wide, parts) : 0;
  const uint32_t part_at = smem_u32(core_smem), ml_at = smem_u32(&ml[0][0]);
  for (int k0 = 0; k0 < mine; k0 += wide) {
    const int k = k0 + tid % wide, grp = tid / wide, out = rank + S * k, r = out / Q4, d = out - r * Q4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    const bool active = grp < groups && k < mine;
    if (active) {
      for (int p = grp; p < parts; p += groups) {
        const uint32_t off_o = part_at + (p % NW) * Core::AHEAD * 2 * Core::HALF + (r * HD + 4 * d) * 4, off_ml = ml_at + ((p % NW) * HEADS + r) * 8;
        float2 y;
        float4 x;
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(y.x), "=f"(y.y) : "r"(cluster_at(off_ml, p / NW)) : "memory");
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(cluster_at(off_o, p / NW)) : "memory");
        if (y.y == 0.f) continue;  // no key there, and nothing written
        const float mx = fmaxf(m, y.x), base = mx == -INFINITY ? 0.f : mx, keep = expf(m - base), w = expf(y.x - base);
        m = mx;
        l = fmaf(w, y.y, l * keep);
        o.x = fmaf(w, x.x, o.x * keep); o.y = fmaf(w, x.y, o.y * keep); o.z = fmaf(w, x.z, o.z * keep); o.w = fmaf(w, x.w, o.w * keep);
      }
      acc[tid] = o;
      acc_ml[tid] = make_float2(m, l);
    }
    __syncthreads();
    if (active && grp == 0) {
      float mx = m;
      for (int i = 1; i < groups; ++i) mx = fmaxf(mx, acc_ml[i * wide + tid].x);
      const float base = mx == -INFINITY ? 0.f : mx;
      float w = expf(m - base);
      l *= w;
      o.x *= w; o.y *= w; o.z *= w; o.w *= w;
      for (int i = 1; i < groups; ++i) {
        const float4 x = acc[i * wide + tid];
        const float2 y = acc_ml[i * wide + tid];
        w = expf(y.x - base);
        l = fmaf(w, y.y, l);
        o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
      }
      const float inv = l == 0.f ? 0.f : 1.0f / l, v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
      const long long row = (long long)item.b * a.H + head0 + r;
      store_out(a, row * HD + 4 * d, v);
      if (a.lse && d == 0) a.lse[row] = mx + logf(l);
    }
    __syncthreads();
  }
  cluster_sync_all();  // the others may still read here
}

// Few keys an item: P warps of a block have it to themselves and join their partials through the block's shared memory.  As paged_item_kernel's, one
// launch and no search; blocks that end make room for others, so that more items than there are places need no even shares.
template <typename Core, typename T, int P, bool STEP>
__global__ void __launch_bounds__(Core::NW * 32, Core::CTAS) paged_whole_kernel(const __grid_constant__ PagedAttnArgs a) {
  constexpr int HD = Core::HD, NW = Core::NW, Q4 = HD / 4, RING = Core::AHEAD * 2 * Core::HALF;
  extern __shared__ __align__(256) uint8_t core_smem[];
  __shared__ Mail<Core::AHEAD> mail[NW];
  __shared__ float2 ml[NW][HEADS];
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / P, way = warp % P, items = a.G * a.blocks;
  const int id = group * gridDim.x + blockIdx.x;  // neighbours on different SMs
  Cursor C{};
  C.b = id / items;
  if (C.b >= a.B) return;
  const int gb = id - C.b * items;
  C.g = gb / a.blocks;
  C.blk = gb - C.g * a.blocks;
  C.len = length_of<STEP>(a, C.b);
  C.nt = tiles_of<Core::TK>(C.len);
  const int heads = C.heads(a);
  const long long row = (long long)C.b * a.H + C.head0(a);
  if (C.nt == 0) {
    const float zero[2] = {0.f, 0.f};
    for (int i = way * 32 + lane; i < heads * (HD / 2); i += P * 32) store_out(a, row * HD + 2 * i, zero);
    if (a.lse && way == 0 && lane < heads) a.lse[row + lane] = -INFINITY;
    return;
  }
  const int from = C.nt * way / P, to = C.nt * (way + 1) / P;
  if (P > 1 && lane < HEADS) ml[warp][lane] = make_float2(-INFINITY, 0.f);  // a warp without tiles
  __syncwarp();
  C.t = from;
  if (from < to)
    stretch<Core, T, STEP>(a, C, 1 + 2 * from, 1 + 2 * to, core_smem, mail[warp], warp, lane, [&](Core& core, const Cursor& c, int, bool, bool, int) {
      core.end(a, P == 1, c, reinterpret_cast<float*>(core_smem + warp * RING), ml[warp], lane);
    });
  if (P == 1) return;
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(P * 32) : "memory");
  for (int i = way * 32 + lane; i < heads * Q4; i += P * 32) {
    const int r = i / Q4, d = i - r * Q4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) m = fmaxf(m, ml[group * P + p][r].x);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float2 y = ml[group * P + p][r];
      if (y.y == 0.f) continue;  // no key there, and nothing written
      const float4 x = *reinterpret_cast<const float4*>(core_smem + (group * P + p) * RING + (r * HD + 4 * d) * 4);
      const float w = expf(y.x - base);
      l = fmaf(w, y.y, l);
      o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l, v[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    store_out(a, (row + r) * HD + 4 * d, v);
    if (a.lse && d == 0) a.lse[row + r] = m + logf(l);
  }
}

cudaError_t launch_join(const PagedAttnArgs& a, int n_sm, cudaStream_t s) {
  g_l3_pdl_next = true;  // the joining launch starts in the tail of the first
  // few items have many partials each, and leave the SMs room for larger blocks
  if (a.n_info * a.heads_blk <= 2 * n_sm) return launch_k(paged_join_kernel<512>, dim3(a.n_info, a.heads_blk), dim3(512), 0, s, a);
  return launch_k(paged_join_kernel<128>, dim3(a.n_info, a.heads_blk), dim3(128), 0, s, a);
}
template <typename Core, typename T, int P, bool STEP> cudaError_t launch_whole(const PagedAttnArgs& a, long long items, cudaStream_t s) {
  const cudaError_t e = allow_smem(paged_whole_kernel<Core, T, P, STEP>, Core::SMEM);
  if (e != cudaSuccess) return e;
  constexpr int groups = Core::NW / P;
  return launch_k(paged_whole_kernel<Core, T, P, STEP>, dim3((unsigned)((items + groups - 1) / groups)), dim3(Core::NW * 32), Core::SMEM, s, a);
}
template <typename Core, typename T, bool STEP>
cudaError_t launch_core(PagedAttnArgs a, int n_sm, cudaStream_t s, int& launches) {
  const int W = n_sm * Core::CTAS * Core::NW;
  const long long items = (long long)a.B * a.G * a.blocks;
  a.by_item = items <= W;
  a.n_info = (int)(a.by_item ? items : W);
  cudaError_t e;
  // Items by themselves where their longest possible keys (what the table is wide) are few tiles: of eight tiles a warp at most, 1 - 4 warps of a
  // block.  One launch : both, us, by items (W warps have room) and tiles: bf16, head size 128, W 1776: 256 4 5.0 : 7.9, 16 8.8 : 10.7, 32 14.5 : 16.5; 512
  // 4 7.6 : 11.9, 16 14.7 : 18.0, 32 22.0 : 25.8; 1600 4 10.7 : 19.6, 16 30.1 : 38.1, 32 44.0 : 57.2.  fp32, head size 48, W 2368: 768 4 6.5 : 9.7, 16 12.7 :
  // 15.3; 1536 4 7.6 : 12.3, 16 21.1 : 22.5, 32 31.2 : 34.0; one of 16 tiles among 1535 of one 10.5 : 8.9.  More items than warps: 2000 (head size 64) 4
  // 15.7 : 20.5, 8000 4 45 : 52, 12800 2 42 : 36, 2048 8 23.8 : 22.1.
  const long long tiles = (((long long)a.max_pages << a.log_page) + Core::TK - 1) / Core::TK;
  int S = 1, P = 1;
  while (S < 8 && items * S <= n_sm) S *= 2;
  while (P < Core::NW && (items * 2 * P <= W || tiles > 8 * P)) P *= 2;
  launches = 1;
  if (tiles <= (S > 1 ? 2 * Core::NW : items <= W ? 8 * P : items <= 4 * W ? 4 : 0))
    return P == 1 ? launch_whole<Core, T, 1, STEP>(a, items, s) : P == 2 ? launch_whole<Core, T, 2, STEP>(a, items, s) : launch_whole<Core, T, Core::NW, STEP>(a, items, s);
  // Fewer items than SMs: a cluster of S blocks an item.  Clusters : blocks as above : two launches, by items of S blocks and tiles: bf16, head size
  // 128, 8 of 8 8 6.9 : 5.4, 16 7.0 : 8.2, 44 8.5 : - : 8.6, 125 11.2 : - : 11.3; 32 of 4 16 7.6 : 8.3; 120 of 2 16 8.3 : 8.6; 128 of 2 32 10.6 : 12.6 : 13.6.
  if (S > 1 && tiles <= 4 * S * Core::NW) {
    if ((e = allow_smem(paged_item_kernel<Core, T, STEP>, Core::SMEM)) != cudaSuccess) return e;
    return launch_kc(paged_item_kernel<Core, T, STEP>, dim3((unsigned)(items * S)), dim3(Core::NW * 32), Core::SMEM, s, S, a, S);
  }
  launches = 2;
  e = allow_smem(paged_attn_kernel<Core, T, STEP>, Core::SMEM);
  if (e == cudaSuccess) e = launch_k(paged_attn_kernel<Core, T, STEP>, dim3(n_sm * Core::CTAS), dim3(Core::NW * 32), Core::SMEM, s, a);
  if (e != cudaSuccess) return e;
  return launch_join(a, n_sm, s);
}
template <int HD, bool STEP> cudaError_t launch_f32(const PagedAttnArgs& a, int n_sm, cudaStream_t s, int& launches) {
  if (a.heads_blk == 1) return launch_core<F32Core<HD, 1>, float, STEP>(a, n_sm, s, launches);
  if (a.heads_blk == 2) return launch_core<F32Core<HD, 2>, float, STEP>(a, n_sm, s, launches);
  if constexpr (HD == 48 || HD == 96) return launch_core<F32Core<HD, 4>, float, STEP>(a, n_sm, s, launches);
  else if (a.heads_blk <= 4) return launch_core<F32Core<HD, 4>, float, STEP>(a, n_sm, s, launches);
  else return launch_core<F32Core<HD, 8>, float, STEP>(a, n_sm, s, launches);
}
template <typename T, int HD, bool STEP> cudaError_t launch_mma(const PagedAttnArgs& a, int n_sm, cudaStream_t s, int& launches) {
  if constexpr (!STEP)  // a step's queries are of the cache's type
    if (a.q_dtype == L3_DTYPE_F32) return launch_core<MmaCore<T, HD, true>, T, false>(a, n_sm, s, launches);
  return launch_core<MmaCore<T, HD, false>, T, STEP>(a, n_sm, s, launches);
}
template <int HD, bool STEP> cudaError_t launch_hd(const PagedAttnArgs& a, int n_sm, cudaStream_t s, int& launches) {
  if (a.kv_dtype == L3_DTYPE_F32) return launch_f32<HD, STEP>(a, n_sm, s, launches);
  if (a.kv_dtype == L3_DTYPE_BF16) return launch_mma<bf16, HD, STEP>(a, n_sm, s, launches);
  return launch_mma<__half, HD, STEP>(a, n_sm, s, launches);
}
// the pools' offsets in units of the largest power of two of bytes (16 at least) that divides every stride: 32 bits of them
bool set_units(PagedAttnArgs& a) {
  const int size = a.kv_dtype == L3_DTYPE_F32 ? 4 : 2;
  unsigned long long bits = 0;
  for (const PagedPool* p : {&a.k, &a.v}) bits |= (unsigned long long)p->sp | (unsigned long long)p->sh | (unsigned long long)p->st;
  bits = bits * size | 1ull << 20;
  int shift = 0;
  while (!(bits >> shift & 1)) ++shift;
  a.unit = 1 << shift;
  uint32_t* to[2][3] = {{&a.ku_page, &a.ku_head, &a.ku_token}, {&a.vu_page, &a.vu_head, &a.vu_token}};
  for (int i = 0; i < 2; ++i) {
    const PagedPool& p = i ? a.v : a.k;
    const unsigned long long last = ((unsigned long long)(a.n_pages - 1) * p.sp + (unsigned long long)(a.G - 1) * p.sh + ((1ull << a.log_page) - 1) * p.st) * size >> shift;
    if (last >> 32) return false;
    *to[i][0] = (uint32_t)((unsigned long long)p.sp * size >> shift);
    *to[i][1] = (uint32_t)((unsigned long long)p.sh * size >> shift);
    *to[i][2] = (uint32_t)((unsigned long long)p.st * size >> shift);
  }
  return true;
}
// query heads that share a reading of their keys: as many as registers hold (fp32, head sizes 48 and 96: 12 dimensions per lane)
int heads_of_item(int H, int G, int HD, int kv_dtype) {
  const int most = kv_dtype == L3_DTYPE_F32 && (HD == 48 || HD == 96) ? HEADS / 2 : HEADS;
  return H / G < most ? H / G : most;
}
template <bool STEP> cudaError_t launch_attention(PagedAttnArgs a, int n_sm, cudaStream_t s, int& launches) {
  const int W = n_sm * MOST_WARPS;
  set_units(a);
  const int size = a.q_dtype == L3_DTYPE_F32 ? 4 : 2;
  a.q_vec = (((uintptr_t)a.q | (uintptr_t)(a.q_sb * size) | (uintptr_t)(a.q_sh * size)) & 15) == 0;
  a.heads_blk = heads_of_item(a.H, a.G, a.HD, a.kv_dtype);
  a.nrep = a.H / a.G;
  a.blocks = (a.nrep + a.heads_blk - 1) / a.heads_blk;
  a.info = (int4*)a.ws;
  a.part_o = (float*)(a.info + W);
  a.part_ml = a.part_o + (size_t)2 * W * a.heads_blk * a.HD;
  switch (a.HD) {
    case 16: return launch_hd<16, STEP>(a, n_sm, s, launches);
    case 32: return launch_hd<32, STEP>(a, n_sm, s, launches);
    case 48: return launch_hd<48, STEP>(a, n_sm, s, launches);
    case 64: return launch_hd<64, STEP>(a, n_sm, s, launches);
    case 96: return launch_hd<96, STEP>(a, n_sm, s, launches);
    case 128: return launch_hd<128, STEP>(a, n_sm, s, launches);
    default: return cudaErrorInvalidValue;
  }
}
}  // namespace

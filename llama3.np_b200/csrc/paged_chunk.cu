// Attention of the rows of a packed step over a key / value cache in pages (L3PagedChunk):
//   s_j = scale q_t . k_j,  o_t = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse_t = m + log sum_j e^(s_j - m),  m = max_j s_j
// over the tokens j that row t sees, j <= its position.  paged_chunk.cuh says how the work is cut.
//
// This file: fp32 caches; and the join of what several CTAs have of an item.  Products as three of TF32 numbers on the tensor cores (mma.sync): a number is
// the nearest one of 11 bits and what that leaves, cut to 11 bits, and x y = xh yh + xh yl + xl yh is off by at most 2^-20 of it - where numbers'
// second parts are not below fp32's normal ones, from 2^-115 on.  (With FFMA what shared memory delivers bounded the kernel, 3200 wavefronts a tile of
// 64 x 64 with heads of 48 in place of 800: 64 prompts of up to 220 tokens, 6 heads of 48, 88 us, now 54.  There
// the tensor pipe is busy for a quarter of the time and 39 % of the issue slots are used: three warps a scheduler wait for one another's products.)
// A CTA's four warps hold 16 rows each and walk their keys, 64 at a time.  Keys and values come row by row through the page table, 16 bytes a
// copy, while the tile before is worked on; rows of no token become zeros.  Rows of tiles are padded to an odd number of 16-byte pieces: eight rows'
// pieces (scores, ldmatrix), and eight columns of four rows two apart (output), lie on different banks.  The weights stay in registers: the lane that has
// row g's keys 2 t and 2 t + 1 takes them for the product's t-th and t + 4-th, in whose place the values' rows are read.
#include <limits.h>

#include <algorithm>

#include "paged_chunk.cuh"
#include "paged_chunk_tc.h"

namespace {
using namespace chunk;
constexpr int TR = 64, BK = 64, NT = 128;
__host__ __device__ constexpr Split f32_split() { return Split{BK, 1, 16, 8, 8}; }
// as registers and shared memory have room for; of heads of 48, three : four: 61.9 : 62.9 us (four's registers spill)
constexpr int ctas_of_sm(int HD) { return HD > 64 ? 2 : 3; }
template <int HD> constexpr int row_ld() { return HD + 4; }
template <int HD> constexpr size_t smem_bytes() { return (size_t)3 * 64 * row_ld<HD>() * 4 + 2 * 2 * BK * 8 + 2 * 8; }

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {  // zeros where !take
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the nearest number of 11 bits, and what that leaves, cut to 11 bits
__device__ __forceinline__ void two_parts(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) & 0xffffe000u;
}
__device__ __forceinline__ void mma_parts(float (&c)[4], const uint32_t (&ah)[4], const uint32_t (&al)[4], uint32_t b0, uint32_t b1) {
  uint32_t h0, l0, h1, l1;
  two_parts(b0, h0, l0);
  two_parts(b1, h1, l1);
  mma_tf32(c, al, h0, h1);
  mma_tf32(c, ah, l0, l1);
  mma_tf32(c, ah, h0, h1);
}

template <int HD>
__global__ void __launch_bounds__(NT, ctas_of_sm(HD)) chunk_f32_kernel(const ChunkArgs a) {
  constexpr Split SPLIT = f32_split();
  constexpr int LD = row_ld<HD>(), KS = HD / 8;
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                     // [64][LD]
  float* sK = sQ + 64 * LD;           // [64][LD]
  float* sV = sK + 64 * LD;           // [64][LD]
  long long* sOff = reinterpret_cast<long long*>(sV + 64 * LD);  // [turn][k, v][64]
  unsigned* sThere = reinterpret_cast<unsigned*>(sOff + 2 * 2 * BK);  // [turn][2] bits of keys that there are
  __shared__ long long room[NT / 32 + 1];
  __shared__ Place place;
  pdl_launch();
  pdl_wait();
  clear_rest<float>(a, threadIdx.x, NT);
  find_share<BK, NT>(a, SPLIT, room, &place);
  if (threadIdx.x == 0) leave_nothing(a, place);
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const float sc = a.scale * 1.4426950408889634f;
  auto token_of = [&](int f) { return a.R == 1 ? f : f / a.R; };
  Cursor<BK> c;
  if (!c.start(a, SPLIT, place)) return;
  do {
    const int* table = a.table + c.b * a.table_stride;
    const int flat0 = c.tile * TR, flats = c.r.n * a.R, row0 = flat0 + warp * 16;
    const int most = c.r.seen(token_of(min(flats, flat0 + TR) - 1));   // keys that any of the rows sees
    const int ours = row0 < flats ? c.r.seen(token_of(min(flats, row0 + 16) - 1)) : 0;  // that any of this warp's rows sees
    // the rows' queries; not where there are no keys: such copies would be in no group, so that nothing waited for them, and the next item's go to the same place
    for (int i = threadIdx.x; c.j0 < c.j1 && i < TR * (HD / 4); i += NT) {
      const int r = i / (HD / 4), p = i - r * (HD / 4), f = flat0 + r, t = token_of(f);
      const bool in = f < flats;
      cp16(smem_u32(sQ + r * LD + p * 4), in ? (const float*)a.q + (c.r.s0 + t) * a.q_st + (c.g * a.R + f - t * a.R) * a.q_sh + p * 4 : (const float*)a.q, in);
    }
    auto offsets = [&](int j) {  // by the first 64 threads
      if (threadIdx.x >= BK) return;
      const int key = j * BK + threadIdx.x, turn = j & 1;
      int page = -1;
      if (key < most) page = table[key >> a.log_page];
      const bool there = (unsigned)page < (unsigned)a.n_pages;
      const long long in = key & ((1 << a.log_page) - 1);
      sOff[turn * 2 * BK + threadIdx.x] = there ? page * a.k.sp + c.g * a.k.sh + in * a.k.st : -1;
      sOff[turn * 2 * BK + BK + threadIdx.x] = there ? page * a.v.sp + c.g * a.v.sh + in * a.v.st : -1;
      const unsigned bits = __ballot_sync(L3_FULL, there);
      if (lane == 0) sThere[turn * 2 + warp] = bits;
    };
    auto copy = [&](int j, bool value) {
      const long long* off = sOff + (j & 1) * 2 * BK + (value ? BK : 0);
      const float* pool = (const float*)(value ? a.v.p : a.k.p);
      float* dst = value ? sV : sK;
      constexpr int PIECES = HD / 4;
      for (int i = threadIdx.x; i < BK * PIECES; i += NT) {
        const int r = i / PIECES, p = i - r * PIECES;
        const long long at = off[r];
        cp16(smem_u32(dst + r * LD + p * 4), at >= 0 ? pool + at + p * 4 : pool, at >= 0);
      }
      cp_commit();
    };
    int seen[2];
    float o[KS][4], m[2], l[2];   // of rows g and g + 8: columns 8 n + 2 t4, + 1
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int f = row0 + g + 8 * i;
      seen[i] = f < flats ? c.r.seen(token_of(f)) : INT_MAX;  // a row behind the last: what it has goes nowhere
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < KS; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    if (c.j0 < c.j1) {
      offsets(c.j0);
      __syncthreads();
      copy(c.j0, false);
      copy(c.j0, true);
    }
    for (int j = c.j0; j < c.j1; ++j) {
      if (j + 1 < c.j1) offsets(j + 1);
      cp_wait<1>();
      __syncthreads();   // the keys are there, and the next ones' places
      const int left = ours - j * BK;  // what lies behind is not multiplied (56 us for 60)
      float s[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      if (left > 0) {
        // ldmatrix of 8 rows of 4 numbers: lane i has row i / 4's number i % 4
        const uint32_t qa = smem_u32(sQ + (warp * 16 + (lane & 15)) * LD + (lane >> 4) * 4);
        const uint32_t ka = smem_u32(sK + ((lane >> 4) * 8 + (lane & 7)) * LD + (lane >> 3 & 1) * 4);
#pragma unroll 2
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t q[4], qh[4], ql[4];
          ldsm_x4(qa + ks * 32, q);
#pragma unroll
          for (int i = 0; i < 4; ++i) two_parts(q[i], qh[i], ql[i]);
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            if (8 * n >= left) break;
            uint32_t k[4];
            ldsm_x4(ka + n * 8 * LD * 4 + ks * 32, k);
            mma_parts(s[n], qh, ql, k[0], k[1]);
            mma_parts(s[n + 1], qh, ql, k[2], k[3]);
          }
        }
      }
      const unsigned there[2] = {sThere[(j & 1) * 2], sThere[(j & 1) * 2 + 1]};
      __syncthreads();   // all have read the keys
      if (j + 1 < c.j1) copy(j + 1, false);
      else cp_commit();
      if (left > 0) {
        const bool masked = __any_sync(L3_FULL, min(seen[0], seen[1]) - j * BK < BK) || (there[0] & there[1]) != L3_FULL;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& x = s[n][2 * i + e];
              x *= sc;
              if (masked) {
                const int key = 8 * n + 2 * t4 + e;
                if (!(j * BK + key < seen[i] && (there[n / 4] >> (key & 31) & 1))) x = -INFINITY;
              }
              mx = fmaxf(mx, x);
            }
          mx = fmaxf(mx, __shfl_xor_sync(L3_FULL, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(L3_FULL, mx, 2));
          const float mn = fmaxf(m[i], mx), from = mn == -INFINITY ? 0.f : mn;
          if (__any_sync(L3_FULL, mn > m[i])) {
            const float alpha = ex2(m[i] - from);
            l[i] *= alpha;
#pragma unroll
            for (int n = 0; n < KS; ++n) {
              o[n][2 * i] *= alpha;
              o[n][2 * i + 1] *= alpha;
            }
          }
          m[i] = mn;
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) l[i] += s[n][2 * i + e] = ex2(s[n][2 * i + e] - from);
        }
      }
      cp_wait<1>();
      __syncthreads();   // the values are there
      if (left > 0) {
        const float* va = sV + 2 * t4 * LD + g;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          if (8 * n >= left) break;
          const uint32_t p[4] = {__float_as_uint(s[n][0]), __float_as_uint(s[n][2]), __float_as_uint(s[n][1]), __float_as_uint(s[n][3])};
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) two_parts(p[i], ph[i], pl[i]);
#pragma unroll
          for (int d = 0; d < KS; ++d) mma_parts(o[d], ph, pl, __float_as_uint(va[8 * n * LD + 8 * d]), __float_as_uint(va[(8 * n + 1) * LD + 8 * d]));
        }
      }
      __syncthreads();   // all have read the values
      if (j + 1 < c.j1) copy(j + 1, true);
      else cp_commit();
    }
    cp_wait<0>();
    // the result, or this CTA's part of it
    const bool whole = c.whole();
    float* part_o = whole ? nullptr : a.part_o + (size_t)(2 * blockIdx.x + c.slot()) * TR * HD;
    float2* part_ml = whole ? nullptr : a.part_ml + (size_t)(2 * blockIdx.x + c.slot()) * TR;
    if (!whole && threadIdx.x == 0) left_of(a, blockIdx.x).part[c.slot()] = make_int4(c.b, c.tile, c.g, c.j1 == c.nb);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int in_tile = warp * 16 + g + 8 * i, f = flat0 + in_tile;
      l[i] += __shfl_xor_sync(L3_FULL, l[i], 1);
      l[i] += __shfl_xor_sync(L3_FULL, l[i], 2);
      bool finite = l[i] < INFINITY;
#pragma unroll
      for (int n = 0; n < KS; ++n) finite = finite && fabsf(o[n][2 * i]) < INFINITY && fabsf(o[n][2 * i + 1]) < INFINITY;
      if (f < flats) {
        if (!finite && whole) left_of(a, blockIdx.x).odd = 1;
        const int t = token_of(f);
        const long long at = (long long)(c.r.s0 + t) * a.H + c.g * a.R + f - t * a.R;
        const float by = !whole ? 1.f : l[i] == 0.f ? 0.f : 1.f / l[i];
        float* to = whole ? (float*)a.out + at * HD : part_o + in_tile * HD;
#pragma unroll
        for (int n = 0; n < KS; ++n) *reinterpret_cast<float2*>(to + 8 * n + 2 * t4) = make_float2(o[n][2 * i] * by, o[n][2 * i + 1] * by);
        if (t4 == 0) {
          if (!whole) part_ml[in_tile] = make_float2(m[i], l[i]);
          else if (a.lse) a.lse[at] = (m[i] + log2f(l[i])) * 0.6931471805599453f;
        }
      }
    }
    __syncthreads();
  } while (c.next(a, SPLIT));
}

// ---------------------------------------------------------------------------------------------------------------- the join
// Block (c, y) joins 16 rows of the item that CTA c began and others ended, o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, and looks after
// the rows of all its items that are not finite.  A thread has four columns of a row: most items are in two or three CTAs, and a warp a row took
// four times as many instructions (48 requests over 8 kv heads of 64: 96 us for 100 in all).
constexpr int JROWS = 16, JT = 256, MOST_CTAS = 1024;
__device__ __forceinline__ void store4(float* to, const float (&o)[4]) { *reinterpret_cast<float4*>(to) = make_float4(o[0], o[1], o[2], o[3]); }
template <typename T> __device__ __forceinline__ void store4(T* to, const float (&o)[4]) {
  struct alignas(8) Four { T x[4]; } four{down<T>(o[0]), down<T>(o[1]), down<T>(o[2]), down<T>(o[3])};
  *reinterpret_cast<Four*>(to) = four;
}
template <typename T, int HD, int BK>
__global__ void __launch_bounds__(JT) chunk_join_kernel(const ChunkArgs a, const Split sp) {
  constexpr int N = (HD + 31) / 32, UNITS = HD / 4;
  __shared__ int list[MOST_CTAS];  // the item's partials, 2 CTA + slot, in the order of the keys
  __shared__ int parts;
  __shared__ unsigned odd_rows;
  pdl_launch();
  pdl_wait();
  const int TR = a.tile_rows;
  const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Left& own = left_of(a, c0);
  const int4 first = own.part[1];
  if (first.x >= 0) {
    const Request r = request(a, first.x);
    const int row0 = blockIdx.y * JROWS, rows = min(JROWS, r.n * a.R - first.y * TR - row0);  // of the tile
    if (rows > 0) {
      if (warp == 0) {  // the CTAs behind, a lane each; those that ended nothing and went on with nothing have no part
        int n = 1;
        for (int c = c0 + 1; c < a.n_cta; c += 32) {
          const int4 its = c + lane < a.n_cta ? left_of(a, c + lane).part[0] : make_int4(-1, 0, 0, 0);
          const unsigned ends = __ballot_sync(L3_FULL, its.x >= 0 && its.w);
          const unsigned has = __ballot_sync(L3_FULL, its.x >= 0 && (!ends || lane < __ffs(ends)));
          if (has >> lane & 1) list[n + __popc(has & ((1u << lane) - 1))] = 2 * (c + lane);
          n += __popc(has);
          if (ends) break;
        }
        if (lane == 0) {
          list[0] = 2 * c0 + 1;
          parts = n;
          odd_rows = 0;
        }
      }
      __syncthreads();
      const int n = parts;
      for (int u = threadIdx.x; u < rows * UNITS; u += JT) {
        const int i = u / UNITS, d = (u - i * UNITS) * 4, in_tile = row0 + i, f = first.y * TR + in_tile;
        const int t = f / a.R, head = first.z * a.R + f - t * a.R;
        float o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll 4
        for (int k = 0; k < n; ++k) m = fmaxf(m, a.part_ml[(size_t)list[k] * TR + in_tile].x);
        const float from = m == -INFINITY ? 0.f : m;
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const size_t at = (size_t)list[k] * TR + in_tile;
          const float2 ml = a.part_ml[at];
          const float4 x = *reinterpret_cast<const float4*>(a.part_o + at * HD + d);
          const float by = ex2(ml.x - from);
          l += ml.y * by;
          o[0] += x.x * by;
          o[1] += x.y * by;
          o[2] += x.z * by;
          o[3] += x.w * by;
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bool odd = !(l < INFINITY);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          odd = odd || !(fabsf(o[e]) < INFINITY);
          o[e] *= inv;
        }
        const long long at = (long long)(r.s0 + t) * a.H + head;
        store4((T*)a.out + at * HD + d, o);
        if (a.lse && d == 0) a.lse[at] = (m + log2f(l)) * 0.6931471805599453f;
        if (odd) atomicOr(&odd_rows, 1u << i);
      }
      __syncthreads();
      for (int i = warp; i < rows; i += JT / 32) {
        if (!(odd_rows >> i & 1)) continue;
        const int f = first.y * TR + row0 + i, t = f / a.R;
        by_formula<T, HD>(a, first.x, first.z, r.s0 + t, first.z * a.R + f - t * a.R, r.seen(t));
      }
    }
  }
  if (!own.odd) return;
  Cursor<BK> c;
  if (c.start(a, sp, own.place)) do {
    if (!c.whole()) continue;
    for (int i = warp; i < JROWS; i += JT / 32) {
      const int f = c.tile * TR + blockIdx.y * JROWS + i;
      if (f >= c.r.n * a.R) break;
      const int t = f / a.R, head = c.g * a.R + f - t * a.R;
      const T* out = (const T*)a.out + ((long long)(c.r.s0 + t) * a.H + head) * HD;
      bool odd = false;
#pragma unroll
      for (int x = 0; x < N; ++x) odd = odd || (lane + 32 * x < HD && !(fabsf(up(out[lane + 32 * x])) < INFINITY));
      if (__any_sync(L3_FULL, odd)) by_formula<T, HD>(a, c.b, c.g, c.r.s0 + t, head, c.r.seen(t));
    }
  } while (c.next(a, sp));
}

size_t partials(int n_cta, int rows, int HD) { return (size_t)n_cta * (2 * rows * ((size_t)HD * 4 + 8) + sizeof(Left)) + PART_ALIGN; }
template <typename T, int BK> cudaError_t join_t(const ChunkArgs& a, const Split& sp, cudaStream_t s) {
  const dim3 grid(a.n_cta, a.tile_rows / JROWS), block(JT);
  g_l3_pdl_next = true;
  switch (a.HD) {
    case 16: return launch_k(chunk_join_kernel<T, 16, BK>, grid, block, 0, s, a, sp);
    case 32: return launch_k(chunk_join_kernel<T, 32, BK>, grid, block, 0, s, a, sp);
    case 48: return launch_k(chunk_join_kernel<T, 48, BK>, grid, block, 0, s, a, sp);
    case 64: return launch_k(chunk_join_kernel<T, 64, BK>, grid, block, 0, s, a, sp);
    case 96: return launch_k(chunk_join_kernel<T, 96, BK>, grid, block, 0, s, a, sp);
    default: return launch_k(chunk_join_kernel<T, 128, BK>, grid, block, 0, s, a, sp);
  }
}
template <int HD> cudaError_t launch_hd(ChunkArgs a, int n_sm, cudaStream_t s) {
  constexpr size_t smem = smem_bytes<HD>();
  a.n_cta = std::min(ctas_of_sm(HD) * n_sm, MOST_CTAS);
  a.tile_rows = TR;
  a.part_o = part_begin(a.ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)a.n_cta * 2 * TR * HD);
  a.left = a.part_ml + (size_t)a.n_cta * 2 * TR;
  cudaError_t e = allow_smem(chunk_f32_kernel<HD>, smem);
  if (e != cudaSuccess) return e;
  if ((e = launch_k(chunk_f32_kernel<HD>, dim3(a.n_cta), dim3(NT), smem, s, a)) != cudaSuccess) return e;
  return join_t<float, BK>(a, f32_split(), s);
}
}  // namespace

cudaError_t launch_chunk_join_tc(const ChunkArgs& a, cudaStream_t s) {
  return a.dtype == L3_DTYPE_BF16 ? join_t<bf16, TC_BK>(a, tc_split(a.HD), s) : join_t<__half, TC_BK>(a, tc_split(a.HD), s);
}

namespace {
// Few rows over few keys as single tokens (paged_packed.cu), which read their request's keys anew each.  us, so : as tiles, 32 heads over 8 kv heads of 128, one
// request, by rows x keys and what is read: bf16 5 x 1505 29 MB 13.9 : 23.0, 16 x 1516 95 MB 23.0 : 23.4, 8 x 6008 188 MB 34.4 : 29.2, 2 x 60002 469 MB 88 : 63;
// fp32 5 x 1505 59 MB 22 : 32, 5 x 6005 235 MB 49 : 65, 16 x 316 40 MB 19 : 28, 16 x 1516 190 MB 43 : 34, 16 x 6016 752 MB 130 : 67.  (That path writes every row.)
bool as_single_tokens(const ChunkArgs& a) {
  const long long size = a.dtype == L3_DTYPE_F32 ? 4 : 2, keys = (long long)a.max_pages << a.log_page;
  return a.clear_rest == 1 && a.B > 0 && a.T <= 16 && a.T * keys * a.G * a.HD * 2 * size <= (size == 4 ? 256LL : 128LL) << 20;
}
PagedAttnArgs single_tokens(const ChunkArgs& a) {
  PagedAttnArgs p{};
  p.q = a.q; p.q_sb = a.q_st; p.q_sh = a.q_sh; p.q_dtype = p.kv_dtype = p.out_dtype = a.dtype;
  p.k = a.k; p.v = a.v; p.n_pages = a.n_pages; p.log_page = a.log_page;
  p.table = a.table; p.table_stride = a.table_stride; p.max_pages = a.max_pages; p.lengths = a.lengths; p.starts = a.starts; p.requests = a.B;
  p.B = a.T; p.H = a.H; p.G = a.G; p.HD = a.HD; p.scale = a.scale; p.out = a.out; p.lse = a.lse; p.ws = a.ws;
  return p;
}
}  // namespace

// of whichever kernels a call takes, and either number of rows
size_t paged_chunk_workspace(int H, int G, int HD, int dtype, int n_sm) {
  return std::max(dtype == L3_DTYPE_F32 ? partials(ctas_of_sm(HD) * n_sm, TR, HD) : partials(n_sm, 256, HD), paged_attn_workspace(H, G, HD, n_sm));
}

cudaError_t launch_paged_chunk(ChunkArgs a, int n_sm, cudaStream_t s) {
  if (as_single_tokens(a)) {
    const PagedAttnArgs p = single_tokens(a);
    if (paged_attn_fits(p)) return launch_paged_attention(p, n_sm, s);
  }
  if (a.dtype != L3_DTYPE_F32) return launch_paged_chunk_tc(a, n_sm, s);
  switch (a.HD) {
    case 16: return launch_hd<16>(a, n_sm, s);
    case 32: return launch_hd<32>(a, n_sm, s);
    case 48: return launch_hd<48>(a, n_sm, s);
    case 64: return launch_hd<64>(a, n_sm, s);
    case 96: return launch_hd<96>(a, n_sm, s);
    case 128: return launch_hd<128>(a, n_sm, s);
    default: return cudaErrorInvalidValue;
  }
}

// Attention of the rows of a packed step over a key / value cache in pages (L3PagedChunk):
//   s_j = scale q_t . k_j,  o_t = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse_t = m + log sum_j e^(s_j - m),  m = max_j s_j
// over the tokens j that row t sees, j <= its position.  paged_chunk.cuh says how the work is cut.
//
// This file: fp32 caches, the products as FFMA; and the join of what several CTAs have of an item.
// A CTA's 256 threads hold 64 rows and walk their keys, 64 at a time.  Keys and values come row by row through the page table, 16 bytes a
// copy, while the tile before is worked on; rows of no token become zeros.
//   scores   a thread has 4 rows x 4 keys, summed as even and odd entries (pairs: fma2); rows padded to an odd number of 16-byte pieces
//   output   a thread has 4 rows x HD / 16 columns, in pairs of rows; the weights arrive through shared memory, [key][row]
#include <algorithm>

#include "paged_chunk.cuh"
#include "paged_chunk_tc.h"

namespace {
using namespace chunk;
constexpr int TR = 64, BK = 64, NT = 256;
__host__ __device__ constexpr Split fma_split() { return Split{BK, 4, 8, TR, 3}; }
constexpr int ctas_of_sm(int HD) { return HD > 64 ? 1 : HD > 48 ? 2 : 3; }  // as shared memory has room for
template <int HD> constexpr int row_ld() { return HD + 4; }
template <int HD> constexpr size_t smem_bytes() { return (size_t)(2 * 64 * row_ld<HD>() + 64 * HD + 64 * (TR + 4)) * 4 + 2 * 2 * BK * 8 + 2 * 8 + 16; }

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {  // zeros where !take
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int HD>
__global__ void __launch_bounds__(NT, ctas_of_sm(HD)) chunk_fma_kernel(const ChunkArgs a) {
  using T = float;
  constexpr Split SPLIT = fma_split();
  constexpr int LD = row_ld<HD>(), PL = TR + 4;
  constexpr int CW = HD % 64 == 0 ? 4 : HD % 32 == 0 ? 2 : 1, NC = HD / (16 * CW);  // columns side by side, and how often
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;                     // [64][LD]
  float* sK = sQ + 64 * LD;           // [64][LD]
  float* sV = sK + 64 * LD;           // [64][HD]
  float* sP = sV + 64 * HD;           // [keys][rows]
  long long* sOff = reinterpret_cast<long long*>(sP + 64 * PL);  // [turn][k, v][64]
  unsigned* sThere = reinterpret_cast<unsigned*>(sOff + 2 * 2 * BK);  // [turn][2] bits of keys that there are
  __shared__ long long room[NT / 32 + 1];
  __shared__ Place place;
  pdl_launch();
  pdl_wait();
  clear_rest<T>(a, threadIdx.x, NT);
  find_share<BK, NT>(a, SPLIT, room, &place);
  if (threadIdx.x == 0) leave_nothing(a, place);
  __syncthreads();
  const int lane = threadIdx.x & 31, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float sc = a.scale * 1.4426950408889634f;
  auto token_of = [&](int f) { return a.R == 1 ? f : f / a.R; };
  Cursor<BK> c;
  if (!c.start(a, SPLIT, place)) return;
  do {
    const int* table = a.table + c.b * a.table_stride;
    const int flat0 = c.tile * TR, flats = c.r.n * a.R;
    const int most = c.r.seen(token_of(min(flats, flat0 + TR) - 1));   // keys that any of the rows sees
    for (int i = threadIdx.x; i < TR * (HD / 4); i += NT) {  // the rows' queries
      const int r = i / (HD / 4), p = i - r * (HD / 4), f = flat0 + r, t = token_of(f);
      const bool in = f < flats;
      cp16(smem_u32(sQ + r * LD + p * 4), in ? (const T*)a.q + (c.r.s0 + t) * a.q_st + (c.g * a.R + f - t * a.R) * a.q_sh + p * 4 : (const T*)a.q, in);
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
      if (lane == 0) sThere[turn * 2 + (threadIdx.x >> 5)] = bits;
    };
    auto copy = [&](int j, bool value) {
      const long long* off = sOff + (j & 1) * 2 * BK + (value ? BK : 0);
      const T* pool = (const T*)(value ? a.v.p : a.k.p);
      float* dst = value ? sV : sK;
      const int ld = value ? HD : LD;
      constexpr int PIECES = HD / 4;
      for (int i = threadIdx.x; i < BK * PIECES; i += NT) {
        const int r = i / PIECES, p = i - r * PIECES;
        const long long at = off[r];
        cp16(smem_u32(dst + r * ld + p * 4), at >= 0 ? pool + at + p * 4 : pool, at >= 0);
      }
      cp_commit();
    };
    int seen[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = flat0 + ty * 4 + i;
      seen[i] = f < flats ? c.r.seen(token_of(f)) : 0;
    }
    float2 o[2][NC * CW];   // pairs of rows
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
#pragma unroll
    for (int x = 0; x < NC * CW; ++x) o[0][x] = o[1][x] = make_float2(0.f, 0.f);
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
      float2 s2[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) s2[i][k] = make_float2(0.f, 0.f);
#pragma unroll 2
      for (int d = 0; d < HD; d += 4) {
        float4 q[4], k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(sQ + (ty * 4 + i) * LD + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const float4*>(sK + (tx + 16 * i) * LD + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s2[i][x] = fma2(make_float2(q[i].x, q[i].y), make_float2(k[x].x, k[x].y), s2[i][x]);
            s2[i][x] = fma2(make_float2(q[i].z, q[i].w), make_float2(k[x].z, k[x].w), s2[i][x]);
          }
      }
      const unsigned there0 = sThere[(j & 1) * 2], there1 = sThere[(j & 1) * 2 + 1];
      __syncthreads();   // all have read the keys
      if (j + 1 < c.j1) copy(j + 1, false);
      else cp_commit();
      float p[4][4], alpha[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = tx + 16 * x;
          const bool in = j * BK + key < seen[i] && ((x < 2 ? there0 : there1) >> (key & 31) & 1);
          p[i][x] = in ? (s2[i][x].x + s2[i][x].y) * sc : -INFINITY;
          mx = fmaxf(mx, p[i][x]);
        }
#pragma unroll
        for (int w = 8; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(L3_FULL, mx, w));
        const float mn = fmaxf(m[i], mx), from = mn == -INFINITY ? 0.f : mn;
        alpha[i] = ex2(m[i] - from);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) sum += p[i][x] = ex2(p[i][x] - from);
#pragma unroll
        for (int w = 8; w; w >>= 1) sum += __shfl_xor_sync(L3_FULL, sum, w);
        l[i] = l[i] * alpha[i] + sum;
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) *reinterpret_cast<float4*>(sP + (tx + 16 * x) * PL + ty * 4) = make_float4(p[0][x], p[1][x], p[2][x], p[3][x]);
#pragma unroll
      for (int x = 0; x < NC * CW; ++x) {
        o[0][x].x *= alpha[0]; o[0][x].y *= alpha[1];
        o[1][x].x *= alpha[2]; o[1][x].y *= alpha[3];
      }
      cp_wait<1>();
      __syncthreads();   // the values are there, and the weights
#pragma unroll 2
      for (int k = 0; k < BK; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(sP + k * PL + ty * 4);
        const float2 w01 = make_float2(w.x, w.y), w23 = make_float2(w.z, w.w);
        float v[NC * CW];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          const float* at = sV + k * HD + n * 16 * CW + tx * CW;
          if constexpr (CW == 4) {
            const float4 x = *reinterpret_cast<const float4*>(at);
            v[n * 4] = x.x; v[n * 4 + 1] = x.y; v[n * 4 + 2] = x.z; v[n * 4 + 3] = x.w;
          } else if constexpr (CW == 2) {
            const float2 x = *reinterpret_cast<const float2*>(at);
            v[n * 2] = x.x; v[n * 2 + 1] = x.y;
          } else v[n] = *at;
        }
#pragma unroll
        for (int x = 0; x < NC * CW; ++x) {
          o[0][x] = fma2(w01, make_float2(v[x], v[x]), o[0][x]);
          o[1][x] = fma2(w23, make_float2(v[x], v[x]), o[1][x]);
        }
      }
      __syncthreads();   // all have read the values and the weights
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
    for (int i = 0; i < 4; ++i) {
      const int f = flat0 + ty * 4 + i;
      float y[NC * CW];
      bool finite = l[i] < INFINITY;
#pragma unroll
      for (int x = 0; x < NC * CW; ++x) {
        y[x] = i & 1 ? o[i / 2][x].y : o[i / 2][x].x;
        finite = finite && fabsf(y[x]) < INFINITY;
      }
      if (f < flats) {
        if (!finite && whole) left_of(a, blockIdx.x).odd = 1;
        const int t = token_of(f);
        const long long at = (long long)(c.r.s0 + t) * a.H + c.g * a.R + f - t * a.R;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int e = 0; e < CW; ++e) {
            const int d = n * 16 * CW + tx * CW + e;
            if (whole) ((T*)a.out)[at * HD + d] = down<T>(y[n * CW + e] * inv);
            else part_o[(ty * 4 + i) * HD + d] = y[n * CW + e];
          }
        if (tx == 0) {
          if (!whole) part_ml[ty * 4 + i] = make_float2(m[i], l[i]);
          else if (a.lse) a.lse[at] = (m[i] + log2f(l[i])) * 0.6931471805599453f;
        }
      }
    }
    __syncthreads();
  } while (c.next(a, SPLIT));
}

// ---------------------------------------------------------------------------------------------------------------- the join
// Block (c, y) joins 16 rows of the item that CTA c began and others ended, o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, and looks after
// the rows of all its items that are not finite.
constexpr int JROWS = 16, JT = 256;
template <typename T, int HD, int BK>
__global__ void __launch_bounds__(JT) chunk_join_kernel(const ChunkArgs a, const Split sp) {
  pdl_launch();
  pdl_wait();
  constexpr int N = (HD + 31) / 32;
  const int TR = a.tile_rows;
  const int c0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Left& own = left_of(a, c0);
  const int4 first = own.part[1];
  if (first.x >= 0) {
    const Request r = request(a, first.x);
    for (int i = warp; i < JROWS; i += JT / 32) {
      const int in_tile = blockIdx.y * JROWS + i, f = first.y * TR + in_tile;
      if (f >= r.n * a.R) break;
      const int t = f / a.R, head = first.z * a.R + f - t * a.R;
      const long long at = (long long)(r.s0 + t) * a.H + head;
      float o[N], m, l;
      const size_t p0 = (size_t)(2 * c0 + 1) * TR + in_tile;
      m = a.part_ml[p0].x;
      l = a.part_ml[p0].y;
#pragma unroll
      for (int x = 0; x < N; ++x) o[x] = lane + 32 * x < HD ? a.part_o[p0 * HD + lane + 32 * x] : 0.f;
      // the CTAs behind, 32 at a time, a lane each; those that ended nothing and went on with nothing have no part
      for (int c = c0 + 1;; c += 32) {
        const int4 its = c + lane < a.n_cta ? left_of(a, c + lane).part[0] : make_int4(-1, 0, 0, 0);
        const unsigned ends = __ballot_sync(L3_FULL, its.x >= 0 && its.w);
        const bool part = its.x >= 0 && (!ends || lane < __ffs(ends));
        float2 ml = make_float2(-INFINITY, 0.f);
        if (part) ml = a.part_ml[(size_t)(2 * (c + lane)) * TR + in_tile];
        const float mn = fmaxf(m, warp_max(ml.x)), from = mn == -INFINITY ? 0.f : mn;
        const float f0 = exp2f(m - from), fp = exp2f(ml.x - from);
        l = l * f0 + warp_sum(ml.y * fp);
        m = mn;
#pragma unroll
        for (int x = 0; x < N; ++x) o[x] *= f0;
        unsigned list = __ballot_sync(L3_FULL, part);
        while (list) {
          float f[4], y[4][N];
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // four partials' rows on their way together
            const int of = list ? __ffs(list) - 1 : -1;
            list &= list - 1;
            f[k] = __shfl_sync(L3_FULL, fp, max(of, 0));
#pragma unroll
            for (int x = 0; x < N; ++x)
              y[k][x] = of >= 0 && lane + 32 * x < HD ? a.part_o[((size_t)(2 * (c + of)) * TR + in_tile) * HD + lane + 32 * x] : 0.f;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < N; ++x) o[x] += y[k][x] * f[k];
        }
        if (ends || c + 32 >= a.n_cta) break;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bool odd = !(l < INFINITY);
#pragma unroll
      for (int x = 0; x < N; ++x) {
        odd = odd || !(fabsf(o[x]) < INFINITY);
        if (lane + 32 * x < HD) ((T*)a.out)[at * HD + lane + 32 * x] = down<T>(o[x] * inv);
      }
      if (a.lse && lane == 0) a.lse[at] = (m + log2f(l)) * 0.6931471805599453f;
      if (__any_sync(L3_FULL, odd)) by_formula<T, HD>(a, first.x, first.z, r.s0 + t, head, r.seen(t));
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

size_t partials(int n_cta, int rows, int HD) { return (size_t)n_cta * (2 * rows * ((size_t)HD * 4 + 8) + sizeof(Left)); }
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
  a.n_cta = ctas_of_sm(HD) * n_sm;
  a.tile_rows = TR;
  a.part_o = (float*)a.ws;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)a.n_cta * 2 * TR * HD);
  a.left = a.part_ml + (size_t)a.n_cta * 2 * TR;
  cudaError_t e = allow_smem(chunk_fma_kernel<HD>, smem);
  if (e != cudaSuccess) return e;
  if ((e = launch_k(chunk_fma_kernel<HD>, dim3(a.n_cta), dim3(NT), smem, s, a)) != cudaSuccess) return e;
  return join_t<float, BK>(a, fma_split(), s);
}
}  // namespace

cudaError_t launch_chunk_join_tc(const ChunkArgs& a, cudaStream_t s) {
  return a.dtype == L3_DTYPE_BF16 ? join_t<bf16, TC_BK>(a, tc_split(a.HD), s) : join_t<__half, TC_BK>(a, tc_split(a.HD), s);
}

namespace {
// Few rows over few keys as single tokens (paged.cu), which read their request's keys anew each.  us, so : as tiles, 32 heads over 8 kv heads of 128, one
// request, by rows x keys and what is read: bf16 5 x 1505 29 MB 14.2 : 23.0, 16 x 1516 95 MB 23.0 : 23.4, 8 x 6008 188 MB 34.4 : 29.2, 2 x 60002 469 MB 88 : 63;
// fp32 5 x 6005 235 MB 50 : 75, 8 x 6008 376 MB 72 : 78, 16 x 6016 752 MB 130 : 82.  (That path writes every row.)
bool as_single_tokens(const ChunkArgs& a) {
  const long long size = a.dtype == L3_DTYPE_F32 ? 4 : 2, keys = (long long)a.max_pages << a.log_page;
  return a.clear_rest && a.B > 0 && a.T <= 16 && a.T * keys * a.G * a.HD * 2 * size <= (size == 4 ? 384LL : 128LL) << 20;
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

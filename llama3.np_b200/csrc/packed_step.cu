// A packed step's bookkeeping on the device, and rotary positions with the writing of keys and values to their slots.
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "packed.h"

namespace {
// ------------------------------------------------------------------------------------------- tables, positions and slots
// Request b gets n_b = min(count_b, what is left of the T rows) rows and ceil((len_b + n_b) / P) - ceil(len_b / P) pages: two running sums over
// the requests.  Bound by latency: lengths and counts, a page number, the results - three trips to memory.  Every CTA runs both sums
// over all requests by itself (ET threads, a stretch of neighbouring requests each), keeps them per thread in shared memory, and finds the requests
// of its own rows there; a second launch or a wait between CTAs would cost more than the sums.  The row of a new page's first token writes
// the page into the table.  32 requests of one token each 3.6 us, 301 requests with 10000 rows between them 4.1, of which 2.2 are any launch's.
constexpr int ET = 512;
__device__ __forceinline__ int positive(int x) { return x > 0 ? x : 0; }

// exclusive sum over the block; `all`: the whole sum
__device__ __forceinline__ long long scan(long long x, long long* warps, long long& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long run = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(L3_FULL, run, o);
    if (lane >= o) run += y;
  }
  __syncthreads();  // `warps` may still be read
  if (lane == 31) warps[warp] = run;
  __syncthreads();
  long long before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < ET / 32; ++w) {
    if (w < warp) before += warps[w];
    all += warps[w];
  }
  return before + run - x;
}
struct Request {  // what its rows need to know
  int len, n;       // tokens it had, rows it gets
  int had, pages;   // pages then and now
};
__device__ __forceinline__ Request request(const PagedExtendArgs& a, int b, long long rows_before) {
  Request r;
  r.len = positive(a.lengths[b]);
  const long long most = min((long long)a.T - rows_before, (long long)INT_MAX - r.len);  // a length stays an int
  r.n = (int)max(min((long long)a.counts[b], most), 0LL);
  const long long page = 1LL << a.log_page;
  r.had = (int)((r.len + page - 1) >> a.log_page);
  r.pages = (int)((r.len + (long long)r.n + page - 1) >> a.log_page);
  return r;
}
__global__ void __launch_bounds__(ET) paged_extend_kernel(const PagedExtendArgs a) {
  __shared__ long long warps[ET / 32];
  __shared__ long long rows_at[ET], pages_at[ET];   // ahead of a thread's first request
  pdl_launch();
  pdl_wait();
  const int each = (a.B + ET - 1) / ET, b0 = min((int)threadIdx.x * each, a.B), b1 = min(b0 + each, a.B);
  long long sum = 0, all_rows, all_pages;
  // rows that requests ask for; the cut to T comes in with the sums (it never takes a row from one ahead of another that keeps one)
  for (int b = b0; b < b1; ++b) sum += min(positive(a.counts[b]), INT_MAX - positive(a.lengths[b]));
  const long long row0 = scan(sum, warps, all_rows);
  sum = 0;
  long long at = row0;
  for (int b = b0; b < b1; ++b) {
    const Request r = request(a, b, min(at, (long long)a.T));
    at += min(positive(a.counts[b]), INT_MAX - r.len);
    sum += r.pages - r.had;
  }
  const long long page0 = scan(sum, warps, all_pages);
  rows_at[threadIdx.x] = row0;
  pages_at[threadIdx.x] = page0;
  __syncthreads();
  if (blockIdx.x == 0) {
    at = row0;
    for (int b = b0; b < b1; ++b) {
      const Request r = request(a, b, min(at, (long long)a.T));
      a.out_starts[b] = (int)min(at, (long long)a.T);
      a.out_lengths[b] = r.len + r.n;
      at += min(positive(a.counts[b]), INT_MAX - r.len);
    }
    if (threadIdx.x == 0) {
      a.out_starts[a.B] = (int)min(all_rows, (long long)a.T);
      *a.out_used = (int)min(all_pages, (long long)INT_MAX);
    }
  }
  const int threads = (a.B + each - 1) / max(each, 1);  // that have requests
  for (long long t = (long long)blockIdx.x * ET + threadIdx.x; t < a.T; t += (long long)gridDim.x * ET) {
    int position = -1;
    long long slot = -1;
    if (t < all_rows) {
      int lo = 0, hi = threads - 1;      // the last thread whose requests begin at or ahead of row t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (rows_at[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      int b = lo * each;
      long long start = rows_at[lo], pages = pages_at[lo];
      Request r = request(a, b, start);
      while (t >= start + r.n) {
        start += r.n;
        pages += r.pages - r.had;
        r = request(a, ++b, start);
      }
      position = r.len + (int)(t - start);
      const int column = position >> a.log_page, in = position & ((1 << a.log_page) - 1);
      int page = -1;
      if (column < r.had) {
        if (column < a.max_pages) page = a.table[b * a.table_stride + column];
      } else {
        const long long i = pages + column - r.had;
        if (i < a.n_free) page = a.free_pages[i];
        if (column < a.max_pages) {
          if (in == 0) a.table[b * a.table_stride + column] = page;
        } else page = -1;
      }
      if (page >= 0) slot = ((long long)page << a.log_page) + in;
    }
    a.out_positions[t] = position;
    a.out_slots[t] = slot;
  }
}

// ------------------------------------------------------------------------------------------------------ rotary positions
// (a, b) -> (a cos - b sin, b cos + a sin).  Bound by the rows' bytes, in once and out once.  A CTA takes TOK rows with all their heads: the angles are
// taken once for all heads, in 64 bits as parts of a whole turn - position * frequency / 2 pi less its nearest integer, so that far positions lose
// nothing - and go as cosines and sines to shared memory; then a thread turns two pieces of E entries at a time.  8191 rows of 32 + 8 heads of 128 in bf16, keys
// and values to their slots: 39.2 us, 5.1 TB/s (79 % of a copy's rate), 70 % of the issue slots.  A step's 32 rows: 3.6 us, latency.
constexpr int RT = 256;
template <typename T> __device__ __forceinline__ float up(T x) { return to_f32(x); }
template <> __device__ __forceinline__ float up<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T down(float x) { return from_f32<T>(x); }
template <> __device__ __forceinline__ __half down<__half>(float x) { return __float2half_rn(x); }

template <typename T, int E> struct alignas(sizeof(T) * E) Entries { T v[E]; };

template <typename T, int E, int TOK>
__global__ void __launch_bounds__(RT) rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turn[];   // [TOK][dims / 2]: cosine, sine
  __shared__ int at[TOK];            // the rows' positions, if anything is turned
  using En = Entries<T, E>;
  const long long row0 = (long long)blockIdx.x * TOK, rows = (long long)a.B * a.L;
  const int half = a.dims / 2;
  pdl_launch();
  pdl_wait();
  for (int i = threadIdx.x; i < TOK * half; i += RT) {
    const int t = i / half, p = i - t * half;
    const int position = row0 + t < rows ? a.positions[row0 + t] : -1;
    float2 cs = make_float2(1.f, 0.f);
    if (position >= 0) {
      double x = position * (a.freqs[p] * 0.15915494309189535);
      x -= rint(x);
      float s, c;
      sincospif((float)(x + x), &s, &c);
      cs = make_float2(c * a.amplitude, (a.inverse ? -s : s) * a.amplitude);
    }
    turn[i] = cs;
    if (p == 0) at[t] = position;
  }
  __syncthreads();
  const int turned = half / E, tail = (a.D - a.dims) / E, units = turned + (tail + 1) / 2;  // of a head: two pieces each, the last perhaps one
  const int per = (a.H + 2 * a.G) * units;
  for (int i = threadIdx.x; i < TOK * per; i += RT) {
    const int t = i / per, rest = i - t * per, head = rest / units, u = rest - head * units;
    const long long row = row0 + t;
    if (row >= rows) break;
    const T* from;
    T* to;
    bool rotate = u < turned && at[t] >= 0;  // the others are copied: a product with 1 and 0 would make NaN of an infinite entry's partner
    if (head < a.H) {
      const long long b = row / a.L, l = row - b * a.L;
      from = (const T*)a.x + b * a.x_sb + l * a.x_st + head * a.x_sh;
      to = (T*)a.out + b * a.o_sb + l * a.o_st + head * a.o_sh;
    } else {
      const int g = head - a.H < a.G ? head - a.H : head - a.H - a.G;
      const bool value = head - a.H >= a.G;
      const long long slot = a.slots[row];
      if ((unsigned long long)slot >= (unsigned long long)a.n_pages << a.log_page) continue;
      const PagedPool& p = value ? a.vp : a.kp;
      from = value ? (const T*)a.v + row * a.v_st + g * a.v_sh : (const T*)a.k + row * a.k_st + g * a.k_sh;
      to = (T*)p.p + (slot >> a.log_page) * p.sp + g * p.sh + (slot & ((1LL << a.log_page) - 1)) * p.st;
      rotate = rotate && !value;
    }
    int first, second;
    bool two = true;
    if (u < turned) {
      first = a.layout ? u * E : 2 * u * E;
      second = a.layout ? half + u * E : first + E;
    } else {
      first = a.dims + 2 * (u - turned) * E;
      second = first + E;
      two = second < a.D;
    }
    En x = *reinterpret_cast<const En*>(from + first), y{};
    if (two) y = *reinterpret_cast<const En*>(from + second);
    if (rotate) {
      const float2* cs = turn + t * half + u * E;
      if (a.layout || E == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float p = up(x.v[e]), q = up(y.v[e]);
          x.v[e] = down<T>(p * cs[e].x - q * cs[e].y);
          y.v[e] = down<T>(q * cs[e].x + p * cs[e].y);
        }
      } else {
#pragma unroll
        for (int e = 0; e + 1 < E; e += 2) {
          const float p = up(x.v[e]), q = up(x.v[e + 1]), r = up(y.v[e]), w = up(y.v[e + 1]);
          const float2 c0 = cs[e / 2], c1 = cs[E / 2 + e / 2];
          x.v[e] = down<T>(p * c0.x - q * c0.y);
          x.v[e + 1] = down<T>(q * c0.x + p * c0.y);
          y.v[e] = down<T>(r * c1.x - w * c1.y);
          y.v[e + 1] = down<T>(w * c1.x + r * c1.y);
        }
      }
    }
    *reinterpret_cast<En*>(to + first) = x;
    if (two) *reinterpret_cast<En*>(to + second) = y;
  }
}
template <typename T, int E> cudaError_t rotary_e(const RotaryArgs& a, int n_sm, cudaStream_t s) {
  const long long rows = (long long)a.B * a.L;
  const size_t per = (size_t)a.dims / 2 * sizeof(float2);
  // rows of a CTA, us, one : four: 600 of 40 heads of 128 in bf16 5.9 : 7.8, 1000 9.2 : 8.1, 3000 17.2 : 16.3, 8000 38 : 34; 1001 of 16 fp32 heads of 96, 24 entries
  // turned, 4.0 : 4.5 (a row has few pieces there, which the rule does not look at)
  if (rows >= 6LL * n_sm) return launch_k(rotary_kernel<T, E, 4>, dim3((unsigned)((rows + 3) / 4)), dim3(RT), 4 * per, s, a);
  return launch_k(rotary_kernel<T, E, 1>, dim3((unsigned)rows), dim3(RT), per, s, a);
}
// entries of a piece: as many as divide what is turned and what is not, and as every address and stride allows
template <typename T> cudaError_t rotary_t(const RotaryArgs& a, int n_sm, cudaStream_t s) {
  uint64_t bits = (uint64_t)(a.dims / 2) | (uint64_t)(a.D - a.dims);
  if (a.H) bits |= (uint64_t)a.x_st | a.x_sh | a.o_st | a.o_sh | a.x_sb | a.o_sb | ((uintptr_t)a.x / sizeof(T)) | ((uintptr_t)a.out / sizeof(T));
  if (a.G)
    bits |= (uint64_t)a.k_st | a.k_sh | a.v_st | a.v_sh | a.kp.sp | a.kp.sh | a.kp.st | a.vp.sp | a.vp.sh | a.vp.st | ((uintptr_t)a.k / sizeof(T)) |
            ((uintptr_t)a.v / sizeof(T)) | ((uintptr_t)a.kp.p / sizeof(T)) | ((uintptr_t)a.vp.p / sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (!(bits & 7)) return rotary_e<T, 8>(a, n_sm, s);
  if (!(bits & 3)) return rotary_e<T, 4>(a, n_sm, s);
  if (!(bits & 1)) return rotary_e<T, 2>(a, n_sm, s);
  return rotary_e<T, 1>(a, n_sm, s);
}
}  // namespace

cudaError_t launch_paged_extend(const PagedExtendArgs& a, int n_sm, cudaStream_t s) {
  const int ctas = (int)min((long long)n_sm, max(1LL, ((long long)a.T + ET - 1) / ET));
  return launch_k(paged_extend_kernel, dim3(ctas), dim3(ET), 0, s, a);
}

cudaError_t launch_rotary(const RotaryArgs& a, int n_sm, cudaStream_t s) {
  if (a.dtype == L3_DTYPE_F32) return rotary_t<float>(a, n_sm, s);
  if (a.dtype == L3_DTYPE_BF16) return rotary_t<bf16>(a, n_sm, s);
  return rotary_t<__half>(a, n_sm, s);
}

// Moving rows: keys and values of new tokens into the pages of a cache, whole pages to other pages, beams' states to the beams that
// continue them.  No arithmetic: bound by the bytes, each read once and written once, 16 bytes a thread where the addresses allow it.
// Measured (B200), and the share of what a copy reaches: 1201 pages of 32 KB in each of 16 pools 193 us (99.6 %); prompts of 7 sequences of up to
// 2047 tokens (8 kv heads of 128, bf16; 67 MB) 14.0 us (73 %; padded rows' CTAs leave at once, and the launch takes 2.4 us of it); six tensors of
// 64 rows of 1 MB, half of them changed, 67.8 us (91 %).  The smallest calls are a launch: 2.4 - 3.5 us.
#include <stdint.h>

#include "../../include/llama3_b200.h"
#include "paged.h"

namespace {
// ------------------------------------------------------------------------------------------------ new tokens into pages
// A token is 2 G HD values, `per` pieces of 16 bytes; a CTA takes TOK tokens of one sequence, a thread the same piece of several.
constexpr int WT = 256, TOK = 8;
__global__ void __launch_bounds__(WT, 4) paged_write_kernel(const PagedWriteArgs a) {
  pdl_launch();
  pdl_wait();
  const int b = blockIdx.y, per = 2 * a.G * a.pieces;
  const int side = per < WT ? WT / per : 1;            // tokens side by side
  const int lane_tok = per < WT ? threadIdx.x / per : 0;
  if (lane_tok >= side) return;
  const int n = a.count ? min(a.count[b], a.L) : a.L, start = a.start[b];
  const int t0 = blockIdx.x * TOK * side + lane_tok;
  if (t0 >= n) return;
  for (int c = per < WT ? threadIdx.x % per : threadIdx.x; c < per; c += WT) {
    const int half = c / (per / 2), in = c % (per / 2), g = in / a.pieces, piece = in % a.pieces;
    const char* src = half ? (const char*)a.v + b * a.v_sb + g * a.v_sh : (const char*)a.k + b * a.k_sb + g * a.k_sh;
    const long long st = half ? a.v_st : a.k_st;
    const PagedPool& p = half ? a.vp : a.kp;
    src += piece * 16;
    char* const to = (char*)p.p + g * p.sh + piece * 16;
    const int* row = a.table + b * a.table_stride;
    const int cap = a.max_pages << a.log_page;
#pragma unroll
    for (int i0 = 0; i0 < TOK; i0 += 4) {
      uint4 x[4];
      int page[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + (i0 + i) * side;
        const unsigned pos = (unsigned)start + t;  // a start near 2^31, or below 0, lies behind the table
        const bool ok = t < n && pos < (unsigned)cap;
        page[i] = ok ? __ldg(row + (pos >> a.log_page)) : -1;
        if (ok) x[i] = ldg_stream16(src + t * st);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((unsigned)page[i] >= (unsigned)a.n_pages) continue;
        const unsigned pos = (unsigned)start + t0 + (i0 + i) * side;
        *reinterpret_cast<uint4*>(to + page[i] * p.sp + (pos & ((1u << a.log_page) - 1)) * p.st) = x[i];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ whole rows
struct Div {  // division by a number fixed for a launch (Granlund and Montgomery's round-up method), operands below 2^31
  unsigned d, mul, sh;
};
Div make_div(unsigned d) {
  unsigned sh = 0;
  while ((1ull << sh) < d) ++sh;
  return Div{d, (unsigned)(((1ull << 32) * ((1ull << sh) - d)) / d + 1), sh};
}
__device__ __forceinline__ unsigned divide(unsigned x, const Div& v) { return v.sh ? (unsigned)(((unsigned long long)__umulhi(x, v.mul) + x) >> v.sh) : x; }

template <typename V> struct Piece {
  __device__ static __forceinline__ V load(const char* p) { return *reinterpret_cast<const V*>(p); }
};
template <> struct Piece<uint4> {
  __device__ static __forceinline__ uint4 load(const char* p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
  }
};

// A launch's tensors with their divisors, as a kernel's parameter: of up to eight tensors 0.5 KB of it in place of 4 (a call of two pools on the
// host 6.1 us with the long one for every call).
template <int MAX> struct Tensors {
  RowsDesc t[MAX];
  Div row[MAX], run[MAX];
};
template <int MAX> Tensors<MAX> tensors_of(const RowsList& l, int n) {
  Tensors<MAX> p;
  for (int i = 0; i < n; ++i) {
    p.t[i] = l.t[i];
    p.row[i] = make_div(l.t[i].outer * l.t[i].run);
    p.run[i] = make_div(l.t[i].run);
  }
  return p;
}
constexpr int CT = 256, CU = 8;  // threads, and pieces of a thread
template <typename V, int MAX>
__global__ void __launch_bounds__(CT) copy_rows_kernel(const __grid_constant__ Tensors<MAX> l, const int* src, const int* dst, int n, int rows) {
  pdl_launch();
  pdl_wait();
  const RowsDesc& d = l.t[blockIdx.y];
  const unsigned per = d.outer * d.run;
  const unsigned long long all = (unsigned long long)per * n, base = (unsigned long long)blockIdx.x * CT * CU;
  if (base >= all) return;
  // pairs are counted from the one that the block begins in, so that the division stays within 32 bits
  const unsigned first = (unsigned)(base / per), off = (unsigned)(base - (unsigned long long)first * per);
  V x[CU];
  char* to[CU];
#pragma unroll
  for (int i = 0; i < CU; ++i) {
    const unsigned at = off + i * CT + threadIdx.x;
    const unsigned pr = divide(at, l.row[blockIdx.y]), rem = at - pr * per, o = divide(rem, l.run[blockIdx.y]), c = rem - o * d.run;
    to[i] = nullptr;
    if (first + pr < (unsigned)n) {
      const int s = __ldg(src + first + pr), t = __ldg(dst + first + pr);
      if ((unsigned)s < (unsigned)rows && (unsigned)t < (unsigned)rows) {
        const long long in = o * d.outer_stride + (long long)c * (int)sizeof(V);
        x[i] = Piece<V>::load(d.base + s * d.row_stride + in);
        to[i] = d.base + t * d.row_stride + in;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < CU; ++i)
    if (to[i]) *reinterpret_cast<V*>(to[i]) = x[i];
}

// A thread has the same pieces of all K rows of a group: it copies those of every row that another one wants into its own places in shared
// memory and then writes the rows that change, so that any permutation works in place without a barrier and without a copy elsewhere.
// RU pieces a turn, asynchronously, the next turn's on their way while one is written, keep enough bytes moving.
template <typename V> __device__ __forceinline__ void fetch(V* to, const char* from) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (sizeof(V) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(from) : "memory");
  else if constexpr (sizeof(V) >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(from), "n"((int)sizeof(V)) : "memory");
  else *to = *reinterpret_cast<const V*>(from);
}
template <typename V, int MAX>
__global__ void reorder_rows_kernel(const __grid_constant__ Tensors<MAX> l, const int* parents, int B, int K, int RU, int turns) {
  extern __shared__ __align__(16) uint8_t places_raw[];
  V* mine = reinterpret_cast<V*>(places_raw) + threadIdx.x;  // [2][RU][K][blockDim.x] (one turn: [RU]...)
  __shared__ unsigned char wanted[ROWS_BEAMS];
  __shared__ short need[ROWS_BEAMS], to[ROWS_BEAMS], from[ROWS_BEAMS];
  __shared__ int needs, moves;
  pdl_launch();
  pdl_wait();
  const RowsDesc& d = l.t[blockIdx.z];
  const unsigned per = d.outer * d.run, step = blockDim.x * RU;
  if (blockIdx.x * step * turns >= per) return;
  const int b = blockIdx.y;
  if (threadIdx.x == 0) needs = moves = 0;
  for (int j = threadIdx.x; j < K; j += blockDim.x) wanted[j] = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < K; j += blockDim.x) {
    const int p = parents[(long long)b * K + j];
    if ((unsigned)p >= (unsigned)K || p == j) continue;  // the row stays
    const int m = atomicAdd(&moves, 1);
    to[m] = (short)j;
    from[m] = (short)p;
    wanted[p] = 1;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < K; j += blockDim.x)
    if (wanted[j]) need[atomicAdd(&needs, 1)] = (short)j;
  __syncthreads();
  const int nn = needs, nm = moves;
  auto piece = [&](unsigned at) {
    const unsigned o = divide(at, l.run[blockIdx.z]), c = at - o * d.run;
    return d.base + (long long)b * K * d.row_stride + o * d.outer_stride + (long long)c * (int)sizeof(V);
  };
  const unsigned base = blockIdx.x * step * turns + threadIdx.x;
  auto get = [&](int t) {
    if (t < turns)
      for (int u = 0; u < RU; ++u) {
        const unsigned at = base + t * step + u * blockDim.x;
        if (at >= per) break;
        const char* p = piece(at);
        for (int i = 0; i < nn; ++i) fetch(mine + (((t & 1) * RU + u) * K + need[i]) * blockDim.x, p + need[i] * d.row_stride);
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  get(0);
  for (int t = 0; t < turns; ++t) {
    get(t + 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    for (int u = 0; u < RU; ++u) {
      const unsigned at = base + t * step + u * blockDim.x;
      if (at >= per) break;
      char* p = piece(at);
#pragma unroll 4
      for (int i = 0; i < nm; ++i) *reinterpret_cast<V*>(p + to[i] * d.row_stride) = mine[(((t & 1) * RU + u) * K + from[i]) * blockDim.x];
    }
  }
}

template <typename V, int MAX>
cudaError_t copy_rows(const RowsList& l, int n_tensors, const int* src, const int* dst, int n, int rows, cudaStream_t s) {
  unsigned long long most = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const unsigned long long all = (unsigned long long)l.t[i].outer * l.t[i].run * n;
    most = all > most ? all : most;
  }
  const unsigned long long blocks = (most + CT * CU - 1) / (CT * CU);
  if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  if (!blocks) return cudaSuccess;
  return launch_k(copy_rows_kernel<V, MAX>, dim3((unsigned)blocks, n_tensors), dim3(CT), 0, s, tensors_of<MAX>(l, n_tensors), src, dst, n, rows);
}
template <typename V, int MAX>
cudaError_t reorder_rows(const RowsList& l, int n_tensors, const int* parents, int B, int K, cudaStream_t s) {
  // a thread's places: K for each of its pieces, of which 32 KB of a CTA and turn hold up to four
  const int fit = 32 * 1024 / (K * (int)sizeof(V)), threads = fit >= 256 ? 256 : fit >= 128 ? 128 : fit >= 64 ? 64 : 32;
  long long all = 0;
  unsigned most = 0;
  for (int i = 0; i < n_tensors; ++i) {
    most = l.t[i].outer * l.t[i].run > most ? l.t[i].outer * l.t[i].run : most;
    all += (long long)l.t[i].outer * l.t[i].run * B;
  }
  int RU = fit / threads > 4 ? 4 : fit / threads < 1 ? 1 : fit / threads, turns = 8;
  while (turns > 1 && all < 1024LL * threads * RU * turns) turns /= 2;  // as long as that leaves every SM some CTAs
  while (RU > 1 && all < 1024LL * threads * RU) RU /= 2;
  if (fit < 32) turns = 1;  // places of one turn already take up to 128 KB
  const size_t smem = (size_t)threads * K * RU * sizeof(V) * (turns > 1 ? 2 : 1);
  const unsigned blocks = (unsigned)(((long long)most + (long long)threads * RU * turns - 1) / ((long long)threads * RU * turns));
  if (!blocks) return cudaSuccess;
  cudaError_t e = allow_smem(reorder_rows_kernel<V, MAX>, smem);
  if (e != cudaSuccess) return e;
  return launch_k(reorder_rows_kernel<V, MAX>, dim3(blocks, B, n_tensors), dim3(threads), smem, s, tensors_of<MAX>(l, n_tensors), parents, B, K, RU, turns);
}
}  // namespace

cudaError_t launch_paged_write(const PagedWriteArgs& a, cudaStream_t s) {
  const int per = 2 * a.G * a.pieces, side = per < WT ? WT / per : 1;
  return launch_k(paged_write_kernel, dim3((a.L + TOK * side - 1) / (TOK * side), a.B), dim3(WT), 0, s, a);
}
template <typename F> static cudaError_t with_piece(int piece, F f) {  // f(a value of the piece's type)
  switch (piece) {
    case 16: return f(uint4{});
    case 8: return f(uint2{});
    case 4: return f(uint32_t{});
    case 2: return f(uint16_t{});
    default: return f(uint8_t{});
  }
}
cudaError_t launch_copy_rows(const RowsList& l, int n_tensors, const int* src, const int* dst, int n, int rows, int piece, cudaStream_t s) {
  return with_piece(piece, [&](auto v) {
    using V = decltype(v);
    return n_tensors <= 8 ? copy_rows<V, 8>(l, n_tensors, src, dst, n, rows, s) : copy_rows<V, ROWS_MAX>(l, n_tensors, src, dst, n, rows, s);
  });
}
cudaError_t launch_reorder_rows(const RowsList& l, int n_tensors, const int* parents, int B, int K, int piece, cudaStream_t s) {
  return with_piece(piece, [&](auto v) {
    using V = decltype(v);
    return n_tensors <= 8 ? reorder_rows<V, 8>(l, n_tensors, parents, B, K, s) : reorder_rows<V, ROWS_MAX>(l, n_tensors, parents, B, K, s);
  });
}

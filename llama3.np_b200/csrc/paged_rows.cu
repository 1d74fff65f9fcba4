// Moving rows: keys and values of new tokens into the pages of a cache, whole pages to other pages, beams' states to the beams that
// continue them.  No arithmetic: bound by the bytes, each read once and written once, 16 bytes a thread where the addresses allow it.
#include <stdint.h>

#include "../../include/llama3_b200.h"
#include "paged.h"

namespace {
// ------------------------------------------------------------------------------------------------ new tokens into pages
// A token is 2 G HD values, `per` pieces of 16 bytes; a CTA takes TOK tokens of one sequence, a thread the same piece of several.
constexpr int WT = 256, TOK = 8;
__global__ void __launch_bounds__(WT) paged_write_kernel(const PagedWriteArgs a) {
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
    uint4 x[TOK];
    int page[TOK];
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      const int t = t0 + i * side;
      const long long pos = (long long)start + t;
      const bool ok = t < n && pos >= 0 && pos < (long long)a.max_pages << a.log_page;
      page[i] = ok ? __ldg(a.table + b * a.table_stride + (pos >> a.log_page)) : -1;
      if (ok) x[i] = ldg_stream16(src + t * st + piece * 16);
    }
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      if ((unsigned)page[i] >= (unsigned)a.n_pages) continue;
      const long long pos = (long long)start + t0 + i * side;
      char* d = (char*)p.p + page[i] * p.sp + g * p.sh + (pos & ((1 << a.log_page) - 1)) * p.st;
      *reinterpret_cast<uint4*>(d + piece * 16) = x[i];
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

constexpr int CT = 256, CU = 8;  // threads, and pieces of a thread
struct CopyDivs { Div row[ROWS_MAX], run[ROWS_MAX]; };
template <typename V>
__global__ void __launch_bounds__(CT) copy_rows_kernel(const __grid_constant__ RowsList l, const __grid_constant__ CopyDivs dv,
                                                       const int* src, const int* dst, int n, int rows) {
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
    const unsigned pr = divide(at, dv.row[blockIdx.y]), rem = at - pr * per, o = divide(rem, dv.run[blockIdx.y]), c = rem - o * d.run;
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

// A thread has the same piece of all K rows of a group: it reads every row that another one wants into its own column of shared
// memory and then writes the rows that change, so that any permutation works in place without a barrier and without a copy elsewhere.
template <typename V>
__global__ void reorder_rows_kernel(const __grid_constant__ RowsList l, const __grid_constant__ CopyDivs dv, const int* parents, int B, int K) {
  extern __shared__ __align__(16) uint8_t cols_raw[];
  V* col = reinterpret_cast<V*>(cols_raw) + threadIdx.x;  // [K][blockDim.x]
  __shared__ short from[ROWS_BEAMS];      // a row's parent, itself where it stays
  __shared__ unsigned char wanted[ROWS_BEAMS];
  pdl_launch();
  pdl_wait();
  const RowsDesc& d = l.t[blockIdx.z];
  const unsigned per = d.outer * d.run;
  if (blockIdx.x * blockDim.x >= per) return;
  const int b = blockIdx.y;
  for (int j = threadIdx.x; j < K; j += blockDim.x) {
    const int p = parents[(long long)b * K + j];
    from[j] = (short)((unsigned)p < (unsigned)K ? p : j);
    wanted[j] = 0;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < K; j += blockDim.x)
    if (from[j] != j) wanted[from[j]] = 1;
  __syncthreads();
  for (unsigned at = blockIdx.x * blockDim.x + threadIdx.x; at < per; at += gridDim.x * blockDim.x) {
    const unsigned o = divide(at, dv.run[blockIdx.z]), c = at - o * d.run;
    char* p = d.base + (long long)b * K * d.row_stride + o * d.outer_stride + (long long)c * (int)sizeof(V);
#pragma unroll 4
    for (int j = 0; j < K; ++j)
      if (wanted[j]) col[j * blockDim.x] = Piece<V>::load(p + j * d.row_stride);
#pragma unroll 4
    for (int j = 0; j < K; ++j)
      if (from[j] != j) *reinterpret_cast<V*>(p + j * d.row_stride) = col[from[j] * blockDim.x];
  }
}

CopyDivs divs_of(const RowsList& l, int n) {
  CopyDivs v{};
  for (int i = 0; i < n; ++i) {
    v.row[i] = make_div(l.t[i].outer * l.t[i].run);
    v.run[i] = make_div(l.t[i].run);
  }
  return v;
}
template <typename V>
cudaError_t copy_rows(const RowsList& l, int n_tensors, const int* src, const int* dst, int n, int rows, cudaStream_t s) {
  unsigned long long most = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const unsigned long long all = (unsigned long long)l.t[i].outer * l.t[i].run * n;
    most = all > most ? all : most;
  }
  const unsigned long long blocks = (most + CT * CU - 1) / (CT * CU);
  if (blocks > 0x7fffffffull) return cudaErrorInvalidConfiguration;
  if (!blocks) return cudaSuccess;
  return launch_k(copy_rows_kernel<V>, dim3((unsigned)blocks, n_tensors), dim3(CT), 0, s, l, divs_of(l, n_tensors), src, dst, n, rows);
}
template <typename V>
cudaError_t reorder_rows(const RowsList& l, int n_tensors, const int* parents, int B, int K, cudaStream_t s) {
  // threads of a CTA: as many columns as 48 KB hold
  const int fit = 48 * 1024 / (K * (int)sizeof(V));
  const int threads = fit >= 256 ? 256 : fit >= 128 ? 128 : fit >= 64 ? 64 : 32;
  const size_t smem = (size_t)threads * K * sizeof(V);
  unsigned most = 0;
  for (int i = 0; i < n_tensors; ++i) most = l.t[i].outer * l.t[i].run > most ? l.t[i].outer * l.t[i].run : most;
  const unsigned blocks = (most + threads - 1) / threads;
  if (!blocks) return cudaSuccess;
  cudaError_t e = allow_smem(reorder_rows_kernel<V>, smem);
  if (e != cudaSuccess) return e;
  return launch_k(reorder_rows_kernel<V>, dim3(blocks, B, n_tensors), dim3(threads), smem, s, l, divs_of(l, n_tensors), parents, B, K);
}
}  // namespace

cudaError_t launch_paged_write(const PagedWriteArgs& a, cudaStream_t s) {
  const int per = 2 * a.G * a.pieces, side = per < WT ? WT / per : 1;
  return launch_k(paged_write_kernel, dim3((a.L + TOK * side - 1) / (TOK * side), a.B), dim3(WT), 0, s, a);
}
cudaError_t launch_copy_rows(const RowsList& l, int n_tensors, const int* src, const int* dst, int n, int rows, int piece, cudaStream_t s) {
  switch (piece) {
    case 16: return copy_rows<uint4>(l, n_tensors, src, dst, n, rows, s);
    case 8: return copy_rows<uint2>(l, n_tensors, src, dst, n, rows, s);
    case 4: return copy_rows<uint32_t>(l, n_tensors, src, dst, n, rows, s);
    case 2: return copy_rows<uint16_t>(l, n_tensors, src, dst, n, rows, s);
    default: return copy_rows<uint8_t>(l, n_tensors, src, dst, n, rows, s);
  }
}
cudaError_t launch_reorder_rows(const RowsList& l, int n_tensors, const int* parents, int B, int K, int piece, cudaStream_t s) {
  switch (piece) {
    case 16: return reorder_rows<uint4>(l, n_tensors, parents, B, K, s);
    case 8: return reorder_rows<uint2>(l, n_tensors, parents, B, K, s);
    case 4: return reorder_rows<uint32_t>(l, n_tensors, parents, B, K, s);
    case 2: return reorder_rows<uint16_t>(l, n_tensors, parents, B, K, s);
    default: return reorder_rows<uint8_t>(l, n_tensors, parents, B, K, s);
  }
}

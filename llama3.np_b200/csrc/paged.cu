// Attention of one new token per sequence over a key / value cache in pages (L3PagedAttn):
//   s_j = scale q_h . k_j,  o_h = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse_h = m + log sum_j e^(s_j - m),  m = max_j s_j
// over the tokens j < length of the sequence; token j lies in page table[j / P] at place j % P.
//
// Bound by the cache's bytes: every key and value is read once for all query heads of its kv head (2 HD values for 4 HD flops per
// query head).  The keys of all (sequence, kv head) items, in tiles of 16, are one long row that the warps of the machine share
// out evenly - lengths of any mixture leave no SM idle, and a single long sequence fills the machine.  A warp works through its
// stretch alone, without a block barrier: a ring of tiles in shared memory filled by 16-byte asynchronous copies (a page's rows can
// lie anywhere; the ring runs on across items), one pass with running maximum and sum.  An item that lies within one warp's stretch
// is written at once; one that several warps share leaves a partial (m, l, o) per warp, and a second, dependent launch joins those
// in the order of the keys, so that results do not change from run to run.
#include <math.h>

#include <type_traits>

#include <cuda_fp16.h>

#include "../../include/llama3_b200.h"
#include "attn_decode.cuh"
#include "paged.h"

namespace {
constexpr int TK = 16;          // keys of a tile
constexpr int MOST_NW = 4;      // warps of a CTA (Core::NW)
constexpr int CTAS = 2;         // CTAs of an SM
constexpr int HEADS = 8;        // most query heads of an item

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes into shared memory, zeros where !take (the address is not read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, bf16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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
__device__ __forceinline__ float2 load_q2(const PagedAttnArgs& a, long long i) {  // two neighbours of q as fp32
  if (a.q_dtype == L3_DTYPE_F32) return make_float2(__ldg((const float*)a.q + i), __ldg((const float*)a.q + i + 1));
  if (a.q_dtype == L3_DTYPE_BF16) {
    const bf16* p = (const bf16*)a.q + i;
    return make_float2(__bfloat162float(p[0]), __bfloat162float(p[1]));
  }
  const __half* p = (const __half*)a.q + i;
  return make_float2(__half2float(p[0]), __half2float(p[1]));
}
__device__ __forceinline__ void store_out2(const PagedAttnArgs& a, long long i, float x, float y) {  // i is even
  if (a.out_dtype == L3_DTYPE_F32) {
    if (a.out_lo) {
      float hx, lx, hy, ly;
      split_tf32(x, hx, lx);
      split_tf32(y, hy, ly);
      *reinterpret_cast<float2*>((float*)a.out + i) = make_float2(hx, hy);
      *reinterpret_cast<float2*>(a.out_lo + i) = make_float2(lx, ly);
    } else *reinterpret_cast<float2*>((float*)a.out + i) = make_float2(x, y);
  } else if (a.out_dtype == L3_DTYPE_BF16) *reinterpret_cast<__nv_bfloat162*>((bf16*)a.out + i) = __floats2bfloat162_rn(x, y);
  else *reinterpret_cast<__half2*>((__half*)a.out + i) = __floats2half2_rn(x, y);
}
__device__ __forceinline__ int asked_length(const PagedAttnArgs& a, int b) { return a.lengths ? a.lengths[b] : *a.pos_ptr + 1; }
__device__ __forceinline__ int length_of(const PagedAttnArgs& a, int b) {
  const long long n = asked_length(a, b), cap = (long long)a.max_pages << a.log_page;
  return (int)(n < 0 ? 0 : n > cap ? cap : n);
}
__device__ __forceinline__ int tiles_of(int len) { return (len + TK - 1) / TK; }

// where a warp is in the long row of tiles: tile t of the nt tiles of item (b, gb)
struct Cursor {
  int b, gb, t, nt, len;
};
__device__ __forceinline__ void next_sequence(const PagedAttnArgs& a, Cursor& c) {
  c.gb = c.t = 0;
  do {
    ++c.b;
    c.len = c.b < a.B ? length_of(a, c.b) : 0;
    c.nt = tiles_of(c.len);
  } while (c.b < a.B && c.nt == 0);
}
__device__ __forceinline__ void advance(const PagedAttnArgs& a, Cursor& c, int items) {
  if (++c.t < c.nt) return;
  c.t = 0;
  if (++c.gb == items) next_sequence(a, c);
}

// ------------------------------------------------------------------------------------------ 16-bit caches: tensor cores
// The item's (up to 8) query heads are rows 0 - 7 of an m16n8k16 tile.  Rows 8 - 15, which a tile has anyway, carry what rounding to 16
// bits leaves of the same heads: the rest of an fp32 query in S = Q K^T, the rest of the weights in O += P V, so that the weights
// enter with 16 (bf16) or 22 (fp16) significant bits at no further instruction.  fp16 weights are scaled by 2^12 ahead of the rounding
// (they are at most 1), which keeps weights down to 2^-36 of the largest off the subnormals.
template <typename T, int HD> struct MmaCore {
  static constexpr int ROW = HD * 2, NCH = ROW / 16, PITCH = ROW + 16;  // the odd number of 16-byte pieces keeps ldmatrix free of conflicts
  static constexpr int TILE = 2 * TK * PITCH;                           // bytes of a tile's keys and values
  static constexpr int KS = HD / 16, NT = HD / 8;
  static constexpr int NW = 4;
  static constexpr float BIAS = std::is_same<T, bf16>::value ? 0.f : 12.f;
  uint32_t qa[KS][4];
  float o[NT][4];
  float m, l;  // of row lane / 4, in units of log 2; l: this lane's share
  float sc;

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, int b, int head0, int heads, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const long long qp = b * a.q_sb + (long long)(head0 + min(g, heads - 1)) * a.q_sh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const float2 x = load_q2(a, qp + ks * 16 + 2 * t), y = load_q2(a, qp + ks * 16 + 8 + 2 * t);
      two_parts<T>(x.x, x.y, qa[ks][0], qa[ks][1]);
      two_parts<T>(y.x, y.y, qa[ks][2], qa[ks][3]);
      if (a.q_dtype != L3_DTYPE_F32) qa[ks][1] = qa[ks][3] = 0u;  // also where an infinity would leave a NaN
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m = -INFINITY;
    l = 0.f;
    sc = a.scale * 1.4426950408889634f;
  }
  __device__ __forceinline__ void tile(uint32_t ksm, uint32_t mask, int lane) {
    const int t = lane & 3, mi = lane >> 3, mr = lane & 7;
    float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
    {
      const uint32_t row = ksm + ((mi >> 1) * 8 + mr) * PITCH + (mi & 1) * 16;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t kb[4];
        ldsm_x4(row + ks * 32, kb);
        mma16816<T>(s0, qa[ks], kb[0], kb[1]);
        mma16816<T>(s1, qa[ks], kb[2], kb[3]);
      }
    }
    const uint32_t mk = mask >> (2 * t);
    const float v00 = mk & 1 ? (s0[0] + s0[2]) * sc : -INFINITY, v01 = mk & 2 ? (s0[1] + s0[3]) * sc : -INFINITY;
    const float v10 = mk & 256 ? (s1[0] + s1[2]) * sc : -INFINITY, v11 = mk & 512 ? (s1[1] + s1[3]) * sc : -INFINITY;
    float mx = fmaxf(fmaxf(v00, v01), fmaxf(v10, v11));
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
    const float p00 = ex2(v00 - from + BIAS), p01 = ex2(v01 - from + BIAS), p10 = ex2(v10 - from + BIAS), p11 = ex2(v11 - from + BIAS);
    l += (p00 + p01) + (p10 + p11);
    uint32_t pa[4];
    two_parts<T>(p00, p01, pa[0], pa[1]);
    two_parts<T>(p10, p11, pa[2], pa[3]);
    {
      const uint32_t row = ksm + TK * PITCH + ((mi & 1) * 8 + mr) * PITCH + (mi >> 1) * 16;
#pragma unroll
      for (int np = 0; np < KS; ++np) {
        uint32_t vb[4];
        ldsm_x4_trans(row + np * 32, vb);
        mma16816<T>(o[2 * np], pa, vb[0], vb[1]);
        mma16816<T>(o[2 * np + 1], pa, vb[2], vb[3]);
      }
    }
  }
  // whole: the result; else the partial of `slot`
  __device__ __forceinline__ void end(const PagedAttnArgs& a, bool whole, int b, int head0, int heads, int slot, int lane) {
    const int g = lane >> 2, t = lane & 3;
    l += __shfl_xor_sync(L3_FULL, l, 1);
    l += __shfl_xor_sync(L3_FULL, l, 2);
    if (g >= heads) return;
    if (whole) {
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      const long long oi = ((long long)b * a.H + head0 + g) * HD;
#pragma unroll
      for (int n = 0; n < NT; ++n) store_out2(a, oi + n * 8 + 2 * t, (o[n][0] + o[n][2]) * inv, (o[n][1] + o[n][3]) * inv);
      if (a.lse && t == 0) a.lse[(long long)b * a.H + head0 + g] = (m - BIAS + log2f(l)) * 0.6931471805599453f;
    } else {
      float* po = a.part_o + ((long long)slot * a.heads_blk + g) * HD;
#pragma unroll
      for (int n = 0; n < NT; ++n)
        *reinterpret_cast<float2*>(po + n * 8 + 2 * t) = make_float2(o[n][0] + o[n][2], o[n][1] + o[n][3]);
      if (t == 0) *reinterpret_cast<float2*>(a.part_ml + ((long long)slot * a.heads_blk + g) * 2) = make_float2((m - BIAS) * 0.6931471805599453f, l);
    }
  }
};

// --------------------------------------------------------------------------------------------------- fp32 caches: FFMA
// LPK lanes share a key (DecodeCfg), KPW keys side by side; NREP query heads of an item (a.heads_blk of them real).  m, l and o are
// kept per lane group and merged over the warp at the end of an item.
template <int HD, int NREP> struct F32Core {
  using C = DecodeCfg<HD, float>;
  static constexpr int ROW = HD * 4, NCH = ROW / 16, PITCH = ROW + 16;
  static constexpr int TILE = 2 * TK * PITCH;
  static constexpr int NW = TILE > 14000 ? 2 : 4;                       // at least two tiles per warp in flight
  static constexpr int EPL = C::EPL, LPK = C::LPK, KPW = C::KPW, PASSES = KPW >= TK ? 1 : TK / KPW;
  static constexpr int U = PASSES < 16 / NREP ? PASSES : 16 / NREP < 2 ? (PASSES < 2 ? PASSES : 2) : 16 / NREP;
  float q[NREP][EPL], o[NREP][EPL], m[NREP], l[NREP];

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, int b, int head0, int heads, int lane) {
    const int sl = lane % LPK;
#pragma unroll
    for (int r = 0; r < NREP; ++r) {
      const long long qp = b * a.q_sb + (long long)(head0 + min(r, heads - 1)) * a.q_sh;
#pragma unroll
      for (int e = 0; e < EPL; e += 2) {
        const float2 x = load_q2(a, qp + C::dim(sl, e));
        q[r][e] = x.x * a.scale;
        q[r][e + 1] = x.y * a.scale;
      }
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[r][e] = 0.f;
      m[r] = -INFINITY;
      l[r] = 0.f;
    }
  }
  __device__ __forceinline__ void row(uint32_t addr, int sl, float (&v)[EPL]) {
#pragma unroll
    for (int c = 0; c < C::CPL; ++c)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[4 * c]), "=f"(v[4 * c + 1]), "=f"(v[4 * c + 2]), "=f"(v[4 * c + 3]) : "r"(addr + (c * LPK + sl) * 16));
  }
  __device__ __forceinline__ void tile(uint32_t ksm, uint32_t mask, int lane) {
    const int sub = lane / LPK, sl = lane % LPK;
#pragma unroll
    for (int p0 = 0; p0 < PASSES; p0 += U) {
      float s[U][NREP];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = (p0 + u) * KPW + sub;  // KPW > TK: lane groups beyond the tile have no key
        float kk[EPL];
        row(ksm + (key < TK ? key : 0) * PITCH, sl, kk);
        const bool ok = key < TK && (mask >> key & 1);
#pragma unroll
        for (int r = 0; r < NREP; ++r) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < EPL; ++e) d = fmaf(q[r][e], kk[e], d);
#pragma unroll
          for (int off = LPK / 2; off > 0; off >>= 1) d += __shfl_xor_sync(L3_FULL, d, off);
          s[u][r] = ok ? d : -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < NREP; ++r) {
        float mx = m[r];
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
        const float from = mx == -INFINITY ? 0.f : mx;
        const float alpha = expf(m[r] - from);
        l[r] *= alpha;
#pragma unroll
        for (int e = 0; e < EPL; ++e) o[r][e] *= alpha;
        m[r] = mx;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[u][r] = expf(s[u][r] - from);
          l[r] += s[u][r];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int key = (p0 + u) * KPW + sub;
        float vv[EPL];
        row(ksm + TK * PITCH + (key < TK ? key : 0) * PITCH, sl, vv);
#pragma unroll
        for (int r = 0; r < NREP; ++r)
#pragma unroll
          for (int e = 0; e < EPL; ++e) o[r][e] = key < TK ? fmaf(s[u][r], vv[e], o[r][e]) : o[r][e];
      }
    }
  }
  __device__ __forceinline__ void end(const PagedAttnArgs& a, bool whole, int b, int head0, int heads, int slot, int lane) {
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
      if (whole) {
        const float inv = l[r] == 0.f ? 0.f : 1.0f / l[r];
        const long long oi = ((long long)b * a.H + head0 + r) * HD;
#pragma unroll
        for (int e = 0; e < EPL; e += 2) store_out2(a, oi + C::dim(sl, e), o[r][e] * inv, o[r][e + 1] * inv);
        if (a.lse && sl == 0) a.lse[(long long)b * a.H + head0 + r] = m[r] + logf(l[r]);
      } else {
        float* po = a.part_o + ((long long)slot * a.heads_blk + r) * HD;
#pragma unroll
        for (int e = 0; e < EPL; e += 2) *reinterpret_cast<float2*>(po + C::dim(sl, e)) = make_float2(o[r][e], o[r][e + 1]);
        if (sl == 0) *reinterpret_cast<float2*>(a.part_ml + ((long long)slot * a.heads_blk + r) * 2) = make_float2(m[r], l[r]);
      }
    }
  }
};

template <typename Core, typename T, int ST>
__global__ void __launch_bounds__(Core::NW * 32, CTAS) paged_attn_kernel(const PagedAttnArgs a) {
  constexpr int NW = Core::NW, HD = Core::ROW / (int)sizeof(T), NCH = Core::NCH, PITCH = Core::PITCH;
  extern __shared__ __align__(16) uint8_t ring_raw[];
  __shared__ uint32_t masks[NW][ST];
  pdl_launch();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int W = gridDim.x * NW, w = warp * gridDim.x + blockIdx.x;  // neighbours in the row of tiles on different SMs
  const int items = a.G * a.blocks;

  // tiles of one item of every sequence, and of all
  long long sum = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    sum += b < a.B ? tiles_of(length_of(a, b)) : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(L3_FULL, sum, o);
  const long long total = sum * items, per = (total + W - 1) / W;
  // sequences without tokens
  for (int b = w; b < a.B; b += W) {
    if (length_of(a, b) > 0) continue;
    for (int i = lane; i < a.H * (HD / 2); i += 32) store_out2(a, (long long)b * a.H * HD + 2 * i, 0.f, 0.f);
    if (a.lse)
      for (int h = lane; h < a.H; h += 32) a.lse[(long long)b * a.H + h] = -INFINITY;
    if (a.by_item)
      for (int i = lane; i < items; i += 32) a.info[(long long)b * items + i] = make_int4(0, 0, 0, 0);
  }
  int4 tail = make_int4(0, 0, 0, 0);  // the item that begins here and goes on in the next warps: first slot, warp, partials, item
  const long long u0 = per * w;
  if (u0 < total) {
    const int n = (int)(total - u0 < per ? total - u0 : per);
    // the sequence that holds tile u0
    Cursor C{};
    {
      long long before = 0;
      for (int b0 = 0;; b0 += 32) {
        const int b = b0 + lane, len = b < a.B ? length_of(a, b) : 0, nt = tiles_of(len);
        long long run = nt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long x = __shfl_up_sync(L3_FULL, run, o);
          if (lane >= o) run += x;
        }
        const uint32_t hit = __ballot_sync(L3_FULL, (before + run) * items > u0);
        if (hit || b0 + 32 >= a.B) {
          const int src = hit ? __ffs(hit) - 1 : 31;
          C.b = b0 + src;
          C.nt = __shfl_sync(L3_FULL, nt, src);
          C.len = __shfl_sync(L3_FULL, len, src);
          const long long at = u0 - (before + __shfl_sync(L3_FULL, run - nt, src)) * items;
          C.gb = (int)(at / C.nt);
          C.t = (int)(at - (long long)C.gb * C.nt);
          break;
        }
        before += __shfl_sync(L3_FULL, run, 31);
      }
    }
    const uint32_t ring = smem_u32(ring_raw) + warp * ST * Core::TILE;
    Cursor L = C;
    int entry = 0;
    auto look = [&] {  // the page of this lane's key of the tile that is loaded next
      const int pos = L.t * TK + (lane & (TK - 1));
      entry = L.b < a.B && pos < L.len ? __ldg(a.table + L.b * a.table_stride + (pos >> a.log_page)) : -1;
    };
    auto load = [&](int stage) {
      const int pos = L.t * TK + (lane & (TK - 1)), g = L.gb / a.blocks;
      const bool ok = pos < L.len && (unsigned)entry < (unsigned)a.n_pages;
      const int in = pos & ((1 << a.log_page) - 1);
      T* kp = (T*)a.k.p + (ok ? entry * a.k.sp + in * a.k.st + g * a.k.sh : 0);
      T* vp = (T*)a.v.p + (ok ? entry * a.v.sp + in * a.v.st + g * a.v.sh : 0);
      const uint32_t mask = __ballot_sync(L3_FULL, ok) & 0xffffu;
      if (lane == 0) masks[warp][stage] = mask;
      // the tile of the new token, unless that lies behind the table: its row comes from k_new / v_new, and goes to its page
      if (a.k_new && L.t == L.nt - 1 && asked_length(a, L.b) == L.len) {
        const int row = (L.len - 1) & (TK - 1);
        T* kn = (T*)a.k_new + L.b * a.kn_sb + g * a.kn_sh;
        T* vn = (T*)a.v_new + L.b * a.vn_sb + g * a.vn_sh;
        if (mask >> row & 1 && L.gb % a.blocks == 0) {
          uint4* kd = (uint4*)__shfl_sync(L3_FULL, (unsigned long long)kp, row);
          uint4* vd = (uint4*)__shfl_sync(L3_FULL, (unsigned long long)vp, row);
          for (int c = lane; c < 2 * NCH; c += 32) {
            if (c < NCH) kd[c] = __ldg((const uint4*)kn + c);
            else vd[c - NCH] = __ldg((const uint4*)vn + c - NCH);
          }
        }
        if ((lane & (TK - 1)) == row) { kp = kn; vp = vn; }
      }
      const uint32_t dst = ring + stage * Core::TILE;
#pragma unroll
      for (int i = 0; i < (TK * NCH + 31) / 32; ++i) {
        const int idx = i * 32 + lane, r = idx / NCH, c = idx % NCH;
        const unsigned long long ks = __shfl_sync(L3_FULL, (unsigned long long)kp, r & (TK - 1));
        const unsigned long long vs = __shfl_sync(L3_FULL, (unsigned long long)vp, r & (TK - 1));
        if (TK * NCH % 32 == 0 || r < TK) {
          const bool take = mask >> r & 1;
          cp16(dst + r * PITCH + c * 16, (const uint4*)ks + c, take);
          cp16(dst + TK * PITCH + r * PITCH + c * 16, (const uint4*)vs + c, take);
        }
      }
      advance(a, L, items);
      look();
    };
    look();
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      if (i < n) load(i);
      cp_commit();
    }
    Core core;
    auto head0 = [&] { return (C.gb / a.blocks) * (a.H / a.G) + (C.gb % a.blocks) * a.heads_blk; };
    auto heads = [&] { return min(a.heads_blk, a.H / a.G - (C.gb % a.blocks) * a.heads_blk); };
    core.begin(a, C.b, head0(), heads(), lane);
    int t0 = C.t;          // first tile of the present item here
    bool first = true;
    int stage = 0, fill = ST - 1;
    for (int i = 0; i < n; ++i) {
      if (i + ST - 1 < n) load(fill);
      cp_commit();
      fill = fill + 1 == ST ? 0 : fill + 1;
      cp_wait<ST - 1>();
      __syncwarp();
      core.tile(ring + stage * Core::TILE, masks[warp][stage], lane);
      __syncwarp();
      stage = stage + 1 == ST ? 0 : stage + 1;
      if (C.t == C.nt - 1 || i == n - 1) {
        const bool starts = t0 == 0, ends = C.t == C.nt - 1;
        const int slot = 2 * w + (first ? 0 : 1);
        core.end(a, starts && ends, C.b, head0(), heads(), slot, lane);
        if (starts) {
          const int parts = ends ? 0 : 1 + (int)((C.nt - 1 - C.t + per - 1) / per);
          const int4 in = make_int4(slot, w, parts, C.b * items + C.gb);
          if (!a.by_item) tail = in;
          else if (lane == 0) a.info[(long long)C.b * items + C.gb] = in;
        }
        first = false;
        if (i < n - 1) {
          advance(a, C, items);
          core.begin(a, C.b, head0(), heads(), lane);
          t0 = 0;
        }
      } else ++C.t;
    }
  }
  if (!a.by_item && lane == 0) a.info[w] = tail;
}

// Joins the partials of one item and query head: weights e^(m_p - m) of the partials, then their sum in the order of the keys.
constexpr int JOIN_T = 128, JOIN_MAX = 2048;
__global__ void __launch_bounds__(JOIN_T) paged_join_kernel(const PagedAttnArgs a) {
  __shared__ float wt[JOIN_MAX];
  __shared__ float red[JOIN_T / 32][2];
  __shared__ float4 acc[JOIN_T];
  pdl_launch();
  pdl_wait();
  const int4 in = a.info[blockIdx.x];
  const int parts = min(in.z, JOIN_MAX), r = blockIdx.y, tid = threadIdx.x;
  if (parts == 0) return;
  const int items = a.G * a.blocks, b = in.w / items, gb = in.w % items;
  if (r >= min(a.heads_blk, a.H / a.G - (gb % a.blocks) * a.heads_blk)) return;
  auto row = [&](int p) { return (long long)(p == 0 ? in.x : 2 * (in.y + p)) * a.heads_blk + r; };
  float mx = -INFINITY;
  for (int p = tid; p < parts; p += JOIN_T) {
    wt[p] = a.part_ml[row(p) * 2];
    mx = fmaxf(mx, wt[p]);
  }
  mx = warp_max(mx);
  if ((tid & 31) == 0) red[tid >> 5][0] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < JOIN_T / 32; ++i) mx = fmaxf(mx, red[i][0]);
  const float from = mx == -INFINITY ? 0.f : mx;
  float l = 0.f;
  for (int p = tid; p < parts; p += JOIN_T) {
    wt[p] = expf(wt[p] - from);
    l = fmaf(a.part_ml[row(p) * 2 + 1], wt[p], l);
  }
  l = warp_sum(l);
  if ((tid & 31) == 0) red[tid >> 5][1] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int i = 0; i < JOIN_T / 32; ++i) l += red[i][1];
  const int q4 = a.HD / 4, d = tid % q4, grp = tid / q4, ngrp = JOIN_T / q4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < ngrp) {
#pragma unroll 4
    for (int p = grp; p < parts; p += ngrp) {
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + row(p) * a.HD + 4 * d);
      const float w = wt[p];
      o.x = fmaf(w, x.x, o.x); o.y = fmaf(w, x.y, o.y); o.z = fmaf(w, x.z, o.z); o.w = fmaf(w, x.w, o.w);
    }
    acc[tid] = o;
  }
  __syncthreads();
  if (grp) return;
  for (int i = 1; i < ngrp; ++i) {
    const float4 x = acc[i * q4 + d];
    o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const int head = (gb / a.blocks) * (a.H / a.G) + (gb % a.blocks) * a.heads_blk + r;
  const long long oi = ((long long)b * a.H + head) * a.HD + 4 * d;
  store_out2(a, oi, o.x * inv, o.y * inv);
  store_out2(a, oi + 2, o.z * inv, o.w * inv);
  if (a.lse && d == 0) a.lse[(long long)b * a.H + head] = mx + logf(l);
}

template <typename Core, typename T>
cudaError_t launch_core(PagedAttnArgs a, int n_sm, cudaStream_t s) {
  // as many tiles in flight as two CTAs of an SM have room for; more than eight gain nothing
  constexpr int NW = Core::NW, room = 110 * 1024 / (NW * Core::TILE), ST = room > 8 ? 8 : room;
  static_assert(ST >= 2, "");
  auto kern = paged_attn_kernel<Core, T, ST>;
  constexpr size_t smem = (size_t)NW * ST * Core::TILE;
  cudaError_t e = allow_smem(kern, smem);
  if (e != cudaSuccess) return e;
  const int W = n_sm * CTAS * NW;
  const long long items = (long long)a.B * a.G * a.blocks;
  a.by_item = items <= W;
  a.n_info = (int)(a.by_item ? items : W);
  if ((e = launch_k(kern, dim3(n_sm * CTAS), dim3(NW * 32), smem, s, a)) != cudaSuccess) return e;
  g_l3_pdl_next = true;  // the joining launch starts in the tail of the first
  return launch_k(paged_join_kernel, dim3(a.n_info, a.heads_blk), dim3(JOIN_T), 0, s, a);
}
template <int HD> cudaError_t launch_f32(const PagedAttnArgs& a, int n_sm, cudaStream_t s) {
  if (a.heads_blk == 1) return launch_core<F32Core<HD, 1>, float>(a, n_sm, s);
  if (a.heads_blk == 2) return launch_core<F32Core<HD, 2>, float>(a, n_sm, s);
  if constexpr (HD == 48 || HD == 96) return launch_core<F32Core<HD, 4>, float>(a, n_sm, s);
  else if (a.heads_blk <= 4) return launch_core<F32Core<HD, 4>, float>(a, n_sm, s);
  else return launch_core<F32Core<HD, 8>, float>(a, n_sm, s);
}
template <int HD> cudaError_t launch_hd(const PagedAttnArgs& a, int n_sm, cudaStream_t s) {
  if (a.kv_dtype == L3_DTYPE_F32) return launch_f32<HD>(a, n_sm, s);
  if (a.kv_dtype == L3_DTYPE_BF16) return launch_core<MmaCore<bf16, HD>, bf16>(a, n_sm, s);
  return launch_core<MmaCore<__half, HD>, __half>(a, n_sm, s);
}
}  // namespace

// query heads that share a reading of their keys: as many as registers hold (fp32, head sizes 48 and 96: 12 dimensions per lane)
static int heads_of_item(int H, int G, int HD, int kv_dtype) {
  const int most = kv_dtype == L3_DTYPE_F32 && (HD == 48 || HD == 96) ? HEADS / 2 : HEADS;
  return H / G < most ? H / G : most;
}
size_t paged_attn_workspace(int H, int G, int HD, int n_sm) {
  const size_t W = (size_t)n_sm * CTAS * MOST_NW;
  return W * sizeof(int4) + 2 * W * (H / G < HEADS ? H / G : HEADS) * ((size_t)HD + 2) * sizeof(float);
}

cudaError_t launch_paged_attention(PagedAttnArgs a, int n_sm, cudaStream_t s) {
  const int W = n_sm * CTAS * MOST_NW;
  if (W > JOIN_MAX) return cudaErrorInvalidConfiguration;
  a.heads_blk = heads_of_item(a.H, a.G, a.HD, a.kv_dtype);
  a.blocks = (a.H / a.G + a.heads_blk - 1) / a.heads_blk;
  a.info = (int4*)a.ws;
  a.part_o = (float*)(a.info + W);
  a.part_ml = a.part_o + (size_t)2 * W * a.heads_blk * a.HD;
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

// Attention of the rows of a packed step over a 16-bit cache in pages (paged_chunk.cu has the formula, paged_chunk.cuh how the work is cut), on
// tcgen05: a CTA an SM, blocks of 128 keys, score tiles of 128 rows x 128 keys.
//
//   warps 10, 11  loaders: the item's queries, then keys and values of its blocks, a page a TMA copy, into a ring of operand tiles (K-major rows of
//                 128 bytes, swizzled); rows of no token become zeros, and their bits go to the softmax warps.  Pages of fewer than 8 tokens,
//                 expanded strides, and queries whose heads do not fill 128 rows evenly go row by row, 16 bytes a copy (cp.async)
//   warp 8        products: S = Q K^T into TMEM, O += P V with P from TMEM and V as it lies, an MN-major operand
//   warps 0 - 7   softmax, a thread a row, four warps a score tile: its 128 scores in registers, exponentials against a maximum that follows
//                 the running one lazily (O is rescaled in TMEM only when that has grown by 2^GROW), weights as 16-bit values over the scores
// The two score tiles take turns: one's softmax runs while the tensor core works on the other's products.  With many rows they are two tiles of
// rows over the same keys, so that every key and value that arrives is used for 256 rows; with few rows they are one tile of rows over every other
// block of keys, and meet at the end.
//
// Bound by latency within the softmax: two score tiles over a block take 3.3 K cycles, their products 2.05 K (heads of 128; the tensor pipe is busy for 57 % of the time, the
// issue slots for 40 %, the exponentials' units for less than half), an item's beginning and end 5.5 K.  32 heads over 8 kv heads of 128 in bf16: 511 rows over 65000 tokens 465 - 481 us (1.14 - 1.17 PFLOP/s, 69 - 71 % of what a large
// product reaches), six prompts of up to 4096 454 - 462; of 64 in fp16, 48 requests of up to 3001 tokens in pages of 32, most with one row, 98 us, 177 MB.
//
// A weight enters the product rounded to the cache's type (half a step: bf16 2^-9 of it, as much as the result's own rounding; sums are of the unrounded
// ones, in fp32).  fp16 weights are scaled by 2^BIAS ahead of the rounding: the largest lies in [2^12, 2^15], what fp16 has no number for is below
// 2^-37 of it.
#include <limits.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "gemm_tc_dev.cuh"
#include "paged_chunk.cuh"

namespace {
using namespace chunk;
constexpr int BK = TC_BK, NT = 384, SOFT = 256, LOADERS = 2, SETS = 4 / LOADERS;  // SETS: of 32 rows of a tile, a loader's
constexpr int POLY = 1;    // of four neighbouring pairs of exponentials, how many are taken by a polynomial
constexpr int THERE = 16;  // blocks whose keys' bits are kept: more than the ring holds

template <typename T, int HD> struct Cfg {
  static constexpr int QS = (HD + 63) / 64;             // slices of 64 entries, rows of 128 bytes
  static constexpr int TILE = QS * 128 * 128;           // bytes of 128 rows
  static constexpr int NS = HD > 64 ? 5 : 8;            // tiles of the ring
  static constexpr int SMEM = 2 * TILE + NS * TILE + THERE * 16 + 256 + 1024;
  static constexpr uint32_t FMT = std::is_same<T, bf16>::value ? 1u : 0u;
  static constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(BK >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_PV = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr float BIAS = FMT ? 0.f : 12.f, GROW = FMT ? 8.f : 3.f;
};
constexpr int T_O = 256, T_COLS = 512;  // TMEM: two score tiles (the weights lie over their first halves), two outputs

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {  // zeros where !take
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok;
}
// Operand descriptors, their lower halves (start address and leading offset): the upper half is the same for all - 8-row groups 1024 bytes apart, 128-byte
// swizzle.  K-major: rows of 128 bytes.  MN-major: rows are the keys (the product's K), atoms of 64 columns are 16384 bytes apart.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29), DESC_K = 1u << 16, DESC_MN = (16384u >> 4) << 16;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) { return (addr & 0x3FFFF) >> 4 | lead; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.b32 p, %4, 0;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accum), "r"(DESC_HI) : "memory");
}
// A from TMEM: a lane a row, two neighbouring entries a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.b32 p, %4, 0;\nmov.b64 y, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accum), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* v) {  // without the wait
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* v) {  // without the wait
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_ld8(uint32_t at, float* v) {  // without the wait
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t at, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <typename T> __device__ __forceinline__ uint32_t pack(float x, float y) {
  if constexpr (std::is_same<T, bf16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ void store32(void* to, const uint32_t* x) {  // to a multiple of 32 bytes
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(to), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
               ::"r"(dst), "l"(tm), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar) : "memory");
}
__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if one of them is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d) : "l"(*reinterpret_cast<const unsigned long long*>(&a)), "l"(*reinterpret_cast<const unsigned long long*>(&b)));
  return *reinterpret_cast<const float2*>(&d);
}
// 2^x without the unit for it, for x <= 20: x = n + f, |f| <= 1/2, by adding and taking off a number whose last bit is 1, and a polynomial of degree 4
// (minimax of the relative error on [-1/2, 1/2] by Remez's exchange: at most 2.65e-6 off, 1.6e-6 in the mean and 4e-8 with its sign; 2.67e-6 with the
// roundings).  Below 2^-126 the result is within 2^-127.  A hidden key's x is -infinity, and its weight has to be nothing, as its value may be the largest
// number there is: x stops just above -127, where n is -127, the polynomial just above 1, and what is left of it 5.3e-44, which both 16-bit types round to 0.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f), minus = make_float2(-1.f, -1.f);
  constexpr float LEAST = -127.f + 0x1p-17f;  // the next number above -127
  x.x = fmaxf(x.x, LEAST);
  x.y = fmaxf(x.y, LEAST);
  const float2 t = add2(x, magic), f = fma2(add2(t, back), minus, x);
  float2 y = make_float2(0.009570102207362652f, 0.009570102207362652f);
  y = fma2(y, f, make_float2(0.05591785907745361f, 0.05591785907745361f));
  y = fma2(y, f, make_float2(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  y = fma2(y, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)));
}
// Maps of the queries (entries, heads, rows) and the pools (entries, tokens, heads, pages, keys or values), where tiles are copied by them.  To make one
// takes the host 2 us: both pools are one, the distance between them a stride.
struct Maps {
  CUtensorMap q, kv;
};

// Barriers of a CTA, 8 bytes each.
struct Bars {
  uint32_t q_full, q_empty, landed, s_full, half_p, p_full, o_full, full, empty;  // s_full .. o_full: of both score tiles
};

template <typename T, int HD>
__global__ void __launch_bounds__(NT, 1) chunk_tc_kernel(const ChunkArgs a, const __grid_constant__ Maps maps, const bool tma_q, const bool tma_kv, const bool keys_first) {
  using C = Cfg<T, HD>;
  constexpr int NS = C::NS, TILE = C::TILE;
  using Cur = Cursor<BK>;
  constexpr Split SPLIT = tc_split(HD);
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long room[NT / 32 + 1];
  __shared__ Place place;
  __shared__ int failed;
  __shared__ float xch[8][32];  // from score tile to score tile
  volatile int* const fail = &failed;
  const uint32_t raw = smem_u32(smem_raw), sQ = (raw + 1023u) & ~1023u, ring = sQ + 2 * TILE;
  uint32_t* const there = reinterpret_cast<uint32_t*>(smem_raw + (ring + NS * TILE - raw));  // [THERE][4]
  const uint32_t bars = ring + NS * TILE + THERE * 16;
  const Bars B{bars, bars + 8, bars + 16, bars + 24, bars + 40, bars + 56, bars + 72, bars + 88, bars + 88 + 8 * NS};
  const uint32_t tmem_slot = B.empty + 8 * NS;
  uint32_t* const tmem_slot_ptr = reinterpret_cast<uint32_t*>(smem_raw + (tmem_slot - raw));
  const int warp = __shfl_sync(L3_FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  pdl_launch();
  if (threadIdx.x == 0) {
    mbar_init(B.q_full, tma_q ? 1 : LOADERS);
    mbar_init(B.q_empty, 1);
    mbar_init(B.landed, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(B.s_full + 8 * w, 1); mbar_init(B.half_p + 8 * w, 4); mbar_init(B.p_full + 8 * w, 4); mbar_init(B.o_full + 8 * w, 1);
    }
    for (int s = 0; s < NS; ++s) { mbar_init(B.full + 8 * s, tma_kv ? 1 : LOADERS); mbar_init(B.empty + 8 * s, 1); }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "n"(T_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  tc_fence_before();
  find_share<BK, NT>(a, SPLIT, room, &place);
  tc_fence_after();
  if (threadIdx.x == 0) leave_nothing(a, place);
  const uint32_t tmem = *tmem_slot_ptr;
  Cur c{};
  // an item of up to 128 rows has one tile of rows, whose blocks the two score tiles share out; else there are two over the same blocks
  auto two_tiles = [&]() { return min(c.r.n * a.R - c.tile * a.tile_rows, a.tile_rows) > 128; };
  // 168 registers a thread at launch: twice 216 and 72 of the warps that share a scheduler
  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");

  if (warp == 8) {  // ------------------------------------------------------------------------------------------- products
    int slot = 0;
    uint32_t phase = 0, q_phase = 0, p_phase[2] = {0, 0};
    auto arrived = [&]() {  // the ring's next tile
      mbar_wait(B.full + 8 * slot, phase, fail);
      tc_fence_after();
      const int s = slot;
      if (++slot == NS) { slot = 0; phase ^= 1; }
      return s;
    };
    auto scores = [&](int w, int q_tile, int s) {
      const uint32_t q = desc_lo(sQ + q_tile * TILE, DESC_K), k = desc_lo(ring + s * TILE, DESC_K);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {  // 32 bytes of a row, 16384 from slice to slice
          const uint32_t step = (kk >> 2) * 1024 + (kk & 3) * 2;
          mma_ss(tmem + w * BK, q + step, k + step, C::IDESC_S, kk > 0);
        }
        tc_commit(B.s_full + 8 * w);
      }
      __syncwarp();
    };
    auto weighted = [&](int w, int s, bool first) {  // a half of the keys as soon as their weights are there
      const uint32_t v = desc_lo(ring + s * TILE, DESC_MN);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mbar_wait((h ? B.p_full : B.half_p) + 8 * w, p_phase[w], fail);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
            mma_ts(tmem + T_O + w * 128, tmem + w * BK + kk * 8, v + kk * 128, C::IDESC_PV, !first || kk > 0);
        }
        __syncwarp();
      }
      p_phase[w] ^= 1;
    };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    if (c.start(a, SPLIT, place)) do {
      const int n = c.j1 - c.j0;
      if (n == 0) continue;
      mbar_wait(B.q_full, q_phase, fail);
      q_phase ^= 1;
      tc_fence_after();
      if (two_tiles()) {
        int k = arrived();
        scores(0, 0, k);
        scores(1, 1, k);
        commit(B.empty + 8 * k);
        if (n == 1) commit(B.q_empty);
        for (int j = 0; j < n; ++j) {
          const bool more = j + 1 < n;
          const int v = arrived();
          k = more ? arrived() : 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            weighted(w, v, j == 0);
            if (more) scores(w, w, k);
            else commit(B.o_full + 8 * w);
          }
          commit(B.empty + 8 * v);
          if (more) commit(B.empty + 8 * k);
          if (j + 2 == n) commit(B.q_empty);
        }
      } else {
        for (int i = 0; i < min(n, 2); ++i) {
          const int k = arrived();
          scores(i, 0, k);
          commit(B.empty + 8 * k);
        }
        if (n <= 2) commit(B.q_empty);
        for (int i = 0; i < n; ++i) {
          const int w = i & 1, v = arrived();
          weighted(w, v, i < 2);
          commit(B.empty + 8 * v);
          if (i + 2 < n) {
            const int k = arrived();
            scores(w, 0, k);
            commit(B.empty + 8 * k);
            if (i + 3 == n) commit(B.q_empty);
          } else commit(B.o_full + 8 * w);
        }
      }
    } while (c.next(a, SPLIT));
  } else if (warp >= 10) {  // ------------------------------------------------------------------------------------- loaders
    constexpr int PIECES = HD / 8;
    const int row0 = (warp - 10) * 32 * SETS;
    int slot = 0, blocks_so_far = 0, waiting = 0;
    const bool first_loader = warp == 10;
    uint32_t phase = 1, q_phase = 1, landed_phase = 0, w0 = 0, w1 = 0;  // waiting: fills that have not been told of, at w0 (the older) and w1
    auto tell = [&](uint32_t bar) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // what the copies wrote -> the tensor core
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto told = [&]() {  // all of them: nobody waits for what this warp only knows of
      if (!waiting) return;
      cp_wait<0>();
      tell(w0);
      if (waiting == 2) tell(w1);
      waiting = 0;
    };
    auto filled = [&](uint32_t bar) {
      cp_commit();
      if (waiting == 2) {
        cp_wait<2>();
        tell(w0);
        w0 = w1;
        w1 = bar;
      } else {
        (waiting ? w1 : w0) = bar;
        ++waiting;
      }
    };
    auto free_to_fill = [&](uint32_t bar, uint32_t parity) {
      if (__all_sync(L3_FULL, mbar_test(bar, parity))) return;
      told();
      mbar_wait(bar, parity, fail);
    };
    // 32 rows, lane r's at src (null: zeros), into rows row0 .. of the tile
    auto rows = [&](const T* src, uint32_t tile, int row0) {
#pragma unroll 4
      for (int i = 0; i < PIECES; ++i) {
        const int at = i * 32 + lane, r = at / PIECES, p = at % PIECES, row = row0 + r;
        const T* from = reinterpret_cast<const T*>(__shfl_sync(L3_FULL, reinterpret_cast<unsigned long long>(src), r));
        cp16(tile + (p >> 3) * 16384 + row * 128 + (((p & 7) ^ (row & 7)) << 4), from ? from + p * 8 : (const T*)a.q, from != nullptr);
      }
    };
    struct Pages { int of[SETS]; };
    if (c.start(a, SPLIT, place)) do {
      const int n = c.j1 - c.j0;
      if (n == 0) continue;
      const int flat0 = c.tile * a.tile_rows, flats = c.r.n * a.R;
      const int most = c.r.seen((min(flats, flat0 + a.tile_rows) - 1) / a.R);
      const int* table = a.table + c.b * a.table_stride;
      const bool two = two_tiles();
      const int ahead = two ? 1 : 2;  // blocks of keys that are multiplied ahead of the first one's values
      auto queries = [&]() {  // behind the first keys: they need not wait for the products of the item before
        if (tma_q) {
          if (first_loader) {
            free_to_fill(B.q_empty, q_phase);
            if (elect_one()) {
              mbar_expect_tx(B.q_full, (two ? 2 : 1) * TILE);
#pragma unroll 1
              for (int h = 0; h < (two ? 2 : 1); ++h)
#pragma unroll
                for (int x = 0; x < C::QS; ++x)
                  tma_3d(sQ + h * TILE + x * 16384, &maps.q, x * 64, c.g * a.R, c.r.s0 + (flat0 + h * 128) / a.R, B.q_full);
            }
            __syncwarp();
          }
        } else {
          free_to_fill(B.q_empty, q_phase);
#pragma unroll 1
          for (int h = 0; h < (two ? 2 : 1) * SETS; ++h) {
            const int in = row0 + h % SETS * 32, f = flat0 + h / SETS * 128 + in + lane, t = f / a.R;
            rows(f < flats ? (const T*)a.q + (c.r.s0 + t) * a.q_st + (c.g * a.R + f - t * a.R) * a.q_sh : nullptr, sQ + h / SETS * TILE, in);
          }
          filled(B.q_full);
          if (tma_kv) told();  // nothing else would
        }
        q_phase ^= 1;
      };
      if (tma_kv) {
        if (!first_loader) {
          queries();
          continue;
        }
        // one lane a page of the block, or the first one for a part of a page
        const int page_size = 1 << a.log_page, box = min(page_size, BK), pages = BK / box;
        auto page_of = [&](int j) {
          const int key = j * BK + lane * box;
          int page = -1;
          if (lane < pages && key < most) page = __ldg(table + (key >> a.log_page));
          return page;
        };
        auto fill = [&](int named, int j, bool keys) {
          const int page = (unsigned)named < (unsigned)a.n_pages ? named : a.n_pages;  // outside: the copy's rows are zeros
          const uint32_t bar = B.full + 8 * slot, tile = ring + slot * TILE;
          mbar_wait(B.empty + 8 * slot, phase, fail);
          if (keys) {
            const uint32_t ok = __ballot_sync(L3_FULL, page < a.n_pages);
            if (lane < 4) {  // the bits of 32 keys
              uint32_t bits = 0;
              if (box >= 32) bits = ok >> (lane * 32 / box) & 1 ? L3_FULL : 0u;
              else
                for (int x = 0; x < 32 / box; ++x) bits |= ok >> (lane * (32 / box) + x) & 1 ? ((1u << box) - 1) << (x * box) : 0u;
              there[(blocks_so_far & (THERE - 1)) * 4 + lane] = bits;
            }
            ++blocks_so_far;
          }
          // values behind the last token that is seen lie in the last page, and may be no numbers: they become 0
          const int left = most - j * BK, stop = min((left + box - 1) & -box, BK);
          const bool clean = !keys && left < BK && left < stop;
          const uint32_t to = clean ? B.landed : bar;
          __syncwarp();  // the bits of all four lanes, ahead of the arrival
          if (lane == 0) mbar_expect_tx(to, TILE);
          __syncwarp();
          if (lane < pages) {
#pragma unroll
            for (int x = 0; x < C::QS; ++x)
              tma_5d(tile + x * 16384 + lane * box * 128, &maps.kv, x * 64, (j * BK) & (page_size - 1) & -box, c.g, page, keys != keys_first, to);
          }
          __syncwarp();
          if (clean) {
            mbar_wait(B.landed, landed_phase, fail);
            landed_phase ^= 1;
            for (int i = left * 8 + lane; i < stop * 8; i += 32)
#pragma unroll
              for (int x = 0; x < C::QS; ++x)
                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + x * 16384 + i * 16), "r"(0) : "memory");
            tell(bar);
          }
          if (++slot == NS) { slot = 0; phase ^= 1; }
        };
        int next = page_of(c.j0), had = next, had1 = next;  // had ..: of the blocks whose values come next
        for (int x = 0; x < min(ahead, n); ++x) {
          (x ? had1 : had) = next;
          const int page = next;
          next = page_of(c.j0 + x + 1);
          fill(page, c.j0 + x, true);
        }
        queries();
        for (int i = 0; i < n; ++i) {
          fill(had, c.j0 + i, false);
          had = had1;
          if (i + ahead < n) {
            (two ? had : had1) = next;
            const int page = next;
            next = page_of(c.j0 + i + ahead + 1);
            fill(page, c.j0 + i + ahead, true);
          }
        }
        continue;
      }
      auto pages_of = [&](int j) {  // of this lane's keys of block j
        Pages p;
#pragma unroll
        for (int x = 0; x < SETS; ++x) {
          const int key = j * BK + row0 + x * 32 + lane;
          p.of[x] = key < most ? __ldg(table + (key >> a.log_page)) : -1;
        }
        return p;
      };
      auto fill = [&](const PagedPool& p, const Pages& pages, int j, bool keys) {
        free_to_fill(B.empty + 8 * slot, phase);
#pragma unroll
        for (int x = 0; x < SETS; ++x) {
          const int in = row0 + x * 32, place = (j * BK + in + lane) & ((1 << a.log_page) - 1);
          const bool ok = (unsigned)pages.of[x] < (unsigned)a.n_pages;
          if (keys) {
            const uint32_t bits = __ballot_sync(L3_FULL, ok);
            if (lane == 0) there[(blocks_so_far & (THERE - 1)) * 4 + in / 32] = bits;
          }
          rows(ok ? (const T*)p.p + pages.of[x] * p.sp + c.g * p.sh + place * p.st : nullptr, ring + slot * TILE, in);
        }
        blocks_so_far += keys;
        filled(B.full + 8 * slot);
        if (++slot == NS) { slot = 0; phase ^= 1; }
      };
      Pages next = pages_of(c.j0), had = next, had1 = next;
      for (int x = 0; x < min(ahead, n); ++x) {
        (x ? had1 : had) = next;
        const Pages page = next;
        next = pages_of(c.j0 + x + 1);
        fill(a.k, page, c.j0 + x, true);
      }
      queries();
      for (int i = 0; i < n; ++i) {
        fill(a.v, had, c.j0 + i, false);
        had = had1;
        if (i + ahead < n) {
          (two ? had : had1) = next;
          const Pages page = next;
          next = pages_of(c.j0 + i + ahead + 1);
          fill(a.k, page, c.j0 + i + ahead, true);
        }
      }
    } while (c.next(a, SPLIT));
    told();
  } else if (warp == 9) {
    clear_rest<T>(a, lane, 32);
  } else if (warp < 8) {  // ---------------------------------------------------------------------------------------- softmax
    const int quarter = warp & 3, w = warp >> 2, r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + w * BK + lanes, tO = tmem + T_O + lanes;
    // log2(e) |scale|: a weight is 2^(s sc - m sc); of 0 the smallest number, so that a score of -infinity keeps its weight of 0
    const float sc = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f), growth = fminf(C::GROW / sc, 3e38f);
    const bool negative = a.scale < 0.f;
    int blocks_so_far = 0;
    uint32_t s_phase = 0, o_phase[2] = {0, 0};
    if (c.start(a, SPLIT, place)) do {
      const int n = c.j1 - c.j0;
      const bool two = two_tiles();
      const int in_tile = (two ? w * 128 : 0) + r, f = c.tile * a.tile_rows + in_tile, flats = c.r.n * a.R, t = f / a.R;
      const int seen = f < flats ? c.r.seen(t) : INT_MAX;  // a row behind the last: what it has goes nowhere, and masks cost time
      float m = -INFINITY, l = 0.f;  // m: of s, what the exponentials are taken against
      bool begun = false;
      for (int j = two ? 0 : w; j < n; j += two ? 1 : 2) {
        mbar_wait(B.s_full + 8 * w, s_phase, fail);
        s_phase ^= 1;
        tc_fence_after();
        float v[BK];
#pragma unroll
        for (int i = 0; i < BK; i += 32) tmem_ld32(tS + i, v + i);
        tmem_ld_wait();
        const int visible = seen - (c.j0 + j) * BK;
        const uint4 bits = *reinterpret_cast<const uint4*>(there + ((blocks_so_far + j) & (THERE - 1)) * 4);
        if (negative) {
#pragma unroll
          for (int i = 0; i < BK; ++i) v[i] = -v[i];
        }
        if (__any_sync(L3_FULL, visible < BK) || (bits.x & bits.y & bits.z & bits.w) != L3_FULL) {
          const uint32_t words[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int of = visible - 32 * k;
            const uint32_t in = of >= 32 ? words[k] : of <= 0 ? 0u : words[k] & ((1u << of) - 1);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(in >> i & 1)) v[32 * k + i] = -INFINITY;
          }
        }
        // NaN where one of the scores is
        float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int i = 4; i < BK; i += 4)
#pragma unroll
          for (int x = 0; x < 4; ++x) top[x] = max_nan(top[x], v[i + x]);
        float mx = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3]));
        if (mx == INFINITY) mx = NAN;  // as the definition has it: infinity less infinity
        if (!begun) m = mx;
        else {
          const bool grow = !(mx <= m + growth);
          if (__any_sync(L3_FULL, grow)) {
            // the scores of this block are there: the products of every block before have ended, and the output rests
            const float alpha = grow ? ex2((m - mx) * sc) : 1.f;
            if (grow) { m = mx; l *= alpha; }
#pragma unroll 1
            for (int d = 0; d < HD; d += 16) {
              float o[16];
              tmem_ld16(tO + w * 128 + d, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= alpha;
              tmem_st16(tO + w * 128 + d, o);
            }
          }
        }
        begun = true;
        const float down = C::BIAS - (m == -INFINITY ? 0.f : m * sc);
        const float2 sc2 = make_float2(sc, sc), down2 = make_float2(down, down);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float2 x = fma2(make_float2(v[64 * h + i], v[64 * h + i + 1]), sc2, down2);
            const float2 e = i % 8 < 2 * POLY ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[i / 2 & 1] = add2(sum[i / 2 & 1], e);
            p[i / 2] = pack<T>(e.x, e.y);
          }
          tmem_st32(tS + 32 * h, p);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive((h ? B.p_full : B.half_p) + 8 * w);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
      }
      blocks_so_far += n;
      if (m == -INFINITY) l = 0.f;  // nothing seen
      // ---- the result, or this CTA's part of it
      const bool whole = c.whole();
      float* const part_o = whole ? nullptr : a.part_o + (size_t)(2 * blockIdx.x + c.slot()) * a.tile_rows * HD;
      float2* const part_ml = whole ? nullptr : a.part_ml + (size_t)(2 * blockIdx.x + c.slot()) * a.tile_rows;
      if (!whole && threadIdx.x == 0) left_of(a, blockIdx.x).part[c.slot()] = make_int4(c.b, c.tile, c.g, c.j1 == c.nb);
      float m2 = m == -INFINITY ? m : m * sc - C::BIAS;  // in units of log 2
      float share = 1.f, share1 = 0.f;                    // of the outputs: this tile's, or the first's and the second's
      if (n) {
        // an output's end is told of only where it has blocks: else the next item's could come before a warp has seen this one's
        const bool second = two || n > 1;
        if (!two || w == 0) mbar_wait(B.o_full, o_phase[0], fail);
        if (second && (!two || w == 1)) mbar_wait(B.o_full + 8, o_phase[1], fail);
        o_phase[0] ^= 1;
        o_phase[1] ^= second;
        __syncwarp();
        if (!two) {
          // one float a row, twice: there is no more room beside the tiles
          xch[warp][lane] = m2;
          asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");
          float2 other;
          other.x = xch[warp ^ 4][lane];
          asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");
          xch[warp][lane] = l;
          asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");
          other.y = xch[warp ^ 4][lane];
          const float both = fmaxf(m2, other.x), from = both == -INFINITY ? 0.f : both;
          const float mf = ex2(m2 - from), of = ex2(other.x - from);
          l = l * mf + other.y * of;
          m2 = both;
          share = w ? of : mf;
          share1 = w ? mf : of;
        }
        tc_fence_after();
      }
      const long long at = (long long)(c.r.s0 + t) * a.H + c.g * a.R + f - t * a.R;
      if (*fail) l = NAN;  // a wait ran out
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bool finite = l < INFINITY;
      if (two) {  // a row's columns, 16 at a time: 32 bytes of the result, 64 of a partial
        const bool wide = ((uintptr_t)a.out & 31) == 0;
#pragma unroll 1
        for (int d = 0; d < HD; d += 16) {
          float o[16];
          if (n) {
            tmem_ld16(tO + w * 128 + d, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) finite = finite && fabsf(o[i]) < INFINITY;
          if (f < flats) {
            if (whole) {
              uint32_t x[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = pack<T>(o[2 * i] * inv, o[2 * i + 1] * inv);
              T* const to = (T*)a.out + at * HD + d;
              if (wide) store32(to, x);
              else {
                *reinterpret_cast<uint4*>(to) = make_uint4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<uint4*>(to + 8) = make_uint4(x[4], x[5], x[6], x[7]);
              }
            } else {
              float* const to = part_o + (size_t)in_tile * HD + d;
              store32(to, reinterpret_cast<const uint32_t*>(o));
              store32(to + 8, reinterpret_cast<const uint32_t*>(o) + 8);
            }
          }
          __syncwarp();
        }
      } else {  // half of a row's columns, 8 at a time, of both outputs
#pragma unroll 1
        for (int d = w * (HD / 2); d < (w + 1) * (HD / 2); d += 8) {
          float o[8], o1[8];
          if (n) {
            tmem_ld8(tO + d, o);
            tmem_ld8(tO + 128 + d, o1);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = n > 1 ? o[i] * share + o1[i] * share1 : o[i] * share;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) finite = finite && fabsf(o[i]) < INFINITY;
          if (f < flats) {
            if (whole) {
              *reinterpret_cast<uint4*>((T*)a.out + at * HD + d) =
                  make_uint4(pack<T>(o[0] * inv, o[1] * inv), pack<T>(o[2] * inv, o[3] * inv), pack<T>(o[4] * inv, o[5] * inv), pack<T>(o[6] * inv, o[7] * inv));
            } else store32(part_o + (size_t)in_tile * HD + d, reinterpret_cast<const uint32_t*>(o));
          }
          __syncwarp();
        }
      }
      if (f < flats && (two || w == 0)) {
        if (!whole) part_ml[in_tile] = make_float2(m2, l);
        else if (a.lse) a.lse[at] = (m2 + log2f(l)) * 0.6931471805599453f;
      }
      tc_fence_before();
      if (whole && f < flats && !finite) left_of(a, blockIdx.x).odd = 1;
      if (!two) asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");  // both have read the outputs
    } while (c.next(a, SPLIT));
  }
  tc_fence_before();
  __syncthreads();
  if (*fail) __nanosleep(1000000);  // copies still in flight land before the shared memory is given up
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(T_COLS));
}

// Rows of an item, 128 or 256: 256 - every key that arrives is used twice as often - where that makes items enough for all SMs, or a request has many rows
// and may have many keys.  us, 128 : 256, 32 heads over 8 kv heads of 128, bf16: 16 x 128 rows over no others 31.7 : 24.8, 2048 over none 79.7 : 69.9,
// 511 over 65000 597 : 472, 20 x 33 over 2000 85.5 : 68.5; but 200 over none 17.5 : 20.5, 200 over 500 27.1 : 30.4, 100 over 4000 33.0 : 38.8; 20 x 33 over 2000,
// 16 heads with keys of their own, 84.4 : 86.2
int rows_of_item(const ChunkArgs& a, int n_sm) {
  const long long rows = (long long)a.T * a.R, keys = (long long)a.max_pages << a.log_page;
  const long long tiles = std::max((rows + 255) / 256, rows > 128LL * a.B ? (long long)a.B : 0) * a.G;
  return tiles >= n_sm || (rows >= 256LL * a.B && tiles * keys >= (long long)n_sm * 2048) ? 256 : 128;
}
// Whether, and how, tiles are copied by TMA: a box is 64 entries of as many rows as lie side by side.  Distances of 0 between different rows are not for it.
bool usable(long long stride, long long n) { return n <= 1 || (stride > 0 && stride < (1LL << 38)); }
bool map_pools(const ChunkArgs& a, CUtensorMap* map, bool* keys_first) {
  const PagedPool &p = a.k, &v = a.v;
  const long long apart = (const char*)v.p - (const char*)p.p;
  *keys_first = apart > 0;
  if (a.log_page < 3 || p.sp != v.sp || p.sh != v.sh || p.st != v.st || apart == 0 || !usable(p.sp, a.n_pages) || !usable(p.sh, a.G) || !usable(p.st, 2) ||
      !usable(std::abs(apart) / 2, 2))
    return false;
  const uint64_t dims[5] = {(uint64_t)a.HD, 1ull << a.log_page, (uint64_t)a.G, (uint64_t)a.n_pages, 2};
  const uint64_t strides[4] = {(uint64_t)p.st * 2, (uint64_t)std::max(p.sh, 8LL) * 2, (uint64_t)std::max(p.sp, 8LL) * 2, (uint64_t)std::abs(apart)};
  const uint32_t box[5] = {64, (uint32_t)std::min(1 << a.log_page, BK), 1, 1, 1};
  return tc_make_map(map, apart > 0 ? p.p : v.p, a.dtype == L3_DTYPE_BF16, 5, dims, strides, box);
}
// us, by TMA : row by row, bf16: six prompts of up to 4096 tokens 455 : 553, 20 x 33 rows over 2000 tokens 81 : 85, 64 rows 16.0 : 17.0
bool map_q(const ChunkArgs& a, CUtensorMap* map) {
  if (128 % a.R || !usable(a.q_sh, a.H) || !usable(a.q_st, a.T)) return false;
  const uint64_t dims[3] = {(uint64_t)a.HD, (uint64_t)a.H, (uint64_t)a.T};
  const uint64_t strides[2] = {(uint64_t)std::max(a.q_sh, 8LL) * 2, (uint64_t)std::max(a.q_st, 8LL) * 2};
  const uint32_t box[3] = {64, (uint32_t)a.R, (uint32_t)(128 / a.R)};
  return tc_make_map(map, a.q, a.dtype == L3_DTYPE_BF16, 3, dims, strides, box);
}
template <typename T, int HD> cudaError_t launch_hd(ChunkArgs a, int n_sm, cudaStream_t s) {
  using C = Cfg<T, HD>;
  a.n_cta = n_sm;
  a.tile_rows = rows_of_item(a, n_sm);
  a.part_o = part_begin(a.ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)a.n_cta * 2 * a.tile_rows * HD);
  a.left = a.part_ml + (size_t)a.n_cta * 2 * a.tile_rows;
  cudaError_t e = allow_smem(chunk_tc_kernel<T, HD>, C::SMEM);
  if (e != cudaSuccess) return e;
  Maps maps{};
  bool keys_first;
  const bool tma_q = map_q(a, &maps.q), tma_kv = map_pools(a, &maps.kv, &keys_first);
  if ((e = launch_k(chunk_tc_kernel<T, HD>, dim3(a.n_cta), dim3(NT), (size_t)C::SMEM, s, a, maps, tma_q, tma_kv, keys_first)) != cudaSuccess) return e;
  return launch_chunk_join_tc(a, s);
}
template <typename T> cudaError_t launch_t(const ChunkArgs& a, int n_sm, cudaStream_t s) {
  switch (a.HD) {
    case 16: return launch_hd<T, 16>(a, n_sm, s);
    case 32: return launch_hd<T, 32>(a, n_sm, s);
    case 48: return launch_hd<T, 48>(a, n_sm, s);
    case 64: return launch_hd<T, 64>(a, n_sm, s);
    case 96: return launch_hd<T, 96>(a, n_sm, s);
    case 128: return launch_hd<T, 128>(a, n_sm, s);
    default: return cudaErrorInvalidValue;
  }
}
}  // namespace

cudaError_t launch_paged_chunk_tc(const ChunkArgs& a, int n_sm, cudaStream_t s) {
  return a.dtype == L3_DTYPE_BF16 ? launch_t<bf16>(a, n_sm, s) : launch_t<__half>(a, n_sm, s);
}

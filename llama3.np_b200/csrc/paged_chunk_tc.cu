// Attention of the rows of a packed step over a 16-bit cache in pages (paged_chunk.cu has the formula, paged_chunk.cuh how the work is cut), on
// tcgen05: a CTA an SM, blocks of 128 keys, score tiles of 128 rows x 128 keys.
//
//   warps 10, 11  loaders: the item's queries, then keys and values of its blocks, row by row through the page table, 16 bytes a copy
//                 (cp.async; any page size and strides), into a ring of operand tiles (K-major rows of 128 bytes, swizzled); rows of no
//                 token become zeros, and their bits go to the softmax warps
//   warp 8        products: S = Q K^T into TMEM, O += P V with P from TMEM and V as it lies, an MN-major operand
//   warps 0 - 7   softmax, a thread a row, four warps a score tile: its 128 scores in registers, exponentials against a maximum that follows
//                 the running one lazily (O is rescaled in TMEM only when that has grown by 2^GROW), weights as 16-bit values over the scores
// The two score tiles take turns: one's softmax runs while the tensor core works on the other's products.  With many rows they are two tiles of
// rows over the same keys, so that every key and value that arrives is used for 256 rows; with few rows they are one tile of rows over every other
// block of keys, and meet at the end.
//
// A weight enters the product rounded to the cache's type (half a step: bf16 2^-9 of it, as much as the result's own rounding; sums are of the unrounded
// ones, in fp32).  fp16 weights are scaled by 2^BIAS ahead of the rounding: the largest lies in [2^12, 2^15], what fp16 has no number for is below
// 2^-37 of it.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "gemm_tc_dev.cuh"
#include "paged_chunk_tc.h"
#include "paged_chunk.cuh"

namespace {
using namespace chunk;
constexpr int BK = TC_BK, NT = 384, SOFT = 256, LOADERS = 2, SETS = 4 / LOADERS;  // SETS: of 32 rows of a tile, a loader's
constexpr int WHOLE = TC_WHOLE, LEAST = 4;
constexpr int THERE = 16;  // blocks whose keys' bits are kept: more than the ring holds

template <typename T, int HD, bool TWO> struct Cfg {
  static constexpr int TR = TWO ? 256 : 128;
  static constexpr int QS = (HD + 63) / 64;             // slices of 64 entries, rows of 128 bytes
  static constexpr int TILE = QS * 128 * 128;           // bytes of 128 rows
  static constexpr int NS = HD > 64 ? 5 : 8;            // tiles of the ring
  static constexpr int AHEAD = TWO ? 1 : 2;             // blocks of keys that are multiplied ahead of the first one's values
  static constexpr int SMEM = (TWO ? 2 : 1) * TILE + NS * TILE + THERE * 16 + (TWO ? 0 : 2 * 128 * 8) + 256 + 1024;
  static constexpr uint32_t FMT = std::is_same<T, bf16>::value ? 1u : 0u;
  static constexpr uint32_t IDESC_S = (1u << 4) | (FMT << 7) | (FMT << 10) | ((uint32_t)(BK >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr uint32_t IDESC_PV = (1u << 4) | (FMT << 7) | (FMT << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((128u >> 4) << 24);
  static constexpr float BIAS = FMT ? 0.f : 12.f, GROW = FMT ? 8.f : 3.f;
};
// TMEM columns: two score tiles (the weights lie over their first halves), two outputs
constexpr int T_O = 256, T_COLS = 512;

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
// MN-major operand, 128-byte swizzle: rows are the keys (the product's K), 8 of them a 1024-byte atom; atoms of 64 columns are lbo bytes apart
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// A from TMEM: a lane a row, two neighbouring entries a column
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accum) : "memory");
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

// Barriers of a CTA, 8 bytes each.
struct Bars {
  uint32_t q_full, q_empty, s_full, p_full, o_full, full, empty;  // s_full, p_full, o_full: of both score tiles
};

template <typename T, int HD, bool TWO>
__global__ void __launch_bounds__(NT, 1) chunk_tc_kernel(const ChunkArgs a) {
  using C = Cfg<T, HD, TWO>;
  constexpr int TR = C::TR, NS = C::NS, TILE = C::TILE, AHEAD = C::AHEAD;
  using Cur = Cursor<TR, BK, WHOLE>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ long long room[NT / 32 + 1];
  __shared__ Place place;
  __shared__ int failed;
  volatile int* const fail = &failed;
  const uint32_t raw = smem_u32(smem_raw), sQ = (raw + 1023u) & ~1023u, ring = sQ + (TWO ? 2 : 1) * TILE;
  uint8_t* const rest = smem_raw + (ring + NS * TILE - raw);
  uint32_t* const there = reinterpret_cast<uint32_t*>(rest);                  // [THERE][4]
  float2* const xch = reinterpret_cast<float2*>(rest + THERE * 16);           // [2][128], one tile of rows
  const uint32_t bars = ring + NS * TILE + THERE * 16 + (TWO ? 0 : 2 * 128 * 8);
  const Bars B{bars, bars + 8, bars + 16, bars + 32, bars + 48, bars + 64, bars + 64 + 8 * NS};
  const uint32_t tmem_slot = B.empty + 8 * NS;
  uint32_t* const tmem_slot_ptr = reinterpret_cast<uint32_t*>(smem_raw + (tmem_slot - raw));
  const int warp = __shfl_sync(L3_FULL, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  pdl_launch();
  pdl_wait();
  clear_rest<T>(a);
  find_share<TR, BK, NT, LEAST>(a, room, &place);
  if (threadIdx.x == 0) leave_nothing(a, place);
  if (place.b < 0) return;
  if (threadIdx.x == 0) {
    mbar_init(B.q_full, LOADERS);
    mbar_init(B.q_empty, 1);
    for (int w = 0; w < 2; ++w) { mbar_init(B.s_full + 8 * w, 1); mbar_init(B.p_full + 8 * w, 4); mbar_init(B.o_full + 8 * w, 1); }
    for (int s = 0; s < NS; ++s) { mbar_init(B.full + 8 * s, LOADERS); mbar_init(B.empty + 8 * s, 1); }
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "n"(T_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  Cur c;
  // 168 registers a thread at launch: twice 216 and 72 of the warps that share a scheduler
  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");

  if (warp == 8) {  // ------------------------------------------------------------------------------------------- products
    int slot = 0;
    uint32_t phase = 0, q_phase = 0, p_phase[2] = {0, 0};
    auto arrived = [&]() {  // the ring's next tile
      mbar_wait(B.full + 8 * slot, phase, fail);
      const int s = slot;
      if (++slot == NS) { slot = 0; phase ^= 1; }
      return s;
    };
    auto scores = [&](int w, int s) {
      const uint32_t q = sQ + (TWO ? w * TILE : 0), k = ring + s * TILE;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint64_t step = (uint64_t)((kk & 3) * 2);
          tc_mma<TC_BF16>(tmem + w * BK, umma_desc_sw128(q + (kk >> 2) * 16384) + step, umma_desc_sw128(k + (kk >> 2) * 16384) + step, C::IDESC_S, kk > 0);
        }
        tc_commit(B.s_full + 8 * w);
      }
      __syncwarp();
    };
    auto weighted = [&](int w, int s, bool first) {
      mbar_wait(B.p_full + 8 * w, p_phase[w], fail);
      p_phase[w] ^= 1;
      tc_fence_after();
      const uint32_t v = ring + s * TILE;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk)
          mma_ts(tmem + T_O + w * 128, tmem + w * BK + kk * 8, desc_mn(v + kk * 2048, 16384), C::IDESC_PV, !first || kk > 0);
      }
      __syncwarp();
    };
    auto commit = [&](uint32_t bar) {
      if (elect_one()) tc_commit(bar);
      __syncwarp();
    };
    if (c.start(a, place)) do {
      const int n = c.j1 - c.j0;
      if (n == 0) continue;
      mbar_wait(B.q_full, q_phase, fail);
      q_phase ^= 1;
      tc_fence_after();
      if constexpr (TWO) {
        int k = arrived();
        tc_fence_after();
        scores(0, k);
        scores(1, k);
        commit(B.empty + 8 * k);
        if (n == 1) commit(B.q_empty);
        for (int j = 0; j < n; ++j) {
          const bool more = j + 1 < n;
          const int v = arrived();
          k = more ? arrived() : 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            weighted(w, v, j == 0);
            if (more) scores(w, k);
            else commit(B.o_full + 8 * w);
          }
          commit(B.empty + 8 * v);
          if (more) commit(B.empty + 8 * k);
          if (j + 2 == n) commit(B.q_empty);
        }
      } else {
        for (int i = 0; i < min(n, 2); ++i) {
          const int k = arrived();
          tc_fence_after();
          scores(i, k);
          commit(B.empty + 8 * k);
        }
        if (n <= 2) commit(B.q_empty);
        if (n == 1) commit(B.o_full + 8);  // it has no block
        for (int i = 0; i < n; ++i) {
          const int w = i & 1, v = arrived();
          weighted(w, v, i < 2);
          if (i + 2 < n) {
            commit(B.empty + 8 * v);
            const int k = arrived();
            tc_fence_after();
            scores(w, k);
            commit(B.empty + 8 * k);
            if (i + 3 == n) commit(B.q_empty);
          } else {
            commit(B.o_full + 8 * w);
            commit(B.empty + 8 * v);
          }
        }
      }
    } while (c.next(a));
  } else if (warp >= 10) {  // ------------------------------------------------------------------------------------- loaders
    constexpr int PIECES = HD / 8;
    const int row0 = (warp - 10) * 32 * SETS;
    int slot = 0, blocks_so_far = 0, waiting = 0;
    uint32_t phase = 1, q_phase = 1, w0 = 0, w1 = 0;  // waiting: fills that have not been told of, at w0 (the older) and w1
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
      if (mbar_test(bar, parity)) return;
      told();
      mbar_wait(bar, parity, fail);
    };
    // 32 rows, lane r's at src (null: zeros), into rows row0 .. of the tile
    auto rows = [&](const T* src, uint32_t tile, int row0) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int at = i * 32 + lane, r = at / PIECES, p = at % PIECES, row = row0 + r;
        const T* from = reinterpret_cast<const T*>(__shfl_sync(L3_FULL, reinterpret_cast<unsigned long long>(src), r));
        cp16(tile + (p >> 3) * 16384 + row * 128 + (((p & 7) ^ (row & 7)) << 4), from ? from + p * 8 : (const T*)a.q, from != nullptr);
      }
    };
    struct Pages { int of[SETS]; };
    if (c.start(a, place)) do {
      const int n = c.j1 - c.j0;
      if (n == 0) continue;
      const int flat0 = c.tile * TR, flats = c.r.n * a.R;
      const int most = c.r.seen((min(flats, flat0 + TR) - 1) / a.R);
      const int* table = a.table + c.b * a.table_stride;
      free_to_fill(B.q_empty, q_phase);
      q_phase ^= 1;
#pragma unroll 1
      for (int h = 0; h < TR / 128 * SETS; ++h) {
        const int in = row0 + h % SETS * 32, f = flat0 + h / SETS * 128 + in + lane, t = f / a.R;
        rows(f < flats ? (const T*)a.q + (c.r.s0 + t) * a.q_st + (c.g * a.R + f - t * a.R) * a.q_sh : nullptr, sQ + h / SETS * TILE, in);
      }
      filled(B.q_full);
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
      Pages next = pages_of(c.j0), had[AHEAD];
#pragma unroll
      for (int x = 0; x < AHEAD; ++x)
        if (x < n) {
          had[x] = next;
          next = pages_of(c.j0 + x + 1);
          fill(a.k, had[x], c.j0 + x, true);
        }
      for (int i = 0; i < n; ++i) {
        fill(a.v, had[0], c.j0 + i, false);
#pragma unroll
        for (int x = 0; x + 1 < AHEAD; ++x) had[x] = had[x + 1];
        if (i + AHEAD < n) {
          had[AHEAD - 1] = next;
          next = pages_of(c.j0 + i + AHEAD + 1);
          fill(a.k, had[AHEAD - 1], c.j0 + i + AHEAD, true);
        }
      }
    } while (c.next(a));
    told();
  } else if (warp < 8) {  // ---------------------------------------------------------------------------------------- softmax
    const int quarter = warp & 3, w = warp >> 2, r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, tS = tmem + w * BK + lanes, tO = tmem + T_O + lanes;
    // log2(e) |scale|: a weight is 2^(s sc - m sc); of 0 the smallest number, so that a score of -infinity keeps its weight of 0
    const float sc = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.4e-45f);
    const bool negative = a.scale < 0.f;
    int blocks_so_far = 0;
    uint32_t s_phase = 0, o_phase = 0;
    if (c.start(a, place)) do {
      const int n = c.j1 - c.j0;
      const int in_tile = (TWO ? w * 128 : 0) + r, f = c.tile * TR + in_tile, flats = c.r.n * a.R, t = f / a.R;
      const int seen = f < flats ? c.r.seen(t) : 0;
      float m = -INFINITY, l = 0.f;  // m: of s, what the exponentials are taken against
      bool begun = false;
      for (int j = TWO ? 0 : w; j < n; j += TWO ? 1 : 2) {
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
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < BK; i += 4)
#pragma unroll
          for (int x = 0; x < 4; ++x) top[x] = fmaxf(top[x], v[i + x]);
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (!begun) m = mx;
        else {
          // the scores of block j are there: the products of every block before have ended, and the output rests
          const bool grow = (mx - m) * sc > C::GROW;
          if (__any_sync(L3_FULL, grow)) {
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
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float x = ex2(fmaf(v[64 * h + i], sc, down)), y = ex2(fmaf(v[64 * h + i + 1], sc, down));
            sum[i & 2] += x;
            sum[(i & 2) + 1] += y;
            p[i / 2] = pack<T>(x, y);
          }
          tmem_st32(tS + 32 * h, p);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(B.p_full + 8 * w);
      }
      blocks_so_far += n;
      // ---- the result, or this CTA's part of it
      const bool whole = c.whole();
      float* const part_o = whole ? nullptr : a.part_o + (size_t)(2 * blockIdx.x + c.slot()) * TR * HD;
      float2* const part_ml = whole ? nullptr : a.part_ml + (size_t)(2 * blockIdx.x + c.slot()) * TR;
      if (!whole && threadIdx.x == 0) left_of(a, blockIdx.x).part[c.slot()] = make_int4(c.b, c.tile, c.g, c.j1 == c.nb);
      float m2 = m == -INFINITY ? m : m * sc - C::BIAS;  // in units of log 2
      float share = 1.f, share1 = 0.f;                    // of the outputs: this tile's, or the first's and the second's
      if (n) {
        mbar_wait(B.o_full + 8 * w, o_phase, fail);
        if constexpr (!TWO) {
          mbar_wait(B.o_full + 8 * (w ^ 1), o_phase, fail);
          xch[w * 128 + r] = make_float2(m2, l);
          asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");
          const float2 other = xch[(w ^ 1) * 128 + r];
          const float both = fmaxf(m2, other.x), from = both == -INFINITY ? 0.f : both;
          const float mine = ex2(m2 - from), its = ex2(other.x - from);
          l = l * mine + other.y * its;
          m2 = both;
          share = w ? its : mine;
          share1 = w ? mine : its;
        }
        o_phase ^= 1;
        tc_fence_after();
      }
      constexpr int D0 = TWO ? HD : HD / 2, STEP = D0 % 16 ? 8 : 16;  // columns of this thread
      const int first = TWO ? 0 : w * D0;
      const long long at = (long long)(c.r.s0 + t) * a.H + c.g * a.R + f - t * a.R;
      const float inv = *fail ? NAN : l == 0.f ? 0.f : 1.f / l;
      bool finite = l < INFINITY;
#pragma unroll 1
      for (int d = first; d < first + D0; d += STEP) {
        float o[STEP];
        if (n) {
          if constexpr (STEP == 16) tmem_ld16(tO + (TWO ? w * 128 : 0) + d, o);
          else tmem_ld8(tO + d, o);
          if constexpr (!TWO) {
            float o1[STEP];
            if constexpr (STEP == 16) tmem_ld16(tO + 128 + d, o1);
            else tmem_ld8(tO + 128 + d, o1);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < STEP; ++i) o[i] = n > 1 ? o[i] * share + o1[i] * share1 : o[i] * share;
          } else tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < STEP; ++i) o[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < STEP; ++i) finite = finite && fabsf(o[i]) < INFINITY;
        if (f < flats) {
          if (whole) {
            uint32_t x[STEP / 2];
#pragma unroll
            for (int i = 0; i < STEP; i += 2) x[i / 2] = pack<T>(o[i] * inv, o[i + 1] * inv);
#pragma unroll
            for (int i = 0; i < STEP / 2; i += 4) *reinterpret_cast<uint4*>((T*)a.out + at * HD + d + 2 * i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < STEP; i += 4) *reinterpret_cast<float4*>(part_o + (size_t)in_tile * HD + d + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      if (f < flats && (TWO || w == 0)) {
        if (!whole) part_ml[in_tile] = make_float2(*fail ? NAN : m2, l);
        else if (a.lse) a.lse[at] = (m2 + log2f(l)) * 0.6931471805599453f;
      }
      tc_fence_before();
      if (whole && f < flats && !finite) left_of(a, blockIdx.x).odd = 1;
      if constexpr (!TWO) asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory");  // both have read the outputs, and the other's maximum
    } while (c.next(a));
  }
  tc_fence_before();
  __syncthreads();
  if (*fail) __nanosleep(1000000);  // copies still in flight land before the shared memory is given up
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(T_COLS));
}

template <typename T, int HD, bool TWO> cudaError_t launch_one(ChunkArgs a, int n_sm, cudaStream_t s) {
  using C = Cfg<T, HD, TWO>;
  a.n_cta = n_sm;
  a.part_o = (float*)a.ws;
  a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)a.n_cta * 2 * C::TR * HD);
  a.left = a.part_ml + (size_t)a.n_cta * 2 * C::TR;
  cudaError_t e = allow_smem(chunk_tc_kernel<T, HD, TWO>, C::SMEM);
  if (e != cudaSuccess) return e;
  if ((e = launch_k(chunk_tc_kernel<T, HD, TWO>, dim3(a.n_cta), dim3(NT), (size_t)C::SMEM, s, a)) != cudaSuccess) return e;
  return launch_chunk_join_tc(a, C::TR, s);
}
// Two tiles of rows where there are enough of them for all SMs, or a request has many rows and may have many keys.
template <typename T, int HD> cudaError_t launch_hd(const ChunkArgs& a, int n_sm, cudaStream_t s) {
  if (paged_chunk_tc_rows(a.T, a.H, a.G, a.B, a.max_pages << a.log_page, n_sm) == 256) return launch_one<T, HD, true>(a, n_sm, s);
  return launch_one<T, HD, false>(a, n_sm, s);
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

int paged_chunk_tc_rows(int T, int H, int G, int B, long long keys, int n_sm) {
  const long long rows = (long long)T * (H / G), tiles = (rows + 255) / 256 * G;  // about
  return tiles >= n_sm || (rows >= 256LL * B && tiles * keys >= (long long)n_sm * 2048) ? 256 : 128;
}
cudaError_t launch_paged_chunk_tc(const ChunkArgs& a, int n_sm, cudaStream_t s) {
  return a.dtype == L3_DTYPE_BF16 ? launch_t<bf16>(a, n_sm, s) : launch_t<__half>(a, n_sm, s);
}

// Attention of a few query tokens per sequence over the FP8 paged cache, on
// the tensor cores (head sizes 64 and 128), sm_100a.
//
// Bound: the cache is read once, one byte per value, so HBM; at 23 B per clock
// and SM a tile of 128 keys (32 KB of K and V at D = 128) is due every 1.4 k
// clocks.  Nothing but the softmax runs on the CUDA cores: the cache's E4M3
// codes go from HBM through TMA straight into tcgen05 (kind::f8f6f4).
//
// * S^T = K q^T per tile: the 128 keys are the M rows, the up to 64 query rows
//   that share the key head the N columns, so few rows waste no tensor work
//   and a thread of the epilogue holds one key's scores.
// * O^T += V^T p^T: V as it lies in the cache is the MN-major A operand.
// * q and p are each fed as TWO E4M3 terms, hi = the nearest E4M3 value and
//   lo = the nearest to what remains: q (8 significant bits) is exact over ten
//   octaves below the row's largest value, p is within 2^-9.  The terms are
//   columns side by side of one product (2 N columns; a small product's time
//   goes by its A operand), added where they are read; no code is ever widened.
// * Scales are powers of two: the page scale of K goes into the exponent's
//   factor, that of V into p before it is rounded.
// * Running maxima are lazy.  A column's p are taken relative to a reference
//   that only moves when some p would pass 2^4 (of the row) or its scaled E4M3
//   value 448, found by a vote of the tile's threads; O is then rescaled in
//   TMEM.  After the first tile this is rare, so the common tile costs one
//   vote and no cross-thread maximum.
//
// Work: all (sequence, key head, row chunk) units' key tiles in one line, cut
// into equal shares, one per CTA (whatever the lengths, every SM gets the same
// bytes).  A CTA runs its share as pieces of units; two softmax warpgroups
// take a piece's tiles alternately, each with its own statistics and O, and
// join at the piece's end.  Pieces of a unit that several CTAs share are
// joined by the one that arrives last, in CTA order: the result does not
// depend on which one that is.
#pragma once

#include "wd_attn_fp8.cuh"
#include "wd_router_scored.cuh"  // order_key
#include "wd_tc.cuh"

namespace wdb {

constexpr int AT_TILE = 128;       // keys of a tile
constexpr int AT_THREADS = 320;    // producer, MMA, two warpgroups of four warps
constexpr int AT_MAX_PAGES = 8;    // pages of a tile (16 tokens each)
constexpr int AT_MAX_STAGES = 12;
// log2 of the E4M3 value that the largest p is stored as when references are
// set: 7 x room to grow before they move again, E4M3's quantum 2^-9 at 2^-15.
constexpr float AT_HEAD = 6.f;
constexpr int AT_MAX_CTAS = 160;   // pieces of a unit: their factors fit where q and p lay
constexpr int AT_COUNTERS = 1024;  // bytes of counters at the workspace's start, one of 4 per CTA

template <int kD, int kN>
struct AttnTcShape {
  static constexpr int kKvBytes = AT_TILE * kD;              // K or V of a tile
  static constexpr int kQBytes = kN * kD;                    // one term of q
  static constexpr int kPBytes = AT_TILE * kN;               // one term of p
  // Score tiles in TMEM: with four, the product of a warpgroup's next tile is
  // done while it still works on this one (512 columns hold two at N = 64).
  static constexpr int kScores = kN == 64 ? 2 : 4;
  static constexpr int kTmem = kN == 16 ? 256 : 512;  // columns: scores and both O, 2 N each
  static constexpr int kStages = kD == 64 ? (kN == 64 ? 9 : 10) : (kN == 64 ? 5 : 6);
  static constexpr int kOffQ = kStages * 2 * kKvBytes;
  static constexpr int kOffP = kOffQ + 2 * kQBytes;
  static constexpr int kMiscBytes = kN == 64 ? 10240 : 6144;
  static constexpr int kOffMisc = kOffP + 4 * kPBytes;
  static constexpr int kSmem = kOffMisc + kMiscBytes + 1024;  // + alignment slack
  // floats of one split piece in the workspace: O [N][D], then l, m, M of each column
  static constexpr int kSlotFloats = kN * kD + 3 * kN;
};

struct AttnTcArgs {
  AttnArgs a;
  uint32_t* counters;  // one per CTA; zero between calls
  float* slots;        // two per CTA
  int chunks;          // row chunks of a (sequence, key head)
  int min_tiles;       // least tiles of a CTA's share
  int reach;           // tokens that the block table can address
  int page_shift;
};

// Keys [kmin, kmax] that the rows of chunk c see, as far as the table reaches,
// and their tiles; none: one tile, all masked.
__device__ __forceinline__ void attn_unit(const AttnTcArgs& t, int len, int G, int rows, int kN, int c,
                                          int* kmin, int* kmax, int* tiles) {
  const int r0 = c * kN, r1 = min(r0 + kN, rows);
  const int p0 = len - t.a.Sq + r0 / G, p1 = min(len - t.a.Sq + (r1 - 1) / G, t.reach - 1);
  *kmax = p1;
  *kmin = t.a.window > 0 ? max(0, p0 - t.a.window + 1) : 0;
  *tiles = p1 < *kmin ? 1 : p1 / AT_TILE - *kmin / AT_TILE + 1;
}

// Equal shares of `total` tiles over `ctas` CTAs: first tile of CTA i, CTA of a tile.
struct AttnShares {
  int each, more;  // the first `more` CTAs take one tile more
  __device__ __forceinline__ int first(int i) const { return i * each + min(i, more); }
  __device__ __forceinline__ int cta_of(int tile) const {
    const int wide = more * (each + 1);
    return tile < wide ? tile / (each + 1) : more + (tile - wide) / each;
  }
};

// A CTA's share of the tiles, as pieces of units; every role walks the same.
struct AttnWalk {
  int pos, end, unit;  // next tile, end of the share, first tile of the current unit
  int b, h, c, len;
  int kmin, kmax, tiles;     // of the current unit
};

template <int kN>
__device__ __forceinline__ void walk_unit(const AttnTcArgs& t, int G, int rows, AttnWalk& w) {
  attn_unit(t, w.len, G, rows, kN, w.c, &w.kmin, &w.kmax, &w.tiles);
}

template <int kN>
__device__ __forceinline__ void walk_next(const AttnTcArgs& t, int G, int rows, AttnWalk& w) {
  w.unit += w.tiles;
  if (++w.c == t.chunks) {
    w.c = 0;
    if (++w.h == t.a.Hkv) {
      w.h = 0;
      ++w.b;
      if (w.b < t.a.B) w.len = __ldg(t.a.seq_lens + w.b);
    }
  }
  walk_unit<kN>(t, G, rows, w);
}

__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// One lane of the (converged) warp; the compiler knows that it is one.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0u;
}

// Largest of the warp's values (NaN only if all are).
__device__ __forceinline__ float warp_max_f32(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// `bar` arrivals without waiting, to pair with named_barrier_sync.
__device__ __forceinline__ void named_barrier_arrive(int id, int nthreads) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// Instruction descriptor for kind::f8f6f4: fp32 D, E4M3 A and B; a_mn / b_mn:
// the operand is MN-major (its M or N index is the contiguous one).
__host__ __device__ constexpr uint32_t tc_idesc_e4m3(int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(M >> 4) << 24);
}

// Shared-memory matrix descriptor: byte offsets, layout 0 none, 2 128-byte
// swizzle, 4 64-byte swizzle.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr, uint32_t leading, uint32_t stride, uint32_t layout) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((leading >> 4) & 0x3FFFu) << 16 |
         (uint64_t)((stride >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)layout << 61;
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}

// Barrier `id` over `n` threads that also tells every one whether some thread's
// `p` holds.
__device__ __forceinline__ bool named_barrier_any(int id, int n, bool p) {
  uint32_t r;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred a, b;\n\t"
      "setp.ne.u32 a, %3, 0;\n\t"
      "barrier.cta.red.or.pred b, %1, %2, a;\n\t"
      "selp.u32 %0, 1, 0, b;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"((uint32_t)p)
      : "memory");
  return r != 0u;
}

// v[0..kN): one value per column in every lane.  Afterwards v[j], j < kN / 32
// (1 for kN = 16), holds the warp's sum of column columns_of(lane, j).
template <int kN>
__device__ __forceinline__ void warp_sum_columns(float (&v)[kN], int lane) {
  constexpr int kHalvings = kN >= 32 ? 5 : 4;
#pragma unroll
  for (int s = 0; s < kHalvings; ++s) {
    const int o = (kN >= 32 ? 16 : 8) >> s, n = kN >> (s + 1);
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int j = 0; j < n; ++j) {
      const float send = up ? v[j] : v[j + n], keep = up ? v[j + n] : v[j];
      v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  if (kN == 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 16);
}
// Column of v[j] after warp_sum_columns: the lane's bits choose the halves.
template <int kN>
__device__ __forceinline__ int column_of(int lane, int j) {
  int col = j;
  constexpr int kHalvings = kN >= 32 ? 5 : 4;
#pragma unroll
  for (int s = 0; s < kHalvings; ++s)
    if (lane & ((kN >= 32 ? 16 : 8) >> s)) col += kN >> (s + 1);
  return col;
}

template <int kD, int kN>
__global__ void __launch_bounds__(AT_THREADS, 1)
    attn_fp8_tc_kernel(const AttnTcArgs t, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
  using Shape = AttnTcShape<kD, kN>;
  constexpr int kStages = Shape::kStages;
  constexpr uint32_t kSwz = kD == 128 ? 2u : 4u;       // layout of K, V and q tiles
  constexpr uint32_t kAtom = kD == 128 ? 1024u : 512u;  // bytes of 8 rows
  const AttnArgs& a = t.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.Hkv, rows = a.Sq * G;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem + Shape::kOffQ;
  uint8_t* s_p = smem + Shape::kOffP;
  // the small arrays
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Shape::kOffMisc);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = bars + AT_MAX_STAGES;
  uint64_t* s_full = bars + 2 * AT_MAX_STAGES;   // [kScores]
  uint64_t* p_full = s_full + 4;                 // [2]
  uint64_t* pv_done = s_full + 6;                // [2]
  uint64_t* q_full = s_full + 8;
  uint64_t* drained = s_full + 9;
  float2* s_sc = reinterpret_cast<float2*>(bars + 2 * AT_MAX_STAGES + 10);  // [stages][8] scales of K, V
  int* s_bad = reinterpret_cast<int*>(s_sc + AT_MAX_STAGES * AT_MAX_PAGES);  // [stages] some page invalid
  int* s_lo = s_bad + AT_MAX_STAGES;             // [N] first and last key that a column sees
  int* s_hi = s_lo + kN;
  float* s_qf = reinterpret_cast<float*>(s_hi + kN);  // [N] score factor of a column
  int* s_row = reinterpret_cast<int*>(s_qf + kN);  // [N] row of the output, from the unit's first
  float* s_m = reinterpret_cast<float*>(s_row + kN);                        // [2][N] reference of p, log2
  float* s_M = s_m + 2 * kN;                     // [2][N] reference of O, log2
  float* s_c = s_M + 2 * kN;                     // [2][N] 2^(m - M)
  float* s_f = s_c + 2 * kN;                     // [2][N] factor of a rescale; sums at the end
  float* s_red = s_f + 2 * kN;                   // [2][4][2][N] warp maxima, warp sums
  uint32_t* s_nan = reinterpret_cast<uint32_t*>(s_red + 16 * kN);  // [D][2] columns that see a NaN value
  int* s_ctl = reinterpret_cast<int*>(s_nan + 2 * kD);  // abort, tmem, last, b, prefix (2 words)
  volatile int* s_abort = s_ctl;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_ctl + 1);
  static_assert(8 * (2 * AT_MAX_STAGES + 10) + 8 * AT_MAX_STAGES * AT_MAX_PAGES + 4 * AT_MAX_STAGES +
                        4 * (4 * kN + 8 * kN + 16 * kN) + 8 * kD + 64 <=
                    Shape::kMiscBytes,
                "small arrays");

  // ---- set-up, spread over the warps; the producer does not wait for it ----
  if (warp == 0) {
    if (lane == 0) {
      *s_abort = 0;
      for (int i = 0; i < kStages; ++i) {
        mbar_init(kv_full + i, 1);
        mbar_init(kv_empty + i, 1);
      }
      for (int i = 0; i < Shape::kScores; ++i) mbar_init(s_full + i, 1);
      for (int w = 0; w < 2; ++w) {
        mbar_init(p_full + w, 4);
        mbar_init(pv_done + w, 1);
      }
      mbar_init(q_full, 8);
      mbar_init(drained, 1);
      fence_mbar_init();
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(s_tmem, Shape::kTmem);
    tmem_relinquish();
    tc_fence_before();
  }
  // ---- this CTA's share, found by every warp for itself ----
  AttnWalk walk;
  AttnShares shares;
  {
    const int per = (a.B + 31) / 32;  // sequences of a lane, in order
    const int b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B);
    auto tiles_of = [&](int b) {
      const int len = __ldg(a.seq_lens + b);
      int n = 0;
      for (int c = 0; c < t.chunks; ++c) {
        int lo, hi, k;
        attn_unit(t, len, G, rows, kN, c, &lo, &hi, &k);
        n += k;
      }
      return n * a.Hkv;
    };
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(b);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    const int ctas = min((int)gridDim.x, max(1, total / t.min_tiles));
    shares.each = total / ctas;
    shares.more = total - shares.each * ctas;
    const bool idle = (int)blockIdx.x >= ctas;  // the whole CTA: it has no tiles
    walk.pos = idle ? 0 : shares.first(blockIdx.x);
    walk.end = idle ? 0 : shares.first(blockIdx.x + 1);
    int at = incl - mine, b = b0;
    const uint32_t owner = __ballot_sync(0xffffffffu, walk.pos >= at && walk.pos < at + mine);
    if (walk.pos >= at && walk.pos < at + mine) {
      for (int n; b < b1 && walk.pos >= at + (n = tiles_of(b)); ++b) at += n;
    }
    walk.b = __shfl_sync(0xffffffffu, b, __ffs(owner) - 1);
    walk.unit = __shfl_sync(0xffffffffu, at, __ffs(owner) - 1);
    walk.h = walk.c = 0;
    walk.len = __ldg(a.seq_lens + walk.b);
    walk_unit<kN>(t, G, rows, walk);
    while (walk.unit + walk.tiles <= walk.pos) walk_next<kN>(t, G, rows, walk);
  }
  uint32_t tmem = 0;
  if (warp == 0) {
    named_barrier_arrive(4, AT_THREADS);
  } else {
    named_barrier_sync(4, AT_THREADS);
    tc_fence_after();
    tmem = *s_tmem;
  }

  // Bounded wait; once one gave up, none waits and nothing more is issued, but
  // every role still runs its loop to the end, so no barrier is left short.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t it = 1;; ++it) {
      if (mbar_try_wait(bar, parity)) return true;
      if ((it & 31u) == 0) {
        if (*s_abort) return false;
        if (globaltimer_ns() - t0 > WD_WAIT_LIMIT_NS) {
          *s_abort = 1;
          raise_status(a.status, WD_STATUS_WAIT_TIMEOUT);
          return false;
        }
      }
    }
  };

  if (warp == 0) {
    // ---- producer: pages of K and V, and their scales --------------------
    const int per_tile = AT_TILE >> t.page_shift;
    const uint64_t policy = l2_policy_evict_first();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    while (walk.pos < walk.end) {
      const int first = walk.kmin / AT_TILE + walk.pos - walk.unit;  // key tile of the piece's start
      const int n = min(walk.unit + walk.tiles, walk.end) - walk.pos;
      // columns of the table that the piece needs, 32 at a time, one batch ahead
      const int c_lo = max(first * per_tile, walk.kmin >> t.page_shift);
      const int c_hi = walk.kmax < walk.kmin ? -1 : min((first + n) * per_tile - 1, walk.kmax >> t.page_shift);
      const int32_t* table = a.table + (size_t)walk.b * a.table_stride;
      if (walk.len > t.reach && lane == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
      auto page_at = [&](int col) {
        int pid = -1;
        if (col >= c_lo && col <= c_hi && col < a.table_stride) pid = __ldg(table + col);
        return pid >= 0 && pid < a.pages ? pid : -1;
      };
      int batch = first * per_tile, used = 0;
      int pid = page_at(batch + lane), pid_next = page_at(batch + 32 + lane);
      uint32_t kb = 0, vb = 0;
      if (pid >= 0) {
        kb = __ldg(a.ks + (size_t)pid * a.Hkv + walk.h);
        vb = __ldg(a.vs + (size_t)pid * a.Hkv + walk.h);
      }
      for (int j = 0; j < n; ++j) {
        if (used == 32) {
          used = 0;
          batch += 32;
          pid = pid_next;
          kb = vb = 0;
          if (pid >= 0) {
            kb = __ldg(a.ks + (size_t)pid * a.Hkv + walk.h);
            vb = __ldg(a.vs + (size_t)pid * a.Hkv + walk.h);
          }
          pid_next = page_at(batch + 32 + lane);
        }
        const int col = batch + lane;
        const bool mine = lane >= used && lane < used + per_tile;
        const bool needed = mine && col >= c_lo && col <= c_hi;
        const bool good = needed && pid >= 0;
        const uint32_t bad = __ballot_sync(0xffffffffu, needed && pid < 0);
        const uint32_t loads = __popc(__ballot_sync(0xffffffffu, good));
        if (bad && lane == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
        const bool free = wait(kv_empty + stage, phase ^ 1u);
        if (__all_sync(0xffffffffu, free)) {
          if (lane == 0) mbar_expect_tx(kv_full + stage, loads * 2u * (uint32_t)(a.page * kD));
          __syncwarp();
          uint8_t* dst = smem + stage * 2 * Shape::kKvBytes;
          if (good) {
            const int row = (pid * a.Hkv + walk.h) * a.page, off = (lane - used) * a.page * kD;
            tma_load_2d(dst + off, &tm_k, 0, row, kv_full + stage, policy);
            tma_load_2d(dst + Shape::kKvBytes + off, &tm_v, 0, row, kv_full + stage, policy);
          }
          if (mine)
            s_sc[stage * AT_MAX_PAGES + lane - used] =
                good ? make_float2(ue8m0_to_f32(kb), ue8m0_to_f32(vb)) : make_float2(-1.f, 0.f);
          if (lane == 0) s_bad[stage] = bad != 0u;
          __syncwarp();
          if (lane == 0) mbar_arrive(kv_full + stage);
          ++issued;
        }
        used += per_tile;
        if (++stage == kStages) stage = 0, phase ^= 1u;
      }
      walk.pos += n;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0) {
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_wait(kv_full + i % kStages, (uint32_t)(i / kStages) & 1u);
    }
  } else if (warp == 1) {
    // ---- MMA issuer ------------------------------------------------------
    constexpr uint32_t kIdQK = tc_idesc_e4m3(AT_TILE, 2 * kN, false, false);
    constexpr uint32_t kIdPV = tc_idesc_e4m3(128, 2 * kN, true, true);
    // Descriptors of the first stage and buffer; the others are at a distance.
    const uint64_t d_k = tc_desc(smem_u32(smem), 16, kAtom, kSwz);
    const uint64_t d_v = tc_desc(smem_u32(smem) + Shape::kKvBytes, 0, kAtom, kSwz);
    const uint64_t d_q = tc_desc(smem_u32(s_q), 16, kAtom, kSwz);
    const uint64_t d_p = tc_desc(smem_u32(s_p), 128, 2048, 0);
    int stage = 0;
    uint32_t phase = 0, q_phase = 0, p_phase[2] = {0, 0};
    auto next_stage = [&](int& s, uint32_t& ph) {
      if (++s == kStages) s = 0, ph ^= 1u;
    };
    while (walk.pos < walk.end) {
      const int n = min(walk.unit + walk.tiles, walk.end) - walk.pos;
      const bool q_in = wait(q_full, q_phase);
      q_phase ^= 1u;
      int st = stage;  // stage of the next QK
      uint32_t ph = phase;
      auto qk = [&](int j) {
        const bool in = wait(kv_full + st, ph);
        tc_fence_after();
        if (__all_sync(0xffffffffu, in && q_in) && elect_one()) {
          const uint64_t k = d_k + (uint32_t)(st * 2 * Shape::kKvBytes / 16);
#pragma unroll
          for (int s = 0; s < kD / 32; ++s)
            tc_mma_f8(tmem + j % Shape::kScores * 2 * kN, k + 2 * s, d_q + 2 * s, kIdQK, s > 0);
          tc_commit(s_full + j % Shape::kScores);
        }
        __syncwarp();
        next_stage(st, ph);
      };
      // the scores of tile j + kScores - 1 replace those of tile j - 1, which
      // have been read when its p is there
      for (int j = 0; j < min(n, Shape::kScores - 1); ++j) qk(j);
      for (int j = 0; j < n; ++j) {
        const int w = j & 1;
        if (j + Shape::kScores - 1 < n) qk(j + Shape::kScores - 1);
        const bool in = wait(p_full + w, p_phase[w]);
        p_phase[w] ^= 1u;
        tc_fence_after();
        if (__all_sync(0xffffffffu, in) && elect_one()) {
          const uint64_t v = d_v + (uint32_t)(stage * 2 * Shape::kKvBytes / 16);
          const uint64_t p = d_p + (uint32_t)(w * 2 * Shape::kPBytes / 16);
#pragma unroll
          for (int s = 0; s < AT_TILE / 32; ++s)
            tc_mma_f8(tmem + (Shape::kScores + w) * 2 * kN, v + s * 2 * kD, p + s * 32, kIdPV, j >= 2 || s > 0);
          tc_commit(kv_empty + stage);
          tc_commit(pv_done + w);
        }
        __syncwarp();
        next_stage(stage, phase);
      }
      walk.pos += n;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
    // After an abort let what was issued end before TMEM is freed.
    __syncwarp();
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained);
      mbar_wait(drained, 0);
    }
    __syncwarp();
  } else {
    // ---- softmax warpgroups ----------------------------------------------
    const int wg = (warp - 2) >> 2;
    const int quarter = warp & 3;              // TMEM lanes of this warp
    const int row = quarter * 32 + lane;       // key of the tile; value index d of O
    const int wtid = tid - 64;                 // of both warpgroups
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21);
    const uint32_t t_o = lanes + (Shape::kScores + wg) * 2 * kN;
    uint8_t* my_p = s_p + wg * 2 * Shape::kPBytes;
    float* my_m = s_m + wg * kN;
    float* my_M = s_M + wg * kN;
    float* my_c = s_c + wg * kN;
    float* my_f = s_f + wg * kN;
    float* my_red = s_red + wg * 8 * kN;
    constexpr int kPerLane = (AT_MAX_CTAS + 31) / 32;
    static_assert(2 * Shape::kQBytes + 4 * Shape::kPBytes >= AT_MAX_CTAS * kN * 4 && 4 * AT_MAX_CTAS <= AT_COUNTERS,
                  "room for a factor per piece and column");
    constexpr float kNone = -1e30f;  // no reference yet: any weight lies beyond it
    int stage = 0;
    uint32_t phase = 0, s_phase = 0, pv_phase = 0;
    while (walk.pos < walk.end) {
      const int first = walk.kmin / AT_TILE + walk.pos - walk.unit;
      const int n = min(walk.unit + walk.tiles, walk.end) - walk.pos;
      const int r0 = walk.c * kN, live = min(kN, rows - r0);  // columns in use
      // q of the unit as two E4M3 terms: a warp per row
      for (int r = warp - 2; r < kN; r += 8) {
        constexpr int kPer = kD / 32;
        float x[kPer];
        uint32_t most = 0u;
        const int i = (r0 + r) / G, head = walk.h * G + (r0 + r) % G;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          x[e] = 0.f;
          if (r < live) {
            x[e] = __bfloat162float(a.q[(long long)walk.b * a.q_bs + (long long)i * a.q_ts +
                                        (long long)head * a.q_hs + lane * kPer + e]);
            const uint32_t u = __float_as_uint(x[e]) & 0x7fffffffu;
            if (u < 0x7f800000u)
              most = max(most, u);
            else
              x[e] = __uint_as_float(0x7fc00000u);  // an infinite q makes its whole row NaN
          }
        }
        most = __reduce_max_sync(0xffffffffu, most);
        const int byte = scale_byte(most);
        const float inv = exp2_int(127 - byte);
        uint32_t hi = 0u, lo = 0u;
#pragma unroll
        for (int e = 0; e < kPer; e += 2) {
          const float u = x[e] * inv, v = x[e + 1] * inv;
          const uint32_t h2 = __nv_cvt_float2_to_fp8x2(make_float2(u, v), __NV_SATFINITE, __NV_E4M3);
          const float2 back = e4m3x2_to_f32(h2);
          const uint32_t l2 =
              __nv_cvt_float2_to_fp8x2(make_float2(u - back.x, v - back.y), __NV_SATFINITE, __NV_E4M3);
          hi |= h2 << (8 * e);
          lo |= l2 << (8 * e);
        }
        const int d = lane * kPer;
        const int sw = kD == 128 ? (r & 7) : ((r >> 1) & 3);
        const int off = r * kD + (((d >> 4) ^ sw) << 4) + (d & 15);
        if constexpr (kPer == 4) {
          *reinterpret_cast<uint32_t*>(s_q + off) = hi;
          *reinterpret_cast<uint32_t*>(s_q + Shape::kQBytes + off) = lo;
        } else {
          *reinterpret_cast<uint16_t*>(s_q + off) = (uint16_t)hi;
          *reinterpret_cast<uint16_t*>(s_q + Shape::kQBytes + off) = (uint16_t)lo;
        }
        if (lane == 0) {
          const int rr = min(r, live - 1);  // columns past the rows: like the last row
          const int last = walk.len - a.Sq + (r0 + rr) / G;
          s_hi[r] = last;
          s_lo[r] = a.window > 0 ? max(0, last - a.window + 1) : 0;
          s_qf[r] = exp2_int(byte - 127) * a.scale_log2;
          s_row[r] = (r0 + rr) / G * a.Hq + (r0 + rr) % G;
        }
      }
      for (int i = wtid; i < 2 * kN; i += 256) {
        s_m[i] = kNone;
        s_M[i] = kNone;
        s_c[i] = 0.f;
      }
      for (int i = wtid; i < 2 * kD; i += 256) s_nan[i] = 0u;
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      named_barrier_sync(3, 256);

      const int lo_min = s_lo[0], lo_max = s_lo[live - 1];  // rows are in token order
      const int hi_min = s_hi[0], hi_max = s_hi[live - 1];
      float l[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) l[i] = 0.f;
      int st = stage + wg;
      uint32_t ph = phase;
      if (st >= kStages) st -= kStages, ph ^= 1u;
      bool any_pv = false;
      for (int j = wg; j < n; j += 2) {
        const int key = (first + j) * AT_TILE + row;
        const int sb = j % Shape::kScores;
        const uint32_t t_s = lanes + sb * 2 * kN;
        wait(s_full + sb, (s_phase >> sb) & 1u);
        s_phase ^= 1u << sb;
        tc_fence_after();
        wait(kv_full + st, ph);  // completed long ago: makes the scales visible here
        const float2 sc = s_sc[st * AT_MAX_PAGES + (row >> t.page_shift)];
        const int tile0 = (first + j) * AT_TILE;
        const bool whole = tile0 >= lo_max && tile0 + AT_TILE - 1 <= hi_min && s_bad[st] == 0;
        float vf = sc.y;
        bool page_ok = true;
        if (!whole) {
          page_ok = !(sc.x < 0.f);
          uint8_t* v = smem + st * 2 * Shape::kKvBytes + Shape::kKvBytes + row * kD;
          if (key < lo_min || key > hi_max || !page_ok) {
            // what lies here is nobody's: it must not reach the product as NaN
            vf = 0.f;
#pragma unroll
            for (int i = 0; i < kD / 16; ++i) reinterpret_cast<uint4*>(v)[i] = make_uint4(0u, 0u, 0u, 0u);
          } else if (key < lo_max || key > hi_min) {
            // seen by some columns only: NaN values are taken out and noted
            // for those columns, for 0 times NaN would reach the others
            const int sw = kD == 128 ? (row & 7) : ((row >> 1) & 3);
            const bool all = vf != vf;
            if (all) vf = 0.f;
            uint32_t* words = reinterpret_cast<uint32_t*>(v);
            for (int i = 0; i < kD / 4; ++i) {
              const uint32_t word = words[i];
              if (!all && (((word & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) == 0u) continue;
              uint32_t clean = word;
              for (int e = 0; e < 4; ++e) {
                if (!all && ((word >> (8 * e)) & 0x7fu) != 0x7fu) continue;
                clean &= ~(0xffu << (8 * e));
                const int d = (((i >> 2) ^ sw) << 4) + (i & 3) * 4 + e;
                for (int c = 0; c < live; ++c)
                  if (key >= s_lo[c] && key <= s_hi[c]) atomicOr(s_nan + 2 * d + (c >> 5), 1u << (c & 31));
              }
              words[i] = clean;
            }
          }
        }
        const float kf = sc.x;
        // the tile's scores as exponents of 2, less `ref` of their column
        auto weights = [&](float (&x)[kN], auto ref) {
#pragma unroll
          for (int cb = 0; cb < kN / 16; ++cb) {
            uint32_t v[16], v_lo[16];
            tmem_ld_x16(t_s + cb * 16, v);
            tmem_ld_x16(t_s + kN + cb * 16, v_lo);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + __uint_as_float(v_lo[i]));
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const float4 qf = *reinterpret_cast<const float4*>(s_qf + cb * 16 + i);
              const float4 m = ref(cb * 16 + i);
              x[cb * 16 + i] = fmaf(__uint_as_float(v[i]) * kf, qf.x, -m.x);
              x[cb * 16 + i + 1] = fmaf(__uint_as_float(v[i + 1]) * kf, qf.y, -m.y);
              x[cb * 16 + i + 2] = fmaf(__uint_as_float(v[i + 2]) * kf, qf.z, -m.z);
              x[cb * 16 + i + 3] = fmaf(__uint_as_float(v[i + 3]) * kf, qf.w, -m.w);
            }
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < kN; ++i)
              if (!page_ok || key < s_lo[i] || key > s_hi[i]) x[i] = -INFINITY;
          }
        };
        auto reference = [&](int i) { return *reinterpret_cast<const float4*>(my_m + i); };
        float x[kN];
        weights(x, reference);
        // does some weight leave the range that the references allow?
        float over = 0.f;
#pragma unroll
        for (int i = 0; i < kN; i += 4) {
          const float4 c = *reinterpret_cast<const float4*>(my_c + i);
          const float cc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[i + e] = ex2_approx(x[i + e]);
            over = fmaxf(over, fmaxf(x[i + e] * 28.f, x[i + e] * cc[e] * vf));
          }
        }
        if (named_barrier_any(1 + wg, 128, over > 448.f)) {
          // new references: the columns' maxima of x and of x + log2(scale of V)
          weights(x, [](int) { return make_float4(0.f, 0.f, 0.f, 0.f); });
          const float lv = __log2f(vf);
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            const float xm = warp_max_f32(x[i]), tm = warp_max_f32(x[i] + lv);
            if (lane == 0) {
              my_red[quarter * 2 * kN + i] = xm;
              my_red[quarter * 2 * kN + kN + i] = tm;
            }
          }
          named_barrier_sync(1 + wg, 128);
          if (row < kN) {
            float xm = my_red[row], tm = my_red[kN + row];
#pragma unroll
            for (int w = 1; w < 4; ++w) {
              xm = fmaxf(xm, my_red[w * 2 * kN + row]);
              tm = fmaxf(tm, my_red[w * 2 * kN + kN + row]);
            }
            const float m0 = my_m[row], M0 = my_M[row];
            const float m1 = fmaxf(m0, xm);
            // O's reference lies AT_HEAD below the largest, and at most 2^120 below that of p
            const float M1 = fmaxf(M0, fmaxf(tm - AT_HEAD, m1 - 120.f));
            my_f[row] = ex2_approx(m0 - m1);    // of the sums
            my_red[row] = ex2_approx(M0 - M1);  // of O
            my_m[row] = m1;
            my_M[row] = M1;
            my_c[row] = ex2_approx(m1 - M1);
          }
          named_barrier_sync(1 + wg, 128);
#pragma unroll
          for (int i = 0; i < kN; ++i) l[i] *= my_f[i];
          if (any_pv) {
            wait(pv_done + wg, pv_phase);
            tc_fence_after();
#pragma unroll
            for (int cb = 0; cb < 2 * kN / 16; ++cb) {
              uint32_t v[16];
              tmem_ld_x16(t_o + cb * 16, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                v[i] = __float_as_uint(__uint_as_float(v[i]) * my_red[cb * 16 % kN + i]);
              tmem_st_x16(t_o + cb * 16, v);
            }
            tmem_wait_st();
          }
          weights(x, reference);
#pragma unroll
          for (int i = 0; i < kN; ++i) x[i] = ex2_approx(x[i]);
        }
        tc_fence_before();
        if (any_pv) {  // p of the previous tile has been read
          wait(pv_done + wg, pv_phase);
          pv_phase ^= 1u;
        }
        any_pv = true;
#pragma unroll
        for (int cb = 0; cb < kN / 16; ++cb) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 c = *reinterpret_cast<const float2*>(my_c + cb * 16 + i);
            float s[2], r[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              l[cb * 16 + i + e] += x[cb * 16 + i + e];
              const float p = x[cb * 16 + i + e] * (e ? c.y : c.x) * vf;
              // the nearest value of four significant bits
              s[e] = __uint_as_float((__float_as_uint(p) + 0x00080000u) & 0xfff00000u);
              r[e] = p - s[e];
            }
            const uint32_t h2 = __nv_cvt_float2_to_fp8x2(make_float2(s[0], s[1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t l2 = __nv_cvt_float2_to_fp8x2(make_float2(r[0], r[1]), __NV_SATFINITE, __NV_E4M3);
            if (i % 4 == 0) {
              hi[i / 4] = h2;
              lo[i / 4] = l2;
            } else {
              hi[i / 4] |= h2 << 16;
              lo[i / 4] |= l2 << 16;
            }
          }
          *reinterpret_cast<uint4*>(my_p + cb * 2048 + row * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(my_p + Shape::kPBytes + cb * 2048 + row * 16) =
              make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + wg);
        st += 2;
        if (st >= kStages) st -= kStages, ph ^= 1u;
      }
      stage += n % kStages;
      phase ^= (uint32_t)(n / kStages) & 1u;
      if (stage >= kStages) stage -= kStages, phase ^= 1u;

      // ---- the piece's end: sums over the keys, then both warpgroups join --
      if (any_pv) {
        wait(pv_done + wg, pv_phase);
        pv_phase ^= 1u;
        tc_fence_after();
      }
      warp_sum_columns<kN>(l, lane);
#pragma unroll
      for (int i = 0; i < (kN + 31) / 32; ++i) my_red[quarter * kN + column_of<kN>(lane, i)] = l[i];
      constexpr int kHalf = kN / 2;
      float o[kHalf];
      // columns [wg * N/2, ...) are finished here, the others by the other warpgroup
      float* give = reinterpret_cast<float*>(my_p);  // [N/2][128]
      const float* take = reinterpret_cast<const float*>(s_p + (1 - wg) * 2 * Shape::kPBytes);
#pragma unroll
      for (int cb = 0; cb < kN / 8; ++cb) {
        uint32_t v[8], v_lo[8];
        if (any_pv) {
          tmem_ld_x8(t_o + cb * 8, v);
          tmem_ld_x8(t_o + kN + cb * 8, v_lo);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = v_lo[i] = 0u;
        }
        const bool keep = (cb * 8 >= kHalf) == (wg == 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int col = (cb * 8 + i) % kHalf;
          const float y = __uint_as_float(v[i]) + __uint_as_float(v_lo[i]);
          if (keep)
            o[col] = y;
          else
            give[col * 128 + row] = y;
        }
      }
      tc_fence_before();
      named_barrier_sync(3, 256);
      const int u0 = walk.unit, u1 = walk.unit + walk.tiles;
      const bool split = walk.pos > u0 || walk.pos + n < u1;
      float* slot = t.slots + (size_t)(2 * blockIdx.x + (walk.pos > shares.first(blockIdx.x) ? 1 : 0)) *
                                  Shape::kSlotFloats;
      const size_t out0 = (size_t)walk.b * a.Sq * a.Hq + walk.h * G;  // output row of the unit's first
      // a thread per column: its statistics, and the factors of both O
      if (wtid < kN) {
        const float m0 = s_m[wtid], m1 = s_m[kN + wtid], M0 = s_M[wtid], M1 = s_M[kN + wtid];
        const float m = fmaxf(m0, m1), M = fmaxf(M0, M1);
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l0 += s_red[w * kN + wtid], l1 += s_red[8 * kN + w * kN + wtid];
        const float sum = l0 * ex2_approx(m0 - m) + l1 * ex2_approx(m1 - m);
        float f = 1.f;
        if (split) {
          __stcg(slot + kN * kD + wtid, sum);
          __stcg(slot + kN * kD + kN + wtid, m);
          __stcg(slot + kN * kD + 2 * kN + wtid, M);
        } else {
          f = sum == 0.f ? 0.f : ex2_approx(M - m) / sum;
          if (a.lse && wtid < live)
            a.lse[out0 + s_row[wtid]] = sum == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(sum);
        }
        s_f[wtid] = f * ex2_approx(M0 - M);
        s_f[kN + wtid] = f * ex2_approx(M1 - M);
      }
      named_barrier_sync(3, 256);
      if (row < kD) {
        const uint64_t poison = (uint64_t)s_nan[2 * row] | (uint64_t)s_nan[2 * row + 1] << 32;
        const float* f_mine = s_f + wg * kN + wg * kHalf;
        const float* f_take = s_f + (1 - wg) * kN + wg * kHalf;
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
          const int col = wg * kHalf + i;
          if (col >= live) break;
          float y = o[i] * f_mine[i] + take[i * 128 + row] * f_take[i];
          if ((poison >> col) & 1ull) y = __uint_as_float(0x7fc00000u);
          if (split)
            __stcg(slot + col * kD + row, y);
          else
            a.out[(out0 + s_row[col]) * kD + row] = __float2bfloat16_rn(y);
        }
      }
      if (split) {
        const int ca = shares.cta_of(u0), cz = shares.cta_of(u1 - 1);
        const int pieces = cz - ca + 1;
        __threadfence();
        named_barrier_sync(3, 256);
        if (wtid == 0) {
          const uint32_t before = atomicAdd(t.counters + ca, 1u);
          const int last = before + 1 == (uint32_t)pieces;
          if (last) t.counters[ca] = 0u;  // nobody else touches it in this call any more
          s_ctl[2] = last;
        }
        named_barrier_sync(3, 256);
        if (s_ctl[2]) {
          __threadfence();
          auto slot_of = [&](int c) {
            return t.slots + (size_t)(2 * c + (shares.first(c) < u0 ? 1 : 0)) * Shape::kSlotFloats;
          };
          // a warp per column: the pieces' common references and their factors,
          // kept where q and p lay
          float* factor = reinterpret_cast<float*>(s_q);  // [pieces][N]
          float* norm = s_f;                              // [N]
          for (int col = warp - 2; col < live; col += 8) {
            float m[kPerLane], M[kPerLane], ls[kPerLane], m_all = kNone, M_all = kNone;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
              const int p = lane + 32 * i;
              m[i] = M[i] = kNone;
              ls[i] = 0.f;
              if (p < pieces) {
                const float* s = slot_of(ca + p) + kN * kD + col;
                ls[i] = __ldcg(s);
                m[i] = __ldcg(s + kN);
                M[i] = __ldcg(s + 2 * kN);
              }
            }
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) m_all = fmaxf(m_all, m[i]), M_all = fmaxf(M_all, M[i]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
              m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
              M_all = fmaxf(M_all, __shfl_xor_sync(0xffffffffu, M_all, o));
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
              sum += ls[i] * ex2_approx(m[i] - m_all);
              if (lane + 32 * i < pieces) factor[(lane + 32 * i) * kN + col] = ex2_approx(M[i] - M_all);
            }
            sum = warp_sum(sum);
            if (lane == 0) {
              norm[col] = sum == 0.f ? 0.f : ex2_approx(M_all - m_all) / sum;
              if (a.lse)
                a.lse[out0 + s_row[col]] = sum == 0.f ? -INFINITY : m_all * 0.6931471805599453f + logf(sum);
            }
          }
          named_barrier_sync(3, 256);
          // four values of a column a thread, the pieces in order
          for (int e = wtid; e < live * (kD / 4); e += 256) {
            const int col = e / (kD / 4), d = (e % (kD / 4)) * 4;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
            for (int p = 0; p < pieces; ++p) {
              const float4 v = __ldcg(reinterpret_cast<const float4*>(slot_of(ca + p) + col * kD + d));
              const float f = factor[p * kN + col];
              y.x = fmaf(v.x, f, y.x), y.y = fmaf(v.y, f, y.y), y.z = fmaf(v.z, f, y.z), y.w = fmaf(v.w, f, y.w);
            }
            const float f = norm[col];
            *reinterpret_cast<uint2*>(a.out + (out0 + s_row[col]) * kD + d) =
                make_uint2(pack_bf16(y.x * f, y.y * f), pack_bf16(y.z * f, y.w * f));
          }
        }
      }
      named_barrier_sync(3, 256);  // q, p and the statistics may be written again
      walk.pos += n;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, Shape::kTmem);
}

}  // namespace wdb

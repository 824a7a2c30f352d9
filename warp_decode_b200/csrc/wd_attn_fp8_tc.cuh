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
//   lo = the nearest to 16 times what remains: q (8 significant bits) is exact
//   over fourteen octaves below the row's largest value, p is within 2^-9, or
//   within 2^-16 of the column's largest (with V's scale).  There the rounding
//   is without bias over the keys, so what thousands of keys weigh together,
//   each below the quantum, is kept (AT_GOLDEN).  The terms are columns side by
//   side of one product (2 N columns; a small product's time goes by its A
//   operand), joined where they are read; no code is ever widened.
// * Scales are powers of two: the page scale of K goes into the exponent's
//   factor, that of V multiplies p before it is rounded.
// * Running maxima are lazy.  p = 2^(x - M) is taken relative to a reference M
//   of its column that only moves when some p times V's scale would pass
//   E4M3's 448 (or 2^90 itself), found by a vote of the tile's threads; sums and
//   O (in TMEM) are then rescaled.  A piece's first tile sets the references;
//   after that a move is rare, and the common tile has no cross-thread maximum.
//   M is set AT_HEAD below the column's largest x + log2(V's scale), so weights
//   keep their precision whatever the magnitudes of the pages' values.
//
// Work: all (sequence, key head, row chunk) units' key tiles in one line, each
// unit with a few tiles' worth of its fixed cost added, cut into equal shares,
// one per CTA (whatever the lengths, the SMs end together).  A CTA runs its
// share as pieces of units: a producer warp loads pages, one warp stages q, one
// issues the products of scores, one those of values, and two softmax
// warpgroups take the CTA's tiles alternately, each with its own statistics and
// O, and join at a piece's end (a whole unit of one tile is one warpgroup's
// alone, so two such units run at once); q, pages and scores of the next pieces
// come in meanwhile.  Pieces of a unit that several CTAs share go through the
// workspace: each CTA but the last of them ends its share there, waits for the
// others (one cooperative launch, a bounded wait) and joins an equal part of
// the unit's values, in CTA order.
//
// Measured (B200): 64 sequences of up to 8192 tokens, 4 key heads of 8 rows, D
// 128, pages of 64 (307 MB) 58 us, 5.3 TB/s; one of 131072 (134 MB) 30 us; 16
// of 8000 with 32 rows a head (131 MB) 42 us, there held by the softmax's
// latency: two warps a scheduler, issue at a third.
#pragma once

#include "wd_attn_fp8.cuh"
#include "wd_tc.cuh"

namespace wdb {

constexpr int AT_TILE = 128;       // keys of a tile
constexpr int AT_THREADS = 384;    // producer, two MMA issuers, q, two warpgroups of four warps
constexpr int AT_MAX_PAGES = 8;    // pages of a tile (16 tokens each)
constexpr int AT_MAX_STAGES = 12;
// log2 of the E4M3 value that the largest p is stored as when references are
// set: 56 x room to grow before they move again (a move costs as much as a tile;
// with 7 x a long row took several), the second term's quantum 2^-13 at 2^-16.
constexpr float AT_HEAD = 3.f;
constexpr float AT_LO = 1.f / 16;  // what a second term counts
// lo's rounding is moved by up to half its quantum 2^-9, by the fraction of key *
// golden ratio, which fills the interval evenly over any regular set of keys: a
// weight below the quantum becomes the quantum for its share of keys, and one of
// 0 stays 0.  Rounded to nearest, a tail of 65536 keys at 2^-20 of the largest
// weight each was lost (half of 0.045 of the output, the half that shared the
// strong key's reference), at the same speed.
constexpr uint32_t AT_GOLDEN = 0x9E3779B1u;
constexpr float AT_SHIFT = 0x1p-41f;  // 2^-32 of the fraction, 2^-9 of the quantum
constexpr float AT_FULL = 8.8f;    // log2 448, rounded down
constexpr float AT_FAR = 90.f;     // log2 of the largest p itself
constexpr float AT_NONE = -1e30f;  // no reference yet: any weight lies beyond it
constexpr int AT_MAX_CTAS = 160;
// Named barriers: 1 and 2 a warpgroup's, 3 both, 4 the set-up, 5 the first
// piece's q, 6 and 7 a split piece written (at the start and at the end of the
// share: the softmax warps may come to the second before the q warp has left
// the first).
constexpr int AT_BAR_SPLIT = 6;
constexpr int AT_COUNTERS = 2048;  // bytes of counters at the workspace's start, two of 4 per CTA

template <int kD, int kN>
struct AttnTcShape {
  static constexpr int kKvBytes = AT_TILE * kD;              // K or V of a tile
  static constexpr int kQBytes = kN * kD;                    // one term of q
  static constexpr int kPBytes = AT_TILE * kN;               // one term of p
  // Score tiles in TMEM: with four, the product of a warpgroup's next tile is
  // done while it still works on this one (512 columns hold two at N = 64).
  static constexpr int kScores = kN == 64 ? 2 : 4;
  static constexpr int kTmem = kN == 16 ? 256 : 512;  // columns: scores and both O, 2 N each
  static constexpr int kStages = kD == 64 ? (kN == 64 ? 9 : 10) : (kN == 64 ? 4 : kN == 32 ? 5 : 6);
  static constexpr int kOffQ = kStages * 2 * kKvBytes;
  static constexpr int kOffP = kOffQ + 4 * kQBytes;          // two q, each of two terms
  static constexpr int kMiscBytes = kN == 64 ? 11776 : 7424;
  static constexpr int kOffMisc = kOffP + 4 * kPBytes;       // two p, each of two terms
  static constexpr int kSmem = kOffMisc + kMiscBytes + 1024;  // + alignment slack
  // What is left of a split piece in the workspace: by each warpgroup (both
  // joined at N = 64, for its size) O [N][D], sums of its warps [N][4],
  // references [N].
  static constexpr int kSlotFloats = kN * kD + 5 * kN;
  static constexpr int kSlots = kN == 64 ? 1 : 2;
};

struct AttnTcArgs {
  AttnArgs a;
  uint32_t* counters;  // per CTA: pieces that came, joiners that went; zero between calls
  float* slots;        // two pieces per CTA
  int chunks;          // row chunks of a (sequence, key head)
  int min_share;       // least share of a CTA, in tiles
  int unit_cost;       // a unit's fixed cost, in tiles
  int reach;           // tokens that the block table can address
  int q_wide;          // q's rows are 16-byte aligned
  int page_shift;
};

constexpr int AT_JOIN_FLOATS = 6;  // of a thread that joins: reference, sum, four values

// Keys [kmin, kmax] that the rows of chunk c see, as far as the table reaches,
// and their tiles; none: one tile, all masked.
__device__ __forceinline__ void attn_unit(const AttnTcArgs& t, int len, int G, int rows, int kN, int c,
                                          int* kmin, int* kmax, int* tiles) {
  int i0 = 0, i1 = t.a.Sq - 1;  // first and last query token of the chunk
  if (t.chunks > 1) {
    i0 = c * kN / G;
    i1 = (min(c * kN + kN, rows) - 1) / G;
  }
  const int p0 = len - t.a.Sq + i0, p1 = min(len - t.a.Sq + i1, t.reach - 1);
  *kmax = p1;
  *kmin = attn_first(p0, t.a.window);
  *tiles = p1 < *kmin ? 1 : p1 / AT_TILE - *kmin / AT_TILE + 1;
}

// Equal shares: first position of CTA i, CTA of a position.
struct AttnShares {
  int each, more;  // the first `more` CTAs take one more
  __device__ __forceinline__ int first(int i) const { return i * each + min(i, more); }
  __device__ __forceinline__ int cta_of(int pos) const {
    const int wide = more * (each + 1);
    return pos < wide ? pos / (each + 1) : more + (pos - wide) / each;
  }
};

// A CTA's share, as pieces of units; every role walks the same.  Positions
// count unit_cost and then the tiles of each unit.
struct AttnWalk {
  int pos, end, unit;  // next position, end of the share, start of the current unit
  int b, h, c, len;
  int kmin, kmax, tiles;     // of the current unit
};

template <int kN>
__device__ __forceinline__ void walk_unit(const AttnTcArgs& t, int G, int rows, AttnWalk& w) {
  attn_unit(t, w.len, G, rows, kN, w.c, &w.kmin, &w.kmax, &w.tiles);
}

template <int kN>
__device__ __forceinline__ void walk_next(const AttnTcArgs& t, int G, int rows, AttnWalk& w) {
  w.unit += t.unit_cost + w.tiles;
  if (++w.c == t.chunks) {
    w.c = 0;
    if (++w.h == t.a.Hkv) {
      w.h = 0;
      ++w.b;
      if (w.b < t.a.B) w.len = attn_length(t.a, w.b);
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

__device__ __forceinline__ uint32_t ld_acquire_u32(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
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

__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
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

// Tiles [j0, j0 + n) of the current unit that lie in the share (n <= 0: none).
__device__ __forceinline__ void walk_piece(const AttnTcArgs& t, const AttnWalk& w, int* j0, int* n) {
  const int tile0 = w.unit + t.unit_cost;
  *j0 = max(0, w.pos - tile0);
  *n = min(w.tiles, w.end - tile0) - *j0;
}

// A share holds two split pieces at most, at its start and at its end: 0, or 1
// for one that comes behind another unit of the share.
__device__ __forceinline__ int piece_slot(const AttnShares& shares, const AttnWalk& w) {
  return shares.first(blockIdx.x) < w.unit ? 1 : 0;
}

// This CTA's part, the `part`-th of `parts`, of joining a unit whose pieces lie
// at slot0 (the first) and from slot1 on, where every second one belongs to a
// CTA's other piece.  All 256 softmax threads; scratch: 256 * AT_JOIN_FLOATS.
template <int kD, int kN>
__device__ __forceinline__ void attn_join(const float* slot0, const float* slot1, int pieces, int live, int part,
                                          int parts, float* scratch, const int* s_row, __nv_bfloat16* out,
                                          float* lse) {
  constexpr int kSlot = AttnTcShape<kD, kN>::kSlotFloats, kSlots = AttnTcShape<kD, kN>::kSlots, kQuads = kD / 4;
  constexpr int kBatch = 6;
  const int wtid = threadIdx.x - 128;
  const int e0 = live * kQuads * part / parts, n = live * kQuads * (part + 1) / parts - e0;  // quads of values
  // four values a thread, relative to the largest reference it meets; where
  // there are fewer, several threads share the pieces
  const int slots = kSlots * pieces, groups = n > 0 && n <= 256 ? min(256 / n, (slots + kBatch - 1) / kBatch) : 1;
  for (int i0 = 0; i0 < n * groups; i0 += 256) {
    const int i = i0 + wtid, g = i / n, e = e0 + i - g * n, col = e / kQuads;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = AT_NONE, sum = 0.f;
    if (i < n * groups) {
      const int p1 = slots * (g + 1) / groups;
      for (int p0 = slots * g / groups; p0 < p1; p0 += kBatch) {
        float M[kBatch];
        float4 l[kBatch], v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {  // all loads in flight at once
          const int p = min(p0 + u, p1 - 1);
          const float* s = (p < kSlots ? slot0 : slot1 + (size_t)(p / kSlots - 1) * (2 * kSlots * kSlot)) +
                           p % kSlots * kSlot;
          v[u] = __ldcg(reinterpret_cast<const float4*>(s + e * 4));
          l[u] = __ldcg(reinterpret_cast<const float4*>(s + kN * kD + 4 * col));
          M[u] = __ldcg(s + kN * kD + 4 * kN + col);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const float here = (l[u].x + l[u].y) + (l[u].z + l[u].w);
          // without a reference and with sums of 0 the column saw no key, and O may
          // not have been written; NaN sums (every score NaN) go on
          if (p0 + u >= p1 || (M[u] == AT_NONE && here == 0.f)) continue;
          const float to = fmaxf(top, M[u]), f = ex2_approx(top - to), w = ex2_approx(M[u] - to);
          top = to;
          sum = fmaf(here, w, sum * f);
          y.x = fmaf(v[u].x, w, y.x * f), y.y = fmaf(v[u].y, w, y.y * f);
          y.z = fmaf(v[u].z, w, y.z * f), y.w = fmaf(v[u].w, w, y.w * f);
        }
      }
    }
    if (groups > 1) {  // n <= 256: one round
      float* at = scratch + wtid * AT_JOIN_FLOATS;
      at[0] = top, at[1] = sum, at[2] = y.x, at[3] = y.y, at[4] = y.z, at[5] = y.w;
      named_barrier_sync(3, 256);
      if (i < n) {
        float all = top;
#pragma unroll 4
        for (int h = 1; h < groups; ++h) all = fmaxf(all, scratch[(h * n + i) * AT_JOIN_FLOATS]);
        sum = 0.f;
        y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int h = 0; h < groups; ++h) {
          const float* s = scratch + (h * n + i) * AT_JOIN_FLOATS;
          const float w = ex2_approx(s[0] - all);
          sum = fmaf(s[1], w, sum);
          y.x = fmaf(s[2], w, y.x), y.y = fmaf(s[3], w, y.y), y.z = fmaf(s[4], w, y.z), y.w = fmaf(s[5], w, y.w);
        }
        top = all;
      }
    }
    if (i < (groups > 1 ? n : n * groups)) {
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(out + (size_t)s_row[col] * kD + (e % kQuads) * 4) =
          make_uint2(pack_bf16(y.x * f, y.y * f), pack_bf16(y.z * f, y.w * f));
      if (lse && e % kQuads == 0)
        lse[s_row[col]] = sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
    }
  }
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
  uint64_t* s_free = s_full + 4;                 // [kScores]
  uint64_t* p_full = s_full + 8;                 // [2]
  uint64_t* pv_done = s_full + 10;               // [2]
  uint64_t* q_full = s_full + 12;                // [2]
  uint64_t* q_free = s_full + 14;                // [2]
  uint64_t* drained = s_full + 16;               // [2]
  float2* s_sc = reinterpret_cast<float2*>(bars + 2 * AT_MAX_STAGES + 18);  // [stages][8] scales of K, V
  int* s_bad = reinterpret_cast<int*>(s_sc + AT_MAX_STAGES * AT_MAX_PAGES);  // [stages] some page invalid
  // of each of the two q in shared memory, [2][N]: first and last key that a
  // column sees, its score factor, its row of the output from the unit's first
  int* s_lo2 = s_bad + AT_MAX_STAGES;
  int* s_hi2 = s_lo2 + 2 * kN;
  float* s_qf2 = reinterpret_cast<float*>(s_hi2 + 2 * kN);
  int* s_row2 = reinterpret_cast<int*>(s_qf2 + 2 * kN);
  float* s_M = reinterpret_cast<float*>(s_row2 + 2 * kN);  // [2][N] reference, log2
  float* s_f = s_M + 2 * kN;                     // [2][N] factors
  float* s_neg = s_f + 2 * kN;                   // [2][N] the references, negated
  float* s_zero = s_neg + 2 * kN;                // [N]
  float* s_red = s_zero + kN;                    // [2][4][2][N] warp maxima, warp sums
  // [2][D][2], by each warpgroup: columns that see a NaN value
  uint32_t* s_nan = reinterpret_cast<uint32_t*>(s_red + 16 * kN);
  int* s_ctl = reinterpret_cast<int*>(s_nan + 4 * kD);  // abort, tmem
  volatile int* s_abort = s_ctl;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(s_ctl + 1);
  static_assert(8 * (2 * AT_MAX_STAGES + 18) + 8 * AT_MAX_STAGES * AT_MAX_PAGES + 4 * AT_MAX_STAGES +
                        4 * (8 * kN + 7 * kN + 16 * kN) + 16 * kD + 64 <=
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
      for (int i = 0; i < Shape::kScores; ++i) {
        mbar_init(s_full + i, 1);
        mbar_init(s_free + i, 4);
      }
      for (int w = 0; w < 2; ++w) {
        mbar_init(p_full + w, 4);
        mbar_init(pv_done + w, 1);
        mbar_init(q_full + w, 1);
        mbar_init(q_free + w, 9);  // the last product that reads q, eight softmax warps
        mbar_init(drained + w, 1);
      }
      fence_mbar_init();
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    __syncwarp();
  } else if (warp == 2) {
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
      const int len = attn_length(a, b);
      int n = 0;
      for (int c = 0; c < t.chunks; ++c) {
        int lo, hi, k;
        attn_unit(t, len, G, rows, kN, c, &lo, &hi, &k);
        n += k;
      }
      return (n + t.chunks * t.unit_cost) * a.Hkv;
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
    const int ctas = min((int)gridDim.x, max(1, total / t.min_share));
    shares.each = total / ctas;
    shares.more = total - shares.each * ctas;
    const bool idle = (int)blockIdx.x >= ctas;  // the whole CTA: it has no tiles
    walk.pos = idle ? 0 : shares.first(blockIdx.x);
    walk.end = idle ? 0 : shares.first(blockIdx.x + 1);
    int at = incl - mine, b = b0;
    const uint32_t owner = __ballot_sync(0xffffffffu, walk.pos >= at && walk.pos < at + mine);
    if (walk.pos >= at && walk.pos < at + mine) {
      for (int n; b + 1 < b1 && walk.pos >= at + (n = tiles_of(b)); ++b) at += n;
    }
    walk.b = __shfl_sync(0xffffffffu, b, __ffs(owner) - 1);
    walk.unit = __shfl_sync(0xffffffffu, at, __ffs(owner) - 1);
    walk.h = walk.c = 0;
    walk.len = attn_length(a, walk.b);
    walk_unit<kN>(t, G, rows, walk);
    while (walk.unit + t.unit_cost + walk.tiles <= walk.pos) walk_next<kN>(t, G, rows, walk);
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

  if (warp >= 3 && walk.pos < walk.end) {
    // ---- q of each piece as two E4M3 terms, and what its columns see: the
    // first piece's by these nine warps together, the others' by warp 3 ahead
    // of the softmax warps, which leave the loop ----
    int qb = 0, publish = -1, publish_slot = 0;  // counter of the split piece before this one, its slot
    uint32_t q_phase = 0;
    int crew = warp - 3, crews = 9;
    auto tell = [&]() {
      named_barrier_sync(AT_BAR_SPLIT + publish_slot, 288);  // the softmax warps have written the piece
      if (lane == 0) {
        __threadfence();
        atomicAdd(t.counters + publish, 1u);
      }
      __syncwarp();
    };
    while (true) {
      int j0, n;
      walk_piece(t, walk, &j0, &n);
      if (n <= 0) break;  // the share ends within the unit's fixed cost
      // The rows as they are into the room of their two terms, then four at a
      // time into terms, eight lanes a row.
      constexpr int kChunks = kD / 8;  // of 16 bytes in a row
      const int r0 = walk.c * kN, live = min(kN, rows - r0);
      const __nv_bfloat16* q0 = a.q + (long long)walk.b * a.q_bs + (long long)walk.h * G * a.q_hs;
      uint8_t* dst = s_q + qb * 2 * Shape::kQBytes;
      auto room_of = [&](int r, int chunk) {
        return dst + (chunk >= kChunks / 2 ? Shape::kQBytes : 0) + r * kD + chunk % (kChunks / 2) * 16;
      };
      wait(q_free + qb, q_phase ^ 1u);
      // lane r has the place of rows r and r + 32, and writes what they see
      long long at_row[2] = {0, 0};
#pragma unroll
      for (int u = 0; u < (kN + 31) / 32; ++u) {
        const int r = lane + 32 * u, rr = r0 + min(r, live - 1);  // columns past the rows: like the last row
        const int i = rr / G, g = rr - i * G, last = walk.len - a.Sq + i;
        at_row[u] = (long long)i * a.q_ts + (long long)g * a.q_hs;
        if (r < kN && crew == 0) {
          s_hi2[qb * kN + r] = min(last, t.reach - 1);  // tokens past the table are masked
          s_lo2[qb * kN + r] = attn_first(last, a.window);
          s_row2[qb * kN + r] = i * a.Hq + g;
        }
      }
      auto row_of = [&](int r) {  // by all lanes
        long long at = __shfl_sync(0xffffffffu, at_row[0], r & 31);
        if (kN > 32) {
          const long long high = __shfl_sync(0xffffffffu, at_row[1], r & 31);
          if (r >= 32) at = high;
        }
        return q0 + at;
      };
      // all loads first: every round a unit a lane, 16 bytes or one value
      const int step = t.q_wide ? 32 * 8 : 32, last = live * kD;
      const int shift = (t.q_wide ? 0 : 3) + (kD == 128 ? 1 : 0), turns = 1 << shift;  // of four rows
      const int fours = (live + 3) / 4;  // with a row in use
      const int rounds = (crews == 1 ? fours : (max(fours - crew, 0) + crews - 1) / crews) << shift;
#pragma unroll 4
      for (int i = 0; i < rounds; ++i) {
        const int v = (crew + (i >> shift) * crews) * 4 * kD + (i & (turns - 1)) * step + (t.q_wide ? lane * 8 : lane);
        const int r = min(v / kD, live - 1), d = v % kD;
        const __nv_bfloat16* src = row_of(r) + d;
        uint8_t* to = room_of(r, d / 8) + d % 8 * 2;
        if (v < last) {
          if (t.q_wide)
            *reinterpret_cast<uint4*>(to) = __ldg(reinterpret_cast<const uint4*>(src));
          else
            *reinterpret_cast<__nv_bfloat16*>(to) = *src;
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int base = 4 * crew; base < kN; base += 4 * crews) {
        constexpr int kPer = kD / 8;  // values of a lane
        const int r = base + (lane >> 3), j = lane & 7;
        uint32_t raw[kPer / 2];
        __nv_bfloat162 top2 = __floats2bfloat162_rn(0.f, 0.f);  // NaN is passed over
#pragma unroll
        for (int c = 0; c < kPer / 8; ++c) {
          const uint4 v = r < live ? *reinterpret_cast<const uint4*>(room_of(r, j * (kPer / 8) + c))
                                   : make_uint4(0u, 0u, 0u, 0u);
          raw[4 * c] = v.x, raw[4 * c + 1] = v.y, raw[4 * c + 2] = v.z, raw[4 * c + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < kPer / 2; ++i)
          top2 = __hmax2(top2, __habs2(*reinterpret_cast<const __nv_bfloat162*>(raw + i)));
        const uint32_t two = *reinterpret_cast<const uint32_t*>(&top2);
        uint32_t most = max(two & 0xffffu, two >> 16) << 16;  // as fp32 bits
        if (most >= 0x7f800000u) {  // an infinite q makes its whole row NaN
          most = 0u;
#pragma unroll
          for (int i = 0; i < kPer / 2; ++i) {
            const uint32_t lo = raw[i] & 0x7fffu, hi = raw[i] >> 16 & 0x7fffu;
            if (lo < 0x7f80u) most = max(most, lo << 16);
            if (hi < 0x7f80u) most = max(most, hi << 16);
            if (lo >= 0x7f80u) raw[i] |= 0x7fffu;
            if (hi >= 0x7f80u) raw[i] |= 0x7fff0000u;
          }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int byte = scale_byte(most);
        const float inv1 = exp2_int(127 - byte);
        const f32x2 inv = pack2(inv1, inv1);
        uint32_t hi[kPer / 4], lo[kPer / 4];
#pragma unroll
        for (int i = 0; i < kPer / 2; ++i) {
          const f32x2 x = mul2(pack2(bf_lo(raw[i]), bf_hi(raw[i])), inv);
          const uint32_t h2 = __nv_cvt_float2_to_fp8x2(unpack2(x), __NV_SATFINITE, __NV_E4M3);
          const float2 back = e4m3x2_to_f32(h2);
          const f32x2 rest = fma2(pack2(back.x, back.y), pack2(-16.f, -16.f), mul2(x, pack2(16.f, 16.f)));
          const uint32_t l2 = __nv_cvt_float2_to_fp8x2(unpack2(rest), __NV_SATFINITE, __NV_E4M3);
          hi[i / 2] = i % 2 ? hi[i / 2] | h2 << 16 : h2;
          lo[i / 2] = i % 2 ? lo[i / 2] | l2 << 16 : l2;
        }
        __syncwarp();  // the rows have been read: their room takes the terms
        if constexpr (kD == 128) {
          uint8_t* at = dst + r * kD + ((j ^ (r & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(at + Shape::kQBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        } else {
          uint8_t* at = dst + r * kD + (((j >> 1) ^ ((r >> 1) & 3)) << 4) + (j & 1) * 8;
          *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(at + Shape::kQBytes) = make_uint2(lo[0], lo[1]);
        }
        if (j == 0) s_qf2[qb * kN + r] = exp2_int(byte - 127) * a.scale_log2;
      }
      fence_proxy_async_smem();
      if (crews > 1) {
        named_barrier_sync(5, 288);
        if (warp > 3) break;
        crew = 0, crews = 1;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full + qb);
      qb ^= 1;
      q_phase ^= qb == 0 ? 1u : 0u;
      if (publish >= 0) tell();
      publish = j0 > 0 || n < walk.tiles ? shares.cta_of(walk.unit + t.unit_cost) : -1;
      publish_slot = piece_slot(shares, walk);
      walk.pos = walk.unit + t.unit_cost + walk.tiles;
      if (walk.pos >= walk.end) break;
      walk_next<kN>(t, G, rows, walk);
    }
    if (warp == 3 && publish >= 0) tell();
  }

  if (warp == 0) {
    // ---- producer: pages of K and V, and their scales --------------------
    const int per_tile = AT_TILE >> t.page_shift;
    const uint64_t policy = l2_policy_evict_first();
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(t, walk, &j0, &n);
      const int first = walk.kmin / AT_TILE + j0;  // key tile of the piece's start
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
          const int row = good ? (pid * a.Hkv + walk.h) * a.page : -1;
          // One lane issues all, as straight code: with a page a turn of a loop
          // the issue was the limit (8 k keys of 16 sequences on pages of 16: 49.4
          // us, two pages a turn 41.7, this 34.0).
          int at[AT_MAX_PAGES];
#pragma unroll
          for (int p = 0; p < AT_MAX_PAGES; ++p) {
            const int r = __shfl_sync(0xffffffffu, row, (used + p) & 31);
            at[p] = p < per_tile ? r : -1;
          }
          if (elect_one()) {
#pragma unroll
            for (int p = 0; p < AT_MAX_PAGES; ++p) {
              uint8_t* to = dst + p * a.page * kD;
              if (at[p] >= 0) {
                tma_load_2d(to, &tm_k, 0, at[p], kv_full + stage, policy);
                tma_load_2d(to + Shape::kKvBytes, &tm_v, 0, at[p], kv_full + stage, policy);
              }
            }
          }
          __syncwarp();
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
      walk.pos = walk.unit + t.unit_cost + walk.tiles;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0) {
      for (int i = max(0, issued - kStages); i < issued; ++i)
        mbar_wait(kv_full + i % kStages, (uint32_t)(i / kStages) & 1u);
    }
  } else if (warp == 1) {
    // ---- products of scores: S = K q^T -----------------------------------
    constexpr uint32_t kId = tc_idesc_e4m3(AT_TILE, 2 * kN, false, false);
    // Descriptors of the first stage and buffer; the others are at a distance.
    const uint64_t d_k = tc_desc(smem_u32(smem), 16, kAtom, kSwz);
    const uint64_t d_q = tc_desc(smem_u32(s_q), 16, kAtom, kSwz);
    int stage = 0, qb = 0;
    uint32_t phase = 0, q_phase = 0, used = 0, tile = 0;
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(t, walk, &j0, &n);
      if (n > 0) {
        bool ok = wait(q_full + qb, q_phase);
        const uint64_t q = d_q + (uint32_t)(qb * 2 * Shape::kQBytes / 16);
        for (int j = 0; j < n; ++j, ++tile) {
          const int sb = tile % Shape::kScores;
          ok = wait(s_free + sb, ((used >> sb) & 1u) ^ 1u) && ok;
          used ^= 1u << sb;
          ok = wait(kv_full + stage, phase) && ok;
          tc_fence_after();
          if (__all_sync(0xffffffffu, ok) && elect_one()) {
            const uint64_t k = d_k + (uint32_t)(stage * 2 * Shape::kKvBytes / 16);
#pragma unroll
            for (int s = 0; s < kD / 32; ++s) tc_mma_f8(tmem + sb * 2 * kN, k + 2 * s, q + 2 * s, kId, s > 0);
            tc_commit(s_full + sb);
            if (j == n - 1) tc_commit(q_free + qb);
          }
          __syncwarp();
          if (++stage == kStages) stage = 0, phase ^= 1u;
        }
        qb ^= 1;
        q_phase ^= qb == 0 ? 1u : 0u;
      }
      walk.pos = walk.unit + t.unit_cost + walk.tiles;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
    // After an abort let what was issued end before TMEM is freed.
    __syncwarp();
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained);
      mbar_wait(drained, 0);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---- products of values: O^T += V^T p^T ------------------------------
    constexpr uint32_t kId = tc_idesc_e4m3(128, 2 * kN, true, true);
    const uint64_t d_v = tc_desc(smem_u32(smem) + Shape::kKvBytes, 0, kAtom, kSwz);
    const uint64_t d_p = tc_desc(smem_u32(s_p), 128, 2048, 0);
    int stage = 0;
    uint32_t p_phase = 0, tile = 0;
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(t, walk, &j0, &n);
      for (int j = 0; j < n; ++j, ++tile) {
        const int w = tile & 1;
        const bool ok = wait(p_full + w, (p_phase >> w) & 1u);
        p_phase ^= 1u << w;
        tc_fence_after();
        if (__all_sync(0xffffffffu, ok) && elect_one()) {
          const uint64_t v = d_v + (uint32_t)(stage * 2 * Shape::kKvBytes / 16);
          const uint64_t p = d_p + (uint32_t)(w * 2 * Shape::kPBytes / 16);
#pragma unroll
          for (int s = 0; s < AT_TILE / 32; ++s)
            tc_mma_f8(tmem + (Shape::kScores + w) * 2 * kN, v + s * 2 * kD, p + s * 32, kId, j >= 2 || s > 0);
          tc_commit(kv_empty + stage);
          tc_commit(pv_done + w);
        }
        __syncwarp();
        if (++stage == kStages) stage = 0;
      }
      walk.pos = walk.unit + t.unit_cost + walk.tiles;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained + 1);
      mbar_wait(drained + 1, 0);
    }
    __syncwarp();
  } else if (warp > 3) {
    // ---- softmax warpgroups ----------------------------------------------
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;              // TMEM lanes of this warp
    const int row = quarter * 32 + lane;       // key of the tile; value index d of O
    const int wtid = tid - 128;                // of both warpgroups
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21);
    const uint32_t t_o = lanes + (Shape::kScores + wg) * 2 * kN;
    uint8_t* my_p = s_p + wg * 2 * Shape::kPBytes;
    float* my_M = s_M + wg * kN;
    float* my_f = s_f + wg * kN;
    float* my_neg = s_neg + wg * kN;
    float* my_red = s_red + wg * 8 * kN;
    uint32_t* my_nan = s_nan + wg * 2 * kD;
    static_assert(4 * Shape::kPBytes >= 256 * AT_JOIN_FLOATS * 4 && 8 * AT_MAX_CTAS <= AT_COUNTERS, "room for joining");
    constexpr bool kKeep = kN <= 32;  // a thread's exponents of a tile stay in registers
    int stage = 0, qb = 0;
    uint32_t phase = 0, s_phase = 0, pv_phase = 0, q_phase = 0, tile = 0;
    if (wtid < kN) s_zero[wtid] = 0.f;
    named_barrier_sync(3, 256);
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(t, walk, &j0, &n);
      if (n <= 0) {  // the share ends within the unit's fixed cost
        walk.pos = walk.end;
        continue;
      }
      const int first = walk.kmin / AT_TILE + j0;
      const int live = min(kN, rows - walk.c * kN);  // columns in use
      const int* s_lo = s_lo2 + qb * kN;
      const int* s_hi = s_hi2 + qb * kN;
      const float* s_qf = s_qf2 + qb * kN;
      const int* s_row = s_row2 + qb * kN;
      const bool split = j0 > 0 || n < walk.tiles;
      // A whole unit of one tile is finished by the warpgroup whose turn it is,
      // while the other works on the next.  Measured with and without (8 key heads
      // of 8 rows, us): 512 sequences of up to 100 tokens 165, 209; 128 of them 39.5,
      // 41.5, at D 64 35.4, 39.2; 1000 of one key head 54.4, 58.8.  Units of one and
      // two tiles in turn pay for it: 128 sequences of up to 250 tokens 52.0, 48.9.
      const bool alone = n == 1 && !split;
      wait(q_full + qb, q_phase);
      if (!alone || (int)(tile & 1u) == wg) {
        if (row < kN) {
          my_M[row] = AT_NONE;
          my_neg[row] = -AT_NONE;
        }
        for (int i = row; i < 2 * kD; i += 128) my_nan[i] = 0u;
        named_barrier_sync(1 + wg, 128);

        const int lo_min = s_lo[0], lo_max = s_lo[live - 1];  // rows are in token order
        const int hi_min = s_hi[0], hi_max = s_hi[live - 1];
        f32x2 l[kN / 2];
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) l[i] = pack2(0.f, 0.f);
        const int first_j = (wg ^ tile) & 1;  // this warpgroup's first tile of the piece
        int st = stage + first_j;
        uint32_t ph = phase;
        if (st >= kStages) st -= kStages, ph ^= 1u;
        bool any_pv = false;
        for (int j = first_j; j < n; j += 2) {
          const int key = (first + j) * AT_TILE + row;
          const int sb = (tile + j) % Shape::kScores;
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
              for (int i = 0; i < kD / 16; ++i)  // lanes at different banks
                reinterpret_cast<uint4*>(v)[(i + lane) % (kD / 16)] = make_uint4(0u, 0u, 0u, 0u);
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
                    if (key >= s_lo[c] && key <= s_hi[c]) atomicOr(my_nan + 2 * d + (c >> 5), 1u << (c & 31));
                }
                words[i] = clean;
              }
            }
          }
          const float kf = sc.x;
          const float lv = __log2f(sc.y);  // the page's, also in lanes whose key is masked
          const float most = fminf(AT_FULL - lv, AT_FAR);  // of an exponent
          // 16 columns of the tile's scores as exponents of 2, plus the column's `neg`
          auto exponents = [&](f32x2* x, int cb, const float* neg) {
            uint32_t v[16], v_lo[16];
            tmem_ld_x16(t_s + cb * 16, v);
            tmem_ld_x16(t_s + kN + cb * 16, v_lo);
            tmem_wait_ld();
            const f32x2 kf2 = pack2(kf, kf);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const ulonglong2 qf = *reinterpret_cast<const ulonglong2*>(s_qf + cb * 16 + i);
              const ulonglong2 m = *reinterpret_cast<const ulonglong2*>(neg + cb * 16 + i);
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                const f32x2 hi = pack2(__uint_as_float(v[i + e]), __uint_as_float(v[i + e + 1]));
                const f32x2 lo = pack2(__uint_as_float(v_lo[i + e]), __uint_as_float(v_lo[i + e + 1]));
                x[(i + e) / 2] = fma2(mul2(fma2(lo, pack2(AT_LO, AT_LO), hi), kf2), e ? qf.y : qf.x, e ? m.y : m.x);
              }
            }
            if (!whole) {
              const int at = page_ok ? key : -1;  // no column sees key -1
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                const int4 lo = *reinterpret_cast<const int4*>(s_lo + cb * 16 + i);
                const int4 hi = *reinterpret_cast<const int4*>(s_hi + cb * 16 + i);
                const float2 a = unpack2(x[i / 2]), b = unpack2(x[i / 2 + 1]);
                x[i / 2] = pack2((at < lo.x) | (at > hi.x) ? -INFINITY : a.x, (at < lo.y) | (at > hi.y) ? -INFINITY : a.y);
                x[i / 2 + 1] = pack2((at < lo.z) | (at > hi.z) ? -INFINITY : b.x, (at < lo.w) | (at > hi.w) ? -INFINITY : b.y);
              }
            }
          };
          f32x2 x[kKeep ? kN / 2 : 8];
          bool move = !any_pv, moved = false;  // a piece's first tile sets the references
          while (true) {
            if (move) {
              // the columns' maxima of x and of x + log2(scale of V)
#pragma unroll 1
              for (int cb = 0; cb < kN / 16; ++cb) {
                f32x2 y2[8];
                float y[16], m[16], mine = 0.f;  // lane i keeps column i's
                exponents(y2, cb, s_zero);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[2 * i] = unpack2(y2[i]).x, y[2 * i + 1] = unpack2(y2[i]).y;
#pragma unroll
                for (int i = 0; i < 16; ++i) m[i] = warp_max_f32(y[i]);
#pragma unroll
                for (int i = 0; i < 16; ++i) mine = lane == i ? m[i] : mine;
                if (lane < 16) my_red[quarter * 2 * kN + cb * 16 + lane] = mine;
                if (t.page_shift >= 5) {  // one page per warp: one scale
                  mine += lv;
                } else {
#pragma unroll
                  for (int i = 0; i < 16; ++i) m[i] = warp_max_f32(y[i] + lv);
#pragma unroll
                  for (int i = 0; i < 16; ++i) mine = lane == i ? m[i] : mine;
                }
                if (lane < 16) my_red[quarter * 2 * kN + kN + cb * 16 + lane] = mine;
              }
              named_barrier_sync(1 + wg, 128);
              if (row < kN) {
                float xm = my_red[row], tm = my_red[kN + row];
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                  xm = fmaxf(xm, my_red[w * 2 * kN + row]);
                  tm = fmaxf(tm, my_red[w * 2 * kN + kN + row]);
                }
                const float M0 = my_M[row], M1 = fmaxf(M0, fmaxf(tm - AT_HEAD, xm - AT_FAR));
                my_f[row] = ex2_approx(M0 - M1);
                my_M[row] = M1;
              my_neg[row] = -M1;
              }
              named_barrier_sync(1 + wg, 128);
              if (any_pv) {
                wait(pv_done + wg, pv_phase);
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < 2 * kN; c += 8) {
                  uint32_t v[8];
                  tmem_ld_x8(t_o + c, v);
                  tmem_wait_ld();
#pragma unroll
                  for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * my_f[c % kN + i]);
                  tmem_st_x8(t_o + c, v);
                }
                tmem_wait_st();
#pragma unroll
                for (int i = 0; i < kN / 2; ++i) l[i] = mul2(l[i], *reinterpret_cast<const f32x2*>(my_f + 2 * i));
              }
              moved = true;
            }
            if (moved && !kKeep) break;
            float top = -INFINITY;
#pragma unroll
            for (int cb = 0; cb < kN / 16; ++cb) {
              f32x2* y = x + (kKeep ? cb * 8 : 0);
              exponents(y, cb, my_neg);
#pragma unroll
              for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(unpack2(y[i]).x, unpack2(y[i]).y));
            }
            if (moved) break;
            move = named_barrier_any(1 + wg, 128, top > most);
            if (!move) break;
          }
          if (any_pv) {  // p of the previous tile has been read
            wait(pv_done + wg, pv_phase);
            pv_phase ^= 1u;
          }
          any_pv = true;
          const f32x2 vf2 = pack2(vf, vf);
          const float shift = (float)(int)((uint32_t)key * AT_GOLDEN) * AT_SHIFT;
          const f32x2 shift2 = pack2(shift, shift);
#pragma unroll
          for (int cb = 0; cb < kN / 16; ++cb) {
            f32x2* y = x + (kKeep ? cb * 8 : 0);
            if (!kKeep) exponents(y, cb, my_neg);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float2 e2 = unpack2(y[i / 2]);
              f32x2 p2 = pack2(ex2_approx(e2.x), ex2_approx(e2.y));
              l[cb * 8 + i / 2] = add2(l[cb * 8 + i / 2], p2);
              p2 = mul2(p2, vf2);
              const f32x2 p16 = fma2(p2, pack2(16.f, 16.f), shift2);
              const float2 p = unpack2(p2);
              // the nearest values of four significant bits, and of multiples of
              // E4M3's quantum 2^-9 below its normal range (2^14 + 2^13 has that ulp)
              f32x2 s2 = pack2(__uint_as_float((__float_as_uint(p.x) + 0x00080000u) & 0xfff00000u),
                               __uint_as_float((__float_as_uint(p.y) + 0x00080000u) & 0xfff00000u));
              s2 = add2(add2(s2, pack2(24576.f, 24576.f)), pack2(-24576.f, -24576.f));
              const float2 s = unpack2(s2), r = unpack2(fma2(s2, pack2(-16.f, -16.f), p16));
              const uint32_t h2 = __nv_cvt_float2_to_fp8x2(s, __NV_SATFINITE, __NV_E4M3);
              const uint32_t l2 = __nv_cvt_float2_to_fp8x2(r, __NV_SATFINITE, __NV_E4M3);
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
          tc_fence_before();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(s_free + sb);
            mbar_arrive(p_full + wg);
          }
          st += 2;
          if (st >= kStages) st -= kStages, ph ^= 1u;
        }

        // ---- the piece's end: sums over the keys, then both warpgroups join --
        if (any_pv) {
          wait(pv_done + wg, pv_phase);
          pv_phase ^= 1u;
          tc_fence_after();
        }
        named_barrier_sync(1 + wg, 128);  // the other warps' notes of NaN values
        float ls[kN];
#pragma unroll
        for (int i = 0; i < kN / 2; ++i) ls[2 * i] = unpack2(l[i]).x, ls[2 * i + 1] = unpack2(l[i]).y;
        warp_sum_columns<kN>(ls, lane);
        const size_t out0 = (size_t)walk.b * a.Sq * a.Hq + walk.h * G;  // output row of the unit's first
        const uint64_t poison = row < kD ? (uint64_t)my_nan[2 * row] | (uint64_t)my_nan[2 * row + 1] << 32 : 0ull;
        constexpr int kSlots = Shape::kSlots;
        float* slot = t.slots + (size_t)(2 * blockIdx.x + piece_slot(shares, walk)) * (kSlots * Shape::kSlotFloats);
        if (split && kSlots == 2) {
          // as it is into the workspace; whoever joins the unit does the rest
          slot += wg * Shape::kSlotFloats;
#pragma unroll
          for (int i = 0; i < (kN + 31) / 32; ++i)
            __stcg(slot + kN * kD + column_of<kN>(lane, i) * 4 + quarter, ls[i]);
          if (row < kN) __stcg(slot + kN * kD + 4 * kN + row, my_M[row]);
          if (any_pv) {
#pragma unroll 1
            for (int cb = 0; cb < live; cb += 8) {
              uint32_t v[8], v_lo[8];
              tmem_ld_x8(t_o + cb, v);
              tmem_ld_x8(t_o + kN + cb, v_lo);
              tmem_wait_ld();
              if (row < kD) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float y = fmaf(__uint_as_float(v_lo[i]), AT_LO, __uint_as_float(v[i]));
                  __stcg(slot + (cb + i) * kD + row, (poison >> (cb + i)) & 1ull ? __uint_as_float(0x7fc00000u) : y);
                }
              }
            }
          }
          tc_fence_before();
        } else if (alone) {
#pragma unroll
          for (int i = 0; i < (kN + 31) / 32; ++i) my_red[quarter * kN + column_of<kN>(lane, i)] = ls[i];
          named_barrier_sync(1 + wg, 128);
          if (row < kN) {
            const float sum = (my_red[row] + my_red[kN + row]) + (my_red[2 * kN + row] + my_red[3 * kN + row]);
            my_f[row] = sum == 0.f ? 0.f : 1.f / sum;
            if (a.lse && row < live)
              a.lse[out0 + s_row[row]] = sum == 0.f ? -INFINITY : my_M[row] * 0.6931471805599453f + logf(sum);
          }
          named_barrier_sync(1 + wg, 128);
#pragma unroll 1
          for (int cb = 0; cb < live; cb += 8) {
            uint32_t v[8], v_lo[8];
            tmem_ld_x8(t_o + cb, v);
            tmem_ld_x8(t_o + kN + cb, v_lo);
            tmem_wait_ld();
            if (row < kD) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int col = cb + i;
                float y = fmaf(__uint_as_float(v_lo[i]), AT_LO, __uint_as_float(v[i])) * my_f[col];
                if ((poison >> col) & 1ull) y = __uint_as_float(0x7fc00000u);
                if (col < live) a.out[(out0 + s_row[col]) * kD + row] = __float2bfloat16_rn(y);
              }
            }
          }
          tc_fence_before();
        } else {
          // columns [wg * N/2, ...) are finished here, the others by the other warpgroup
          constexpr int kHalf = kN / 2;
          float* give = reinterpret_cast<float*>(my_p);  // [N/2][128]
          const float* take = reinterpret_cast<const float*>(s_p + (1 - wg) * 2 * Shape::kPBytes);
#pragma unroll
          for (int i = 0; i < (kN + 31) / 32; ++i) my_red[quarter * kN + column_of<kN>(lane, i)] = ls[i];
#pragma unroll 1
          for (int cb = 0; cb < kHalf; cb += 8) {
            uint32_t v[8], v_lo[8];
            if (any_pv) {
              tmem_ld_x8(t_o + (1 - wg) * kHalf + cb, v);
              tmem_ld_x8(t_o + kN + (1 - wg) * kHalf + cb, v_lo);
              tmem_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float y = any_pv ? fmaf(__uint_as_float(v_lo[i]), AT_LO, __uint_as_float(v[i])) : 0.f;
              if ((poison >> ((1 - wg) * kHalf + cb + i)) & 1ull) y = __uint_as_float(0x7fc00000u);
              give[(cb + i) * 128 + row] = y;
            }
          }
          named_barrier_sync(3, 256);
          // a thread per column: the factors of both O
          if (wtid < kN) {
            const float M0 = s_M[wtid], M1 = s_M[kN + wtid], M = fmaxf(M0, M1);
            const float f0 = ex2_approx(M0 - M), f1 = ex2_approx(M1 - M);
            float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) l0 += s_red[w * kN + wtid], l1 += s_red[8 * kN + w * kN + wtid];
            const float sum = l0 * f0 + l1 * f1;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (split) {
              f = 1.f;
              __stcg(reinterpret_cast<float4*>(slot + kN * kD) + wtid, make_float4(sum, 0.f, 0.f, 0.f));
              __stcg(slot + kN * kD + 4 * kN + wtid, M);
            } else if (a.lse && wtid < live)
              a.lse[out0 + s_row[wtid]] = sum == 0.f ? -INFINITY : M * 0.6931471805599453f + logf(sum);
            s_f[wtid] = f * f0;
            s_f[kN + wtid] = f * f1;
          }
          named_barrier_sync(3, 256);
#pragma unroll 1
          for (int cb = 0; cb < kHalf; cb += 8) {
            const int c0 = wg * kHalf + cb;
            if (c0 >= live) break;
            uint32_t v[8], v_lo[8];
            if (any_pv) {
              tmem_ld_x8(t_o + c0, v);
              tmem_ld_x8(t_o + kN + c0, v_lo);
              tmem_wait_ld();
            }
            if (row < kD) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int col = c0 + i;
                float y = any_pv ? fmaf(__uint_as_float(v_lo[i]), AT_LO, __uint_as_float(v[i])) : 0.f;
                if ((poison >> col) & 1ull) y = __uint_as_float(0x7fc00000u);
                y = y * s_f[wg * kN + col] + take[(cb + i) * 128 + row] * s_f[(1 - wg) * kN + col];
                if (split)
                  __stcg(slot + col * kD + row, y);
                else if (col < live)
                  a.out[(out0 + s_row[col]) * kD + row] = __float2bfloat16_rn(y);
              }
            }
          }
          tc_fence_before();
        }
        if (split) {
          named_barrier_arrive(AT_BAR_SPLIT + piece_slot(shares, walk), 288);  // the q warp tells the others
          const int tile0 = walk.unit + t.unit_cost;
          const int ca = shares.cta_of(tile0), cz = shares.cta_of(tile0 + walk.tiles - 1);
          if ((int)blockIdx.x != cz) {  // this piece ends the share
            const uint32_t pieces = cz - ca + 1;
            uint32_t* came = t.counters + ca;
            if (wtid == 0) {
              const uint64_t t0 = globaltimer_ns();
              while (ld_acquire_u32(came) != pieces) {
                if (*s_abort || globaltimer_ns() - t0 > WD_WAIT_LIMIT_NS) {
                  *s_abort = 1;
                  raise_status(a.status, WD_STATUS_WAIT_TIMEOUT);
                  break;
                }
              }
            }
            named_barrier_sync(3, 256);
            // only the first CTA of a unit can have begun with another unit
            attn_join<kD, kN>(t.slots + (size_t)(2 * ca + (shares.first(ca) < walk.unit ? 1 : 0)) * (kSlots * Shape::kSlotFloats),
                              t.slots + (size_t)(2 * ca + 2) * (kSlots * Shape::kSlotFloats), pieces, live, blockIdx.x - ca,
                              cz - ca, reinterpret_cast<float*>(s_p), s_row, a.out + out0 * kD,
                              a.lse ? a.lse + out0 : nullptr);
            // the last joiner leaves the counters as the next call needs them
            named_barrier_sync(3, 256);
            if (wtid == 0 && atomicAdd(came + AT_MAX_CTAS, 1u) + 1 == pieces - 1) {
              came[0] = 0u;
              came[AT_MAX_CTAS] = 0u;
            }
          }
        }
        // p and the statistics may be written again
        if (alone)
          named_barrier_sync(1 + wg, 128);
        else
          named_barrier_sync(3, 256);
      }
      if (lane == 0) mbar_arrive(q_free + qb);
      qb ^= 1;
      q_phase ^= qb == 0 ? 1u : 0u;
      stage += n % kStages;
      phase ^= (uint32_t)(n / kStages) & 1u;
      if (stage >= kStages) stage -= kStages, phase ^= 1u;
      tile += (uint32_t)n;
      walk.pos = walk.unit + t.unit_cost + walk.tiles;
      if (walk.pos < walk.end) walk_next<kN>(t, G, rows, walk);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2) tmem_dealloc(tmem, Shape::kTmem);
}

}  // namespace wdb

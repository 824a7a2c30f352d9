// Attention over the FP8 paged cache of sequences that begin with the same tokens
// (head sizes 64 and 128), sm_100a: the shared tokens' pages are read once for all
// sequences, each sequence's own tokens after them for itself, in one launch;
// attn_prefix_join_kernel joins the parts.
//
// With O = sum 2^(x + e - m) c and l = sum 2^(x - n) over any set of tokens, whose values
// are c 2^e (codes and their page's scale), two sets join as O = O1 2^(m1 - M) + O2
// 2^(m2 - M), M = max(m1, m2), l and n likewise: the prefix is one set, a sequence's own
// tokens another, both cut further over the CTAs.  In the end out = O 2^(m - n) / l.
//
// The rows that share keys are the M side of the products, 128 of them a tile: over
// the prefix the query tokens and heads of all sequences that share a key head, two
// tiles at once where there are more than 128; over a sequence's own tokens its own.
// * S = q K^T: K's codes straight from the cache through TMA (kind::f8f6f4), q as
//   two E4M3 terms (hi = the nearest, lo = the nearest to what remains) that are
//   products of one sum; exact for ten octaves below a row's largest value, and
//   within 2^-18 of it below. The page's scale of K, a power of two, is a factor
//   of the exponent.
// * O += P V in fp16: P as it is held in TMEM, in the place of the scores it was
//   made of; V's codes widened to fp16, exactly, by four warps once for both row
//   tiles. A weight is rounded to fp16, within 2^-11 of itself or, where that is more,
//   2^-31 of the row's largest (AP_HEAD); in bf16 (2^-8) it made as much of the error as
//   the output's own rounding. The softmax sum is of the weights before that, in fp32.
// * The page's scale of V, a power of two too, is part of the weight's exponent, so
//   that O holds sums of codes: it cannot overflow, and what a masked token's page
//   has for a scale is in no product. l takes the same exponential times 2^(m - e - n).
// * A row is a thread's: no sums or maxima across threads. References (m of O, n of
//   l) are lazy whole numbers: they move when a weight would pass 2^AP_ROOM, and O is
//   then rescaled in TMEM.
//
// Warps: two groups of four for the softmax, a row tile each (or, of a unit with one
// row tile, every second tile of tokens), a warp for each that issues its products,
// four that widen V, one that loads. A tile's scores come as two halves of 64 tokens
// with places of their own, so that a group works on one while the tensor core makes
// the other.
//
// Work: the token tiles of all units, (key head, 256 rows) over the prefix and
// (sequence, key head, 128 rows) over own tokens, in one line, weighted by what they
// cost, cut into equal shares, one a CTA.
//
// Measured (B200, D 128, 4 key heads of 8 rows): 64 sequences with up to 512 tokens of
// their own behind 8192 62 us, 128 with up to 256 behind 16384 109 us (318 TFLOP/s, a
// fifth of cuBLAS's bf16 rate).  attn_decode_fp8 (wd_attn_fp8_tc.cuh) reads the prefix for
// every sequence, keys in the place of rows, and is ahead while B * prefix * key heads is
// below about a million (measured: warp_decode_block.h).
//
// Bound by latency: two softmax warps a scheduler take about 5000 clocks for a tile pair
// whose products are 2048 and whose exponentials are 2048 on the special-function units;
// a unit of own tokens costs about 4000 beside its tiles, for its q, its masks and its
// output come one after the other.
#pragma once

#include <cuda_fp16.h>

#include "wd_attn_fp8_tc.cuh"

namespace wdb {

constexpr int AP_TILE = 128;       // tokens of a tile, rows of a row tile
constexpr int AP_HALF = 64;        // tokens whose scores are made and weighed at once
constexpr int AP_THREADS = 512;    // softmax 2 x 128, V 128, load, 2 x products, an idle warp
constexpr int AP_WARP_V = 8, AP_WARP_LOAD = 12, AP_WARP_MMA = 13;
constexpr int AP_K_STAGES = 3;
constexpr int AP_RING = 8;         // scales of pages, kept until the softmax has used them
constexpr float AP_ROOM = 15.f;    // log2 of the largest weight before a reference moves: fp16 ends at 2^16
// The same of the row's largest when O's reference is set. fp16's quantum is 2^-24: with 2^7
// a million tokens that it loses are 2^-11 of the row's largest together, and the reference
// need not move before the scores have grown by eight octaves.
constexpr float AP_HEAD = 7.f;
// A page's e counts as m - n - AP_FAR at least, so that l finds what it adds up above the
// smallest number: weights whose products are 2^(AP_ROOM - AP_FAR) of the row's largest at most.
constexpr float AP_FAR = 64.f;
// Of a unit, beside its tiles (2 of two row tiles, 1 of one).  Geometric mean of 40 shapes
// (2 to 232 sequences, 1 to 128 heads, up to 36330 shared and 1670 own tokens, cold) with
// 1, 2, 3, 4 and 6: 45.1, 43.6, 43.7, 43.7 and 44.5 us. Flat from 2 to 4: many units of a
// tile or two take less (229 sequences of 8 x 8 rows behind 189 tokens 157, 171 and 183 us
// with 2, 3 and 4), long prefixes and own parts more (128 behind 16384 131, 116 and 112).
constexpr int AP_UNIT_COST = 4;
constexpr int AP_HEADER = 256;     // bytes of the plan, for the join

template <int kD>
struct AttnPrefixShape {
  static constexpr int kQTerm = AP_TILE * kD;        // bytes of a term of a row tile's q
  static constexpr int kKBytes = AP_TILE * kD;
  static constexpr int kVBytes = 2 * AP_TILE * kD;   // fp16
  static constexpr int kUnits = kD / 16;             // 16-byte units of a cached row
  static constexpr int kOffK = 4 * kQTerm;
  static constexpr int kOffRaw = kOffK + AP_K_STAGES * kKBytes;  // two tiles of V as it is cached
  static constexpr int kOffV = kOffRaw + 2 * kKBytes;
  static constexpr int kOffMisc = kOffV + 2 * kVBytes;
  static constexpr int kMiscBytes = 2 * AP_TILE * kUnits * 2 + 2 * AP_TILE * 4 + 3 * AP_RING * 8 * 4 + 768;
  static constexpr int kSmem = kOffMisc + kMiscBytes + 1024;  // + alignment slack
};

struct AttnPrefixArgs {
  AttnArgs a;
  const int32_t* prefix;  // tokens that all sequences share
  uint8_t* plan;          // AP_HEADER bytes
  int32_t* own_start;     // [B] place of a sequence's first unit in the line
  float* slots;           // of prefix units: O [D/4][128][4], statistics [128][4]: O's reference, sum, its reference
  float* own_slots;       // of own units: the same with own_rows for 128
  int row_blocks;         // prefix units of a key head
  int two;                // they have two row tiles
  int own_blocks;         // units of a (sequence, key head)
  int own_rows;           // rows of their slots, at most 128
  int own_slot;           // floats of one, a multiple of 4
  int reach;              // tokens that the block table can address
  int page_shift;
  int q_wide;
};

// What the join needs to find the parts again.
struct AttnPrefixPlan {
  int each, more;     // AttnShares
  int tiles;          // of a prefix unit
  int from;           // first token that is a sequence's own
};

// Whole pages of the prefix that the table holds, in tokens.
__device__ __forceinline__ int prefix_tokens(const AttnPrefixArgs& t) {
  return min(max(__ldg(t.prefix), 0), t.reach) >> t.page_shift << t.page_shift;
}

// The kernel's rare and repeated parts are functions of their own: with all of them
// inlined its code (132 KB) did not stay in the instruction caches, and every role
// waited for instructions (128 sequences behind 16384 tokens 189 us).

// A sequence's own tokens that some row sees: first (of a page) and tiles.
__device__ __noinline__ int own_tiles(const AttnPrefixArgs& t, int len, int from, int* key0) {
  *key0 = max(attn_first(max(len - t.a.Sq, 0), t.a.window) >> t.page_shift << t.page_shift, from);
  return max((min(len, t.reach) - *key0 + AP_TILE - 1) / AP_TILE, 0);
}

// A CTA's share, as pieces of units; every role walks the same. A tile lies where its
// first position does.
struct AttnPrefixWalk {
  int pos, end;              // next position, end of the share
  int start, unit, b, h, c;  // of the current unit: place, number, sequence (-1: prefix), key head, block
  int tiles, shift, key0;    // tiles, log2 of the positions of each, first token
  int limit;                 // tokens that count end here
};

struct AttnPrefixWork {
  int units, tiles, shift, key0, shared;   // of the prefix
  int first, from;                         // first token of it that a row sees; first own token
};

__device__ __noinline__ void own_unit(const AttnPrefixArgs& t, const AttnPrefixWork& p, AttnPrefixWalk& w) {
  const int len = attn_length(t.a, w.b);
  w.tiles = own_tiles(t, len, p.from, &w.key0);
  w.limit = min(len, t.reach);
}

// To the next unit (its tiles may be none: a sequence without own tokens).
__device__ __noinline__ void walk_on(const AttnPrefixArgs& t, const AttnPrefixWork& p, AttnPrefixWalk& w) {
  w.start += AP_UNIT_COST + (w.tiles << w.shift);
  w.pos = w.start;
  ++w.unit;
  if (w.b < 0) {
    if (++w.c == t.row_blocks) w.c = 0, ++w.h;
    if (w.unit < p.units) return;
    w.b = 0, w.h = 0, w.c = 0, w.shift = 0;
  } else {
    if (++w.c < t.own_blocks) return;
    w.c = 0;
    if (++w.h < t.a.Hkv) return;
    w.h = 0, ++w.b;
  }
  while (w.b < t.a.B) {
    own_unit(t, p, w);
    if (w.tiles > 0) return;
    w.unit += t.a.Hkv * t.own_blocks;
    ++w.b;
  }
  w.pos = w.end;
}

// Tiles [j0, j0 + n) of the current unit that lie in the share (n <= 0: none).
__device__ __forceinline__ void walk_piece(const AttnPrefixWalk& w, int* j0, int* n) {
  const int base = w.start + AP_UNIT_COST;
  const int up = (1 << w.shift) - 1;
  *j0 = max(w.pos - base + up, 0) >> w.shift;
  *n = min(w.tiles, max(w.end - base + up, 0) >> w.shift) - *j0;
}

// Instruction descriptor for kind::f16: fp32 D, fp16 A and B (formats 0), both K-major.
__host__ __device__ constexpr uint32_t tc_idesc_f16(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                               bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

// Tie the values to the wait for them.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.wait::ld.sync.aligned;"
      : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
        "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]),
        "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
        "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
      :
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Positions of the own units of a sequence.
__device__ __noinline__ int own_place(const AttnPrefixArgs& t, int len, int from) {
  int key0;
  const int tiles = own_tiles(t, len, from, &key0);
  return tiles > 0 ? t.a.Hkv * t.own_blocks * (AP_UNIT_COST + tiles) : 0;
}

// Eight bf16 values off the 16-byte grid.
__device__ __noinline__ uint4 load_narrow(const __nv_bfloat16* p) {
  uint32_t e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) e[k] = __bfloat16_as_ushort(p[k]);
  return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}

// Sixteen E4M3 codes as fp16, exactly. s.eeee.mmm lies at bits 15 and 13..7 of its half: an
// exponent field of e with bias 15 for 7, hence the factor 2^8, subnormals too. Returns true
// where some code is NaN (magnitude 0x7f), which becomes 480.
__device__ __forceinline__ bool e4m3x16_to_f16(const uint4& v, uint32_t (&p)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  const __half2 two8 = __float2half2_rn(0x1p8f);
  uint32_t zero_bytes = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t h[2];  // two bytes each, with their signs above them
    asm("prmt.b32 %0, %1, 0, 0x9180;" : "=r"(h[0]) : "r"(w[q]));
    asm("prmt.b32 %0, %1, 0, 0xB3A2;" : "=r"(h[1]) : "r"(w[q]));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t bits = h[i] << 7 & 0xbf80bf80u;
      const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&bits), two8);
      p[2 * q + i] = *reinterpret_cast<const uint32_t*>(&y);
    }
    zero_bytes |= (~w[q] & 0x7f7f7f7fu) - 0x01010101u;
  }
  return (zero_bytes & 0x80808080u) != 0u;
}

template <int kD>
__global__ void __launch_bounds__(AP_THREADS, 1)
    attn_prefix_kernel(const AttnPrefixArgs t, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
  using Shape = AttnPrefixShape<kD>;
  constexpr uint32_t kSwz = kD == 128 ? 2u : 4u;
  constexpr uint32_t kAtom = kD == 128 ? 1024u : 512u;
  constexpr int kUnits = Shape::kUnits;
  const AttnArgs& a = t.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.Hkv;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                 // [2 groups][hi, lo]
  uint8_t* s_k = smem + Shape::kOffK;  // [stages]
  uint8_t* s_raw = smem + Shape::kOffRaw;  // [2][128][D] codes of V
  uint8_t* s_v = smem + Shape::kOffV;  // [2][D / 64][128][64]
  uint16_t* s_nan = reinterpret_cast<uint16_t*>(smem + Shape::kOffMisc);  // [2][128][units]: values that are NaN
  float* s_qf = reinterpret_cast<float*>(s_nan + 2 * AP_TILE * kUnits);   // [2][128]
  float* s_kf = s_qf + 2 * AP_TILE;    // [ring][8]: factor of 16 tokens each, -1 where their page is invalid
  float* s_ve = s_kf + AP_RING * 8;    // [ring][8]: log2 of the scale of V of 16 tokens each
  int* s_vb = reinterpret_cast<int*>(s_ve + AP_RING * 8);  // [ring][8]: its byte, or -1
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_vb + AP_RING * 8);
  uint64_t* k_full = bars;                 // [stages]
  uint64_t* k_empty = k_full + AP_K_STAGES;  // [groups][stages]
  uint64_t* kf_full = k_empty + 2 * AP_K_STAGES;  // [ring]
  uint64_t* r_full = kf_full + AP_RING;    // [2]
  uint64_t* r_empty = r_full + 2;          // [2]
  uint64_t* v_full = r_full + 4;           // [2]
  uint64_t* v_empty = r_full + 6;          // [groups][2]
  uint64_t* q_full = r_full + 10;          // [groups]
  uint64_t* s_full = r_full + 12;          // [groups][halves]
  uint64_t* p_full = r_full + 16;          // [groups][halves]
  uint64_t* pv_done = r_full + 20;         // [groups][halves]
  uint64_t* drained = r_full + 24;         // [groups]
  int* s_has_nan = reinterpret_cast<int*>(r_full + 27);  // [2][4 warps], 16-byte aligned: 1 + the last tile of the stage with a NaN value
  int* s_bad = s_has_nan + 8;                            // [ring] some page of the tile is invalid
  volatile int* s_abort = s_bad + AP_RING;
  uint32_t* s_tmem = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(s_abort + 1));
  int* s_start = reinterpret_cast<int*>(s_tmem + 1);     // the share's first unit, the plan
  static_assert((3 * AP_K_STAGES + AP_RING + 27) % 2 == 0 && 8 * (3 * AP_K_STAGES + AP_RING + 27) + 4 * (8 + AP_RING + 2 + 24) <= 768, "small arrays");

  pdl_launch_dependents();  // the join's blocks come as these go, and wait there
  if (warp == AP_WARP_LOAD && lane == 0) {
    *s_abort = 0;
    for (int i = 0; i < AP_K_STAGES; ++i) mbar_init(k_full + i, 1);
    for (int i = 0; i < 2 * AP_K_STAGES; ++i) mbar_init(k_empty + i, 1);
    for (int i = 0; i < AP_RING; ++i) mbar_init(kf_full + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(r_full + i, 1), mbar_init(r_empty + i, 4), mbar_init(v_full + i, 4), mbar_init(q_full + i, 4);
      mbar_init(drained + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(v_empty + i, 1), mbar_init(s_full + i, 1), mbar_init(p_full + i, 4), mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < 8; ++i) s_has_nan[i] = 0;
    fence_mbar_init();
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  } else if (warp == AP_WARP_MMA) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  } else if (warp == 0) {
    // ---- the work and this CTA's share of it ----
    const int from = prefix_tokens(t);
    const int per = (a.B + 31) / 32;  // sequences of a lane, in order
    const int b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B);
    int most = -1, least = 0x7fffffff, mine = 0, at = b0;  // longest, shortest that is not empty, the first longest
#pragma unroll 1
    for (int base = b0; base < b1; base += 4) {
      int len[4];  // in flight together
#pragma unroll
      for (int i = 0; i < 4; ++i) len[i] = base + i < b1 ? attn_length(a, base + i) : -1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (len[i] < 0) continue;
        mine += own_place(t, len[i], from);
        if (len[i] > most) most = len[i], at = base + i;
        if (len[i] > 0) least = min(least, len[i]);
        if (len[i] > t.reach) raise_status(a.status, WD_STATUS_BAD_PAGE);
      }
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const int own = __shfl_sync(0xffffffffu, incl, 31);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int n = __shfl_xor_sync(0xffffffffu, most, o), b = __shfl_xor_sync(0xffffffffu, at, o);
      if (n > most || (n == most && b < at)) most = n, at = b;
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    AttnPrefixWork p;
    p.from = from;
    p.shared = min(from, most);
    p.first = attn_first(max(least - a.Sq, 0), a.window);
    p.key0 = p.first / AP_TILE * AP_TILE;
    p.tiles = max((p.shared - p.key0 + AP_TILE - 1) / AP_TILE, 0);
    p.units = p.tiles > 0 ? a.Hkv * t.row_blocks : 0;
    p.shift = t.two;
    const int first_own = p.units * (AP_UNIT_COST + (p.tiles << p.shift)), total = first_own + own;
    const int ctas = min((int)gridDim.x, max(1, total / 3));
    AttnShares shares;
    shares.each = total / ctas;
    shares.more = total - shares.each * ctas;
    const bool idle = (int)blockIdx.x >= ctas || total == 0;
    AttnPrefixWalk w;
    w.pos = idle ? 0 : shares.first(blockIdx.x);
    w.end = idle ? 0 : shares.first(blockIdx.x + 1);
    int place = first_own + incl - mine;  // of the lane's sequences
    if (idle || w.pos < first_own) {
      const int len = AP_UNIT_COST + (p.tiles << p.shift);
      w.unit = idle ? 0 : w.pos / len;
      w.start = w.unit * len;
      w.b = -1;
      w.h = w.unit / t.row_blocks;
      w.c = w.unit - w.h * t.row_blocks;
      w.tiles = p.tiles, w.shift = p.shift, w.key0 = p.key0, w.limit = p.shared;
      if (lane == 0) *reinterpret_cast<AttnPrefixWalk*>(s_start) = w;
    } else if (w.pos >= place && w.pos < place + mine) {  // the lane with the sequence that the share begins in
      w.b = b0;
      for (int n; w.pos >= place + (n = own_place(t, attn_length(a, w.b), from)); ++w.b) place += n;
      own_unit(t, p, w);
      const int len = AP_UNIT_COST + w.tiles, k = (w.pos - place) / len;
      w.start = place + k * len;
      w.unit = p.units + w.b * a.Hkv * t.own_blocks + k;
      w.h = k / t.own_blocks;
      w.c = k - w.h * t.own_blocks;
      w.shift = 0;
      *reinterpret_cast<AttnPrefixWalk*>(s_start) = w;
    }
    if (lane == 0) {
      *reinterpret_cast<AttnPrefixWork*>(s_start + sizeof(w) / 4) = p;
      s_start[(sizeof(w) + sizeof(p)) / 4] = at;
    }
    static_assert(sizeof(AttnPrefixWalk) + sizeof(AttnPrefixWork) + 4 <= 24 * 4, "room for the share");
    if (blockIdx.x == 0) {  // for the join
      if (lane == 0) *reinterpret_cast<AttnPrefixPlan*>(t.plan) = {shares.each, shares.more, p.tiles, from};
      place = first_own + incl - mine;
#pragma unroll 1
      for (int b = b0; b < b1; ++b) {
        t.own_start[b] = place;
        place += own_place(t, attn_length(a, b), from);
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  AttnPrefixWalk walk = *reinterpret_cast<const AttnPrefixWalk*>(s_start);
  const AttnPrefixWork work = *reinterpret_cast<const AttnPrefixWork*>(s_start + sizeof(walk) / 4);
  const int lead = s_start[(sizeof(walk) + sizeof(work)) / 4];  // the longest sequence

  // Bounded wait of a whole warp; once one gave up, none waits and nothing more is
  // issued, but every role still runs its loop to the end.  The lanes leave together:
  // what follows are warp-wide TMEM accesses.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return wait_on(bar, parity, s_abort, a.status);
  };
  // Of a piece's n tiles from the CTA's `count`-th on: the first that group w takes, how
  // many, and how far apart.
  auto two_of = [&](const AttnPrefixWalk& w) { return w.b < 0 && t.two; };
  auto first_of = [](bool two, int count, int w) { return two ? 0 : (w ^ count) & 1; };
  auto tiles_of = [](bool two, int n, int first) { return two ? n : (n - first + 1) / 2; };

  if (warp < AP_WARP_V) {
    // ---- softmax: a row a thread ---------------------------------------------
    const int w = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21);
    const uint32_t t_o = lanes + 2 * AP_TILE + w * kD;
    uint8_t* my_q = s_q + w * 2 * Shape::kQTerm;
    int count = 0;      // tiles of this CTA before the piece
    uint32_t s_phase = 0;
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(walk, &j0, &n);
      const bool two = two_of(walk), own = walk.b >= 0;
      const int first = first_of(two, count, w), mine = n > 0 ? tiles_of(two, n, first) : 0;
      const int r0 = two ? (2 * walk.c + w) * AP_TILE : walk.c * AP_TILE, piece0 = walk.key0 + j0 * AP_TILE;
      const int live = min((own ? a.Sq * G : a.B * a.Sq * G) - r0, AP_TILE);  // rows in use (or <= 0)
      if (n > 0) {
        // tokens that the row sees, [lo, hi]; a row past the last: all, for no one
        int lo = 0, hi = 0x7fffffff;
        const int s = (r0 + row) / G, b = own ? walk.b : s / a.Sq, i_q = own ? s : s - b * a.Sq;
        long long from_q = 0;
        if (row < live) {
          const int last = attn_length(a, b) - a.Sq + i_q;
          lo = attn_first(last, a.window);
          if (own) lo = max(lo, work.from);
          hi = min(last, walk.limit - 1);
          from_q = (long long)b * a.q_bs + (long long)i_q * a.q_ts + (long long)(walk.h * G + r0 + row - s * G) * a.q_hs;
        }
        float M = AT_NONE, N = AT_NONE;  // references of O and of the sum
        f32x2 l2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
        uint32_t poison[kD / 32];
#pragma unroll
        for (int i = 0; i < kD / 32; ++i) poison[i] = 0u;
        const int here = min(live - quarter * 32, 32);  // rows of this warp
        if (mine > 0) {
          // q of the rows: as they are into the room of their two terms, all loads in
          // flight, then four at a time into terms, eight lanes a row
          constexpr int kPer = kD / 8, kChunks = kD / 8, kRows = 32 / kChunks;  // values of a lane; 16-byte chunks
          uint8_t* mine_q = my_q + quarter * 32 * kD;
          auto room = [&](int r, int c) {
            return reinterpret_cast<uint4*>(mine_q + (c >= kChunks / 2 ? Shape::kQTerm : 0) + r * kD + c % (kChunks / 2) * 16);
          };
          auto from_of = [&](int r) { return a.q + __shfl_sync(0xffffffffu, from_q, r & 31) + lane % kChunks * 8; };
          if (t.q_wide) {
#pragma unroll 8
            for (int base = 0; base < here; base += kRows) {
              const int r = base + lane / kChunks;
              const __nv_bfloat16* src = from_of(r);
              if (r < here) *room(r, lane % kChunks) = __ldg(reinterpret_cast<const uint4*>(src));
            }
          } else {
#pragma unroll 1
            for (int base = 0; base < here; base += kRows) {
              const int r = base + lane / kChunks;
              const __nv_bfloat16* src = from_of(r);
              if (r < here) *room(r, lane % kChunks) = load_narrow(src);
            }
          }
          __syncwarp();
#pragma unroll 1
          for (int base = 0; base < here; base += 4) {
            const int r = base + (lane >> 3), j = lane & 7;
            uint32_t raw[kPer / 2];
            __nv_bfloat162 top2 = __floats2bfloat162_rn(0.f, 0.f);  // NaN is passed over
#pragma unroll
            for (int c = 0; c < kPer / 8; ++c) {
              const uint4 v = r < here ? *room(r, j * (kPer / 8) + c) : make_uint4(0u, 0u, 0u, 0u);
              raw[4 * c] = v.x, raw[4 * c + 1] = v.y, raw[4 * c + 2] = v.z, raw[4 * c + 3] = v.w;
            }
#pragma unroll
            for (int k = 0; k < kPer / 2; ++k)
              top2 = __hmax2(top2, __habs2(*reinterpret_cast<const __nv_bfloat162*>(raw + k)));
            const uint32_t both = *reinterpret_cast<const uint32_t*>(&top2);
            uint32_t most = max(both & 0xffffu, both >> 16) << 16;  // as fp32 bits
            if (most >= 0x7f800000u) {  // an infinite q makes its whole row NaN
              most = 0u;
#pragma unroll
              for (int k = 0; k < kPer / 2; ++k) {
                const uint32_t lo16 = raw[k] & 0x7fffu, hi16 = raw[k] >> 16 & 0x7fffu;
                if (lo16 < 0x7f80u) most = max(most, lo16 << 16); else raw[k] |= 0x7fffu;
                if (hi16 < 0x7f80u) most = max(most, hi16 << 16); else raw[k] |= 0x7fff0000u;
              }
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int byte = scale_byte(most);
            const float inv1 = exp2_int(127 - byte);
            const f32x2 inv = pack2(inv1, inv1);
            uint32_t hi4[kPer / 4], lo4[kPer / 4];
#pragma unroll
            for (int k = 0; k < kPer / 2; ++k) {
              const f32x2 v = mul2(pack2(bf_lo(raw[k]), bf_hi(raw[k])), inv);
              const uint32_t h2 = __nv_cvt_float2_to_fp8x2(unpack2(v), __NV_SATFINITE, __NV_E4M3);
              const float2 back = e4m3x2_to_f32(h2);
              const f32x2 rest = fma2(pack2(back.x, back.y), pack2(-1.f, -1.f), v);
              const uint32_t low = __nv_cvt_float2_to_fp8x2(unpack2(rest), __NV_SATFINITE, __NV_E4M3);
              hi4[k / 2] = k % 2 ? hi4[k / 2] | h2 << 16 : h2;
              lo4[k / 2] = k % 2 ? lo4[k / 2] | low << 16 : low;
            }
            __syncwarp();  // the rows have been read: their room takes the terms
            if constexpr (kD == 128) {
              uint8_t* to = mine_q + r * kD + ((j ^ (r & 7)) << 4);
              *reinterpret_cast<uint4*>(to) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
              *reinterpret_cast<uint4*>(to + Shape::kQTerm) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
            } else {
              uint8_t* to = mine_q + r * kD + (((j >> 1) ^ ((r >> 1) & 3)) << 4) + (j & 1) * 8;
              *reinterpret_cast<uint2*>(to) = make_uint2(hi4[0], hi4[1]);
              *reinterpret_cast<uint2*>(to + Shape::kQTerm) = make_uint2(lo4[0], lo4[1]);
            }
            if (j == 0) s_qf[w * AP_TILE + quarter * 32 + r] = exp2_int(byte - 127) * a.scale_log2;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full + w);
        }
        const float qf = s_qf[w * AP_TILE + row];

#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
          const int j = first + (two ? i : 2 * i);  // tile of the piece
          const int tile = count + j, ring = tile % AP_RING, vs = tile & 1;
          if (here > 0) wait(kf_full + ring, (uint32_t)(tile / AP_RING) & 1u);
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {
            const int key0 = piece0 + j * AP_TILE + hf * AP_HALF;
            const uint32_t t_s = lanes + w * AP_TILE + hf * AP_HALF;
            const float* kf = s_kf + ring * 8 + hf * 4;
            // A score times f(16 tokens) is its exponent of 2; finite, so that a score of 0 stays 0
            float f[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              f[c] = qf * kf[c];
              if (fabsf(f[c]) == INFINITY) f[c] = copysignf(0x1p127f, f[c]);
            }
            wait(s_full + 2 * w + hf, s_phase);
            tc_fence_after();
            if (here > 0) {
              const bool sees = hi >= key0 && lo < key0 + AP_HALF && hi >= lo && row < live;
              // the exponents, and the largest; where it is too far above the reference, that moves
              f32x2 x[32];
              {
                uint32_t v[2][32];
                tmem_ld_x32(t_s, v[0]);
                tmem_ld_x32(t_s + 32, v[1]);
                tmem_wait_ld(v[0]);
                tmem_wait_ld(v[1]);
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  x[e] = mul2(pack2(__uint_as_float(v[e / 16][2 * e % 32]), __uint_as_float(v[e / 16][2 * e % 32 + 1])),
                              pack2(f[e / 8], f[e / 8]));
              }
              if (!__all_sync(0xffffffffu, lo <= key0 && hi >= key0 + AP_HALF - 1) || s_bad[ring] != 0) {
                // a bit for each token that the row sees; none of an invalid page
                const int from = max(lo - key0, 0), to = min(hi - key0, AP_HALF - 1);
                unsigned long long seen = to < from ? 0ull : (~0ull >> (AP_HALF - 1 - (to - from))) << from;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  if (kf[c] < 0.f) seen &= ~(0xffffull << (16 * c));
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float2 y = unpack2(x[e]);
                  x[e] = pack2(seen >> (2 * e) & 1ull ? y.x : -INFINITY, seen >> (2 * e + 1) & 1ull ? y.y : -INFINITY);
                }
              }
              const float* ve = s_ve + ring * 8 + hf * 4;
              float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int e = 0; e < 32; ++e) top[e / 8] = max3(top[e / 8], unpack2(x[e]).x, unpack2(x[e]).y);
              const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
              const float high_v = fmaxf(fmaxf(top[0] + ve[0], top[1] + ve[1]), fmaxf(top[2] + ve[2], top[3] + ve[3]));
              float less[4];  // e - m of 16 tokens each
              auto set = [&] {
                const float m = M == AT_NONE ? 0.f : M, n = N == AT_NONE ? 0.f : N;
#pragma unroll
                for (int c = 0; c < 4; ++c) less[c] = fmaxf(ve[c] - m, -n - AP_FAR);
              };
              set();
              if (__any_sync(0xffffffffu, sees && (high_v > M + AP_ROOM || high > N + AP_ROOM))) {
                const float to = fmaxf(M, ceilf(high_v) - AP_HEAD), f = ex2_approx(M - to);
                const float to_sum = fmaxf(N, ceilf(high)), f_sum = ex2_approx(N - to_sum);
                M = to;
                N = to_sum;
                set();
                l2[0] = mul2(l2[0], pack2(f_sum, f_sum));
                l2[1] = mul2(l2[1], pack2(f_sum, f_sum));
                if (i + hf > 0 && __any_sync(0xffffffffu, f != 1.f)) {
                  // the products of the weights handed over last (those before are done: this
                  // half's scores were made after them)
                  wait(pv_done + 2 * w + (hf ^ 1), s_phase ^ (uint32_t)(hf ^ 1));
                  tc_fence_after();
#pragma unroll 1
                  for (int c = 0; c < kD; c += 16) {
                    uint32_t o[16];
                    tmem_ld_x16(t_o + c, o);
                    tmem_wait_ld(o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_st_x16(t_o + c, o);
                  }
                  tmem_wait_st();
                }
              }
              const float n = N == AT_NONE ? 0.f : N;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float to_m = less[2 * c + e / 8], of_sum = ex2_approx(-to_m - n);
                  const float2 y = unpack2(add2(x[c * 16 + e], pack2(to_m, to_m)));
                  const float2 z = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                  l2[e & 1] = fma2(pack2(z.x, z.y), pack2(of_sum, of_sum), l2[e & 1]);
                  const __half2 z16 = __floats2half2_rn(z.x, z.y);
                  p[e] = *reinterpret_cast<const uint32_t*>(&z16);
                }
                tmem_st_x16(t_s + c * 16, p);  // over scores that have been read
              }
              tmem_wait_st();
              if (hf == 0) wait(v_full + vs, (uint32_t)(tile >> 1) & 1u);
              const int4 flags = *reinterpret_cast<const int4*>(s_has_nan + 4 * vs);
              if (flags.x == tile + 1 || flags.y == tile + 1 || flags.z == tile + 1 || flags.w == tile + 1) {
                for (int k = max(lo - key0, 0); k <= min(hi - key0, AP_HALF - 1); ++k) {
                  const int r = hf * AP_HALF + k;
                  if (s_has_nan[4 * vs + (kUnits == 8 ? r >> 2 & 3 : r >> 3 & 3)] != tile + 1) continue;
                  const uint16_t* bits = s_nan + (vs * AP_TILE + r) * kUnits;
#pragma unroll
                  for (int u = 0; u < kUnits; ++u) poison[u / 2] |= (uint32_t)bits[u] << (16 * (u & 1));
                }
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 2 * w + hf);
          }
          s_phase ^= 1u;
        }
        // ---- the piece's O, reference and sum to its slot --------------------------
        const int slot_rows = own ? t.own_rows : AP_TILE;
        const size_t at = 2 * ((size_t)blockIdx.x + (own ? walk.unit - work.units : walk.unit)) + w;
        float* slot = own ? t.own_slots + at * t.own_slot : t.slots + at * (AP_TILE * (kD + 4));
        if (row < live) {
          const float2 la = unpack2(add2(l2[0], l2[1]));
          __stcg(reinterpret_cast<float4*>(slot + slot_rows * kD) + row, make_float4(M, la.x + la.y, N, 0.f));
        }
        if (mine > 0 && here > 0) {
          wait(pv_done + 2 * w, s_phase ^ 1u);
          wait(pv_done + 2 * w + 1, s_phase ^ 1u);
          tc_fence_after();
          float4* to = reinterpret_cast<float4*>(slot) + row;
#pragma unroll 2
          for (int c = 0; c < kD; c += 32) {
            uint32_t o[32];
            tmem_ld_x32(t_o + c, o);
            uint32_t bad = 0u;
#pragma unroll
            for (int k = 0; k < kD / 32; ++k) bad = c == 32 * k ? poison[k] : bad;
            tmem_wait_ld(o);
            if (__any_sync(0xffffffffu, bad)) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = bad >> e & 1u ? 0x7fc00000u : o[e];
            }
#pragma unroll
            for (int e = 0; e < 32; e += 4, to += slot_rows)
              if (row < live)
                __stcg(to, make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                       __uint_as_float(o[e + 3])));
          }
          tc_fence_before();
        }
        __syncwarp();
        count += n;
      }
      walk_on(t, work, walk);
    }
  } else if (warp < AP_WARP_LOAD) {
    // ---- V's codes as fp16 ------------------------------------------------------
    // Lane pairs of eight take half of two neighbouring rows each, so that a
    // quarter warp's loads and swizzled stores lie in eight different banks' groups.
    const int id = tid - AP_WARP_V * 32;
    constexpr int kPass = 128 / kUnits;  // rows of a pass
    const int pass_row = kUnits == 8 ? (id >> 4) * 2 + ((id >> 2) & 1) : id >> 2;
    const int u = kUnits == 8 ? (id & 3) | ((((id >> 2) & 1) ^ ((id >> 3) & 1)) << 2) : id & 3;
    int tile = 0;
    uint32_t used = 0, uses = 0;  // of the stages (2 bits each): by which groups, and their phases
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(walk, &j0, &n);
      const bool two = two_of(walk);
      for (int j = 0; j < n; ++j, ++tile) {
        const int vs = tile & 1, live = walk.limit - walk.key0 - (j0 + j) * AP_TILE;  // rows that count
        wait(r_full + vs, (uint32_t)(tile >> 1) & 1u);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t bit = 1u << (2 * vs + w);
          if (used & bit) {
            wait(v_empty + 2 * w + vs, uses & bit ? 1u : 0u);
            uses ^= bit;
          }
        }
        used = (used & ~(3u << (2 * vs))) | (two ? 3u : 1u << (tile & 1)) << (2 * vs);
        const int* scales = s_vb + tile % AP_RING * 8;
        const uint8_t* src = s_raw + vs * Shape::kKBytes + u * 16;
        uint8_t* dst = s_v + vs * Shape::kVBytes + (u >> 2) * (AP_TILE * 128);
        const int c = 2 * (u & 3);
        bool odd = false;
#pragma unroll 1
        for (int i0 = 0; i0 < kUnits; i0 += 4) {
        uint4 raw[4];
        int sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (i0 + i) * kPass + pass_row;
          raw[i] = *reinterpret_cast<const uint4*>(src + r * kD);
          sc[i] = scales[r >> 4];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (i0 + i) * kPass + pass_row;
          if (r >= live || sc[i] < 0) raw[i] = make_uint4(0u, 0u, 0u, 0u), sc[i] = 0;
          uint32_t b[8];
          odd |= e4m3x16_to_f16(raw[i], b) || sc[i] == 255;
          uint8_t* at = dst + r * 128;
          *reinterpret_cast<uint4*>(at + ((c ^ (r & 7)) << 4)) = make_uint4(b[0], b[1], b[2], b[3]);
          *reinterpret_cast<uint4*>(at + (((c + 1) ^ (r & 7)) << 4)) = make_uint4(b[4], b[5], b[6], b[7]);
        }
        }
        if (__any_sync(0xffffffffu, odd)) {
          // once more with care: NaN values are taken out and noted, for 0 times NaN would
          // reach rows that do not see them
          if (lane == 0) s_has_nan[4 * vs + warp - AP_WARP_V] = tile + 1;
#pragma unroll 1
          for (int i = 0; i < kUnits; ++i) {
            const int r = i * kPass + pass_row, s = r < live ? scales[r >> 4] : -1;
            const uint4 codes = *reinterpret_cast<const uint4*>(src + r * kD);
            uint32_t x[4] = {codes.x, codes.y, codes.z, codes.w}, b[8], mask = s == 255 ? 0xffffu : 0u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (s < 0 || s == 255) x[e] = 0u;
              const uint32_t m = ((x[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bit 7 of each NaN's byte
              x[e] &= ~((m >> 7) * 0xffu);
              mask |= ((m >> 7 & 1u) | (m >> 14 & 2u) | (m >> 21 & 4u) | (m >> 28 & 8u)) << (4 * e);
            }
            e4m3x16_to_f16(make_uint4(x[0], x[1], x[2], x[3]), b);
            s_nan[(vs * AP_TILE + r) * kUnits + u] = (uint16_t)mask;
            uint8_t* at = dst + r * 128;
            *reinterpret_cast<uint4*>(at + ((c ^ (r & 7)) << 4)) = make_uint4(b[0], b[1], b[2], b[3]);
            *reinterpret_cast<uint4*>(at + (((c + 1) ^ (r & 7)) << 4)) = make_uint4(b[4], b[5], b[6], b[7]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(v_full + vs);
          mbar_arrive(r_empty + vs);
        }
      }
      walk_on(t, work, walk);
    }
  } else if (warp == AP_WARP_LOAD) {
    // ---- pages of K and V, and their scales ------------------------------------
    const int per_tile = AP_TILE >> t.page_shift;
    const uint64_t policy = l2_policy_evict_first();
    int tile = 0, stage = 0;
    uint32_t used = 0, uses = 0;  // of the stages of K (2 bits each): by which groups, and their phases
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(walk, &j0, &n);
      const bool two = two_of(walk);
      const int32_t* table = a.table + (size_t)(walk.b >= 0 ? walk.b : lead) * a.table_stride;
      // pages of 32 columns at a time, one batch ahead
      const int c0 = (walk.key0 >> t.page_shift) + j0 * per_tile;
      const int stop = min(c0 + n * per_tile, (walk.limit + (1 << t.page_shift) - 1) >> t.page_shift);
      const int begin = walk.b >= 0 ? c0 : work.first >> t.page_shift;  // pages before it no row sees
      auto page_at = [&](int col) {
        const int pid = col >= begin && col < stop ? __ldg(table + col) : -1;
        return pid >= 0 && pid < a.pages ? pid : -1;
      };
      int batch = c0, at_lane = 0;
      int pid = page_at(batch + lane), pid_next = page_at(batch + 32 + lane);
      int kb = 0, vb = -1;
      if (pid >= 0) {
        kb = __ldg(a.ks + (size_t)pid * a.Hkv + walk.h);
        vb = __ldg(a.vs + (size_t)pid * a.Hkv + walk.h);
      }
      for (int j = 0; j < n; ++j, ++tile) {
        if (at_lane == 32) {
          at_lane = 0;
          batch += 32;
          pid = pid_next;
          kb = 0, vb = -1;
          if (pid >= 0) {
            kb = __ldg(a.ks + (size_t)pid * a.Hkv + walk.h);
            vb = __ldg(a.vs + (size_t)pid * a.Hkv + walk.h);
          }
          pid_next = page_at(batch + 32 + lane);
        }
        const int col = batch + lane, ring = tile % AP_RING, rs = tile & 1;
        const bool mine = lane >= at_lane && lane < at_lane + per_tile, needed = mine && col >= begin && col < stop;
        const uint32_t bad = __ballot_sync(0xffffffffu, needed && pid < 0);
        const uint32_t there = __ballot_sync(0xffffffffu, needed && pid >= 0);
        const uint32_t bytes = __popc(there) * (uint32_t)(kD << t.page_shift);
        // of pages that no row sees: another's of the tile, so that references stay near
        const int vb_there = __shfl_sync(0xffffffffu, vb, there ? __ffs(there) - 1 : 0);
        if (bad && lane == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
        const int row = needed && pid >= 0 ? (pid * a.Hkv + walk.h) << t.page_shift : -1;
        auto issue = [&](uint8_t* to, const CUtensorMap* map, uint64_t* bar) {
          if (lane == 0) mbar_expect_tx(bar, bytes);
          __syncwarp();
#pragma unroll 1
          for (int p = 0; p < per_tile; ++p) {
            const int at = __shfl_sync(0xffffffffu, row, at_lane + p);
            if (at >= 0 && elect_one()) tma_load_2d(to + (p << t.page_shift) * kD, map, 0, at, bar, policy);
          }
          __syncwarp();
        };
        bool ok = true;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t bit = 1u << (2 * stage + w);
          if (used & bit) {
            ok = wait(k_empty + AP_K_STAGES * w + stage, uses & bit ? 1u : 0u) && ok;
            uses ^= bit;
          }
        }
        used = (used & ~(3u << (2 * stage))) | (two ? 3u : 1u << (tile & 1)) << (2 * stage);
        if (__all_sync(0xffffffffu, ok)) {
          issue(s_k + stage * Shape::kKBytes, &tm_k, k_full + stage);
          // tokens past the last are masked by their number
          const float f = needed && pid < 0 ? -1.f : ue8m0_to_f32((uint32_t)kb);
          const int each = 8 / per_tile;  // groups of 16 tokens of a page
          if (mine) {
            for (int e = 0; e < each; ++e) {
              s_kf[ring * 8 + (lane - at_lane) * each + e] = f;
              s_ve[ring * 8 + (lane - at_lane) * each + e] = (float)((row >= 0 ? vb : there ? vb_there : 127) - 127);
              s_vb[ring * 8 + (lane - at_lane) * each + e] = row >= 0 ? vb : -1;
            }
          }
          if (lane == 0) s_bad[ring] = bad != 0u;
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(k_full + stage);
            mbar_arrive(kf_full + ring);
          }
        }
        if (__all_sync(0xffffffffu, wait(r_empty + rs, ((uint32_t)(tile >> 1) & 1u) ^ 1u))) {
          issue(s_raw + rs * Shape::kKBytes, &tm_v, r_full + rs);
          if (lane == 0) mbar_arrive(r_full + rs);
        }
        __syncwarp();
        at_lane += per_tile;
        if (++stage == AP_K_STAGES) stage = 0;
      }
      walk_on(t, work, walk);
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0) {
      for (int i = max(0, tile - AP_K_STAGES); i < tile; ++i)
        mbar_wait(k_full + i % AP_K_STAGES, (uint32_t)(i / AP_K_STAGES) & 1u);
      for (int i = max(0, tile - 2); i < tile; ++i) mbar_wait(r_full + (i & 1), (uint32_t)(i >> 1) & 1u);
    }
    __syncwarp();
  } else if (warp < AP_WARP_MMA + 2) {
    // ---- products of a group -----------------------------------------------------
    constexpr uint32_t kIdS = tc_idesc_e4m3(AP_TILE, AP_HALF, false, false);
    constexpr uint32_t kIdO = tc_idesc_f16(AP_TILE, kD) | 1u << 16;  // V lies with its values side by side
    const int w = warp - AP_WARP_MMA;
    // (elect_one names the same thread every time: a commit covers what its own thread issued)
    const uint64_t d_q = tc_desc(smem_u32(s_q) + w * 2 * Shape::kQTerm, 16, kAtom, kSwz);
    const uint64_t d_k = tc_desc(smem_u32(s_k), 16, kAtom, kSwz);
    const uint64_t d_v = tc_desc(smem_u32(s_v), AP_TILE * 128, 1024, 2);
    const uint32_t t_s = tmem + w * AP_TILE, t_o = tmem + 2 * AP_TILE + w * kD;
    int count = 0;
    uint32_t q_phase = 0, p_phase = 0;
    while (walk.pos < walk.end) {
      int j0, n;
      walk_piece(walk, &j0, &n);
      if (n > 0) {
        const bool two = two_of(walk);
        const int first = first_of(two, count, w), mine = tiles_of(two, n, first), step = two ? 1 : 2;
        if (mine > 0) {
          bool ok = wait(q_full + w, q_phase);
          q_phase ^= 1u;
          // of each half in turn: values of tile i, then scores of the next, in their place
#pragma unroll 1
          for (int x = -2; x < 2 * mine; ++x) {
            const int hf = x & 1, tile = count + first + (x >> 1) * step, next = tile + step;
            if (x >= 0) {
              const int vs = tile & 1;
              ok = wait(p_full + 2 * w + hf, p_phase) && ok;
              if (hf == 0) ok = wait(v_full + vs, (uint32_t)(tile >> 1) & 1u) && ok;
              tc_fence_after();
              if (__all_sync(0xffffffffu, ok) && elect_one()) {
                const uint64_t v = d_v + (uint32_t)((vs * Shape::kVBytes + hf * AP_HALF * 128) / 16);
#pragma unroll 2
                for (int s = 0; s < AP_HALF / 16; ++s)
                  tc_mma_f16_ts(t_o, t_s + hf * AP_HALF + 8 * s, v + s * 128, kIdO, x + s > 0);
                tc_commit(pv_done + 2 * w + hf);
                if (hf == 1) tc_commit(v_empty + 2 * w + vs);
              }
              __syncwarp();
              if (hf == 1) p_phase ^= 1u;
            }
            if (x + 2 < 2 * mine) {
              const int stage = next % AP_K_STAGES;
              if (hf == 0) ok = wait(k_full + stage, (uint32_t)(next / AP_K_STAGES) & 1u) && ok;
              tc_fence_after();
              if (__all_sync(0xffffffffu, ok) && elect_one()) {
                const uint64_t k = d_k + (uint32_t)((stage * Shape::kKBytes + hf * AP_HALF * kD) / 16);
#pragma unroll 1
                for (int term = 0; term < 2; ++term)
#pragma unroll 2
                  for (int s = 0; s < kD / 32; ++s)
                    tc_mma_f8(t_s + hf * AP_HALF, d_q + term * (Shape::kQTerm / 16) + 2 * s, k + 2 * s, kIdS, term + s > 0);
                tc_commit(s_full + 2 * w + hf);
                if (hf == 1) tc_commit(k_empty + AP_K_STAGES * w + stage);
              }
              __syncwarp();
            }
          }
        }
        count += n;
      }
      walk_on(t, work, walk);
    }
    // After an abort let what was issued end before TMEM is freed.
    __syncwarp();
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained + w);
      mbar_wait(drained + w, 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == AP_WARP_MMA) tmem_dealloc(tmem, 512);
}

// Joins the parts: a thread four values of a row, a block 32 rows of a key head by 32
// values.  Rows are those of the prefix's units, in their order.
template <int kD>
__global__ void __launch_bounds__(256) attn_prefix_join_kernel(const AttnPrefixArgs t) {
  const AttnArgs& a = t.a;
  pdl_wait_primary();
  const AttnPrefixPlan plan = *reinterpret_cast<const AttnPrefixPlan*>(t.plan);
  const int lane = threadIdx.x & 31, quad = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int G = a.Hq / a.Hkv, rows = a.B * a.Sq * G, per_head = (rows + 31) / 32;
  const int h = blockIdx.x / per_head, rr = (blockIdx.x - h * per_head) * 32 + lane;
  if (rr >= rows) return;
  AttnShares shares;
  shares.each = plan.each, shares.more = plan.more;
  const int b = rr / (a.Sq * G), r_own = rr - b * a.Sq * G;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float M = AT_NONE, N = AT_NONE, sum = 0.f;
  // Pieces [0, pieces) of a unit in consecutive slots from `slot0` on.
  auto add = [&](const float* slot0, size_t stride, int pieces, int slot_rows, int row) {
    constexpr int kBatch = 4;
    for (int p0 = 0; p0 < pieces; p0 += kBatch) {
      float4 stats[kBatch], v[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const float* s = slot0 + min(p0 + e, pieces - 1) * stride;
        stats[e] = __ldcg(reinterpret_cast<const float4*>(s + slot_rows * kD) + row);
        v[e] = __ldcg(reinterpret_cast<const float4*>(s) + quad * slot_rows + row);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const float m = stats[e].x, l = stats[e].y, n = stats[e].z;
        if (p0 + e >= pieces || (n == AT_NONE && l == 0.f)) continue;  // no token seen: O may be anything
        const float to_sum = fmaxf(N, n), to = fmaxf(M, m), f = ex2_approx(M - to), w = ex2_approx(m - to);
        sum = fmaf(l, ex2_approx(n - to_sum), sum * ex2_approx(N - to_sum));
        M = to;
        N = to_sum;
        y.x = fmaf(v[e].x, w, y.x * f), y.y = fmaf(v[e].y, w, y.y * f);
        y.z = fmaf(v[e].z, w, y.z * f), y.w = fmaf(v[e].w, w, y.w * f);
      }
    }
  };
  if (plan.tiles > 0) {
    const int block = rr / (AP_TILE << t.two), unit = h * t.row_blocks + block, tile = rr / AP_TILE & 1;
    const int base = unit * (AP_UNIT_COST + (plan.tiles << t.two)) + AP_UNIT_COST;
    const int ca = shares.cta_of(base), cz = shares.cta_of(base + ((plan.tiles - 1) << t.two));
    const size_t slot = (size_t)AP_TILE * (kD + 4);
    const float* s = t.slots + 2 * (size_t)(ca + unit) * slot;
    if (t.two)
      add(s + tile * slot, 2 * slot, cz - ca + 1, AP_TILE, rr % AP_TILE);
    else
      add(s, slot, 2 * (cz - ca + 1), AP_TILE, rr % AP_TILE);
  }
  int key0;
  const int tiles = own_tiles(t, attn_length(a, b), plan.from, &key0);
  if (tiles > 0) {
    const int block = r_own / AP_TILE, k = h * t.own_blocks + block;
    const int base = __ldg(t.own_start + b) + k * (AP_UNIT_COST + tiles) + AP_UNIT_COST;
    const int ca = shares.cta_of(base), cz = shares.cta_of(base + tiles - 1);
    const size_t slot = (size_t)t.own_slot;
    add(t.own_slots + 2 * (size_t)(ca + b * a.Hkv * t.own_blocks + k) * slot, slot, 2 * (cz - ca + 1), t.own_rows,
        r_own - block * AP_TILE);
  }
  const size_t at = (size_t)(rr / G) * a.Hq + h * G + rr % G;  // row of the output
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  const float half = floorf(0.5f * (M - N)), f1 = ex2_approx(half), f2 = ex2_approx(M - N - half);  // both finite
  auto value = [&](float v) { return v * f * f1 * f2; };
  *reinterpret_cast<uint2*>(a.out + at * kD + 4 * quad) =
      make_uint2(pack_bf16(value(y.x), value(y.y)), pack_bf16(value(y.z), value(y.w)));
  if (a.lse && quad == 0) a.lse[at] = sum == 0.f ? -INFINITY : N * 0.6931471805599453f + logf(sum);
}

}  // namespace wdb

// Attention of all sequences of a batch over the tokens that they share, on the
// FP8 paged cache (head sizes 64 and 128), sm_100a; each sequence's own tokens
// are attended by wd_attn_fp8_tc.cuh, and attn_prefix_join_kernel joins both.
//
// With O = sum 2^(x - m) v, l = sum 2^(x - m) over any set of tokens, two sets join
// as O = O1 2^(m1 - M) + O2 2^(m2 - M), l likewise, M = max(m1, m2): the prefix is
// one set, cut further over the CTAs.
//
// The rows of a key head, those of all its sequences' query tokens and heads, are
// the M side of the products: 128 rows a tile, two tiles at once.
// * S = q K^T: K's codes straight from the cache through TMA (kind::f8f6f4), q as
//   two E4M3 terms (hi = the nearest, lo = the nearest to what remains) that are
//   products of one sum; exact for ten octaves below a row's largest value, and
//   within 2^-18 of it below. The page's scale of K, a power of two, is a factor
//   of the exponent.
// * O += P V in bf16: P as it is held in TMEM, in the place of the scores it was
//   made of; V widened to bf16 with its page's scale, exactly, by four warps once
//   for both row tiles. A weight is rounded to bf16, within 2^-9 of itself
//   whatever its size; sums are of the weights before that, in fp32.
// * A row is a thread's: no sums or maxima across threads. References (the m above)
//   are lazy: they move when a weight would pass 2^AP_ROOM, and O is then
//   rescaled in TMEM.
//
// Warps: two groups of four for the softmax of a row tile each, in turn with the
// tensor core (it works on one tile while the other's weights are made), four that
// widen V, one that loads K, one that issues the products.  With at most 128 rows
// a key head both groups take the same rows, and every second tile of tokens.
//
// Work: the token tiles of all (key head, 256 rows) units in one line, cut into
// equal shares, one a CTA.
#pragma once

#include "wd_attn_fp8_tc.cuh"

namespace wdb {

constexpr int AP_TILE = 128;       // tokens of a tile, rows of a row tile
constexpr int AP_THREADS = 512;    // softmax 2 x 128, V 128, loads, products, two idle warps
constexpr int AP_WARP_V = 8, AP_WARP_LOAD = 12, AP_WARP_MMA = 13;
// Registers of a thread: 512 x 128 are launched, and these add up to them.
constexpr int AP_REGS_SOFTMAX = 144, AP_REGS_V = 112, AP_REGS_REST = 112;
static_assert(2 * AP_REGS_SOFTMAX + AP_REGS_V + AP_REGS_REST == 4 * 128, "register split");
constexpr int AP_K_STAGES = 3;
constexpr int AP_RING = 8;         // scales of pages, kept until the softmax has used them
constexpr float AP_ROOM = 16.f;    // log2 of the largest weight before a reference moves
constexpr int AP_HEADER = 256;     // bytes at the workspace's start: the plan, for the join

template <int kD>
struct AttnPrefixShape {
  static constexpr int kQTerm = AP_TILE * kD;        // bytes of a term of a row tile's q
  static constexpr int kKBytes = AP_TILE * kD;
  static constexpr int kVBytes = 2 * AP_TILE * kD;   // bf16
  static constexpr int kUnits = kD / 16;             // 16-byte units of a cached row
  static constexpr int kOffK = 4 * kQTerm;
  static constexpr int kOffRaw = kOffK + AP_K_STAGES * kKBytes;  // two tiles of V as it is cached
  static constexpr int kOffV = kOffRaw + 2 * kKBytes;
  static constexpr int kOffMisc = kOffV + 2 * kVBytes;
  static constexpr int kMiscBytes = 2 * AP_TILE * kUnits * 2 + 2 * AP_TILE * 4 + (2 * AP_RING + 1) * 8 * 4 + 512;
  static constexpr int kSmem = kOffMisc + kMiscBytes + 1024;  // + alignment slack
  static constexpr int kSlotFloats = AP_TILE * (kD + 2);      // O [D/4][128][4], references, sums
};

struct AttnPrefixArgs {
  AttnArgs a;
  const int32_t* prefix;  // tokens that all sequences share
  uint8_t* plan;          // AP_HEADER bytes
  float* slots;
  int row_blocks;         // of a key head
  int reach;              // tokens that the block table can address
  int page_shift;
  int q_wide;
};

// The plan of a call, as the prefix kernel's CTAs find it and leave it to the join.
struct AttnPrefixPlan {
  int tile0, tiles;  // tiles of tokens that some row sees
  int each, more;    // AttnShares
};

__device__ __forceinline__ void tc_mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
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

// kTwo: a unit has two row tiles; else one, and the groups take tiles of tokens in turn.
// Ties the 32 values to the wait for them.
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

template <int kRegs>
__device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int kD, bool kTwo>
__global__ void __launch_bounds__(AP_THREADS, 1)
    attn_prefix_kernel(const AttnPrefixArgs t, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v) {
  using Shape = AttnPrefixShape<kD>;
  constexpr uint32_t kSwz = kD == 128 ? 2u : 4u;
  constexpr uint32_t kAtom = kD == 128 ? 1024u : 512u;
  constexpr int kUnits = Shape::kUnits;
  const AttnArgs& a = t.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.Hkv, rows = a.B * a.Sq * G;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                 // [2 row tiles][hi, lo]
  uint8_t* s_k = smem + Shape::kOffK;  // [stages]
  uint8_t* s_raw = smem + Shape::kOffRaw;  // [2][128][D] codes of V
  uint8_t* s_v = smem + Shape::kOffV;  // [2][D / 64][128][64]
  uint16_t* s_nan = reinterpret_cast<uint16_t*>(smem + Shape::kOffMisc);  // [2][128][units]: values that are NaN
  float* s_qf = reinterpret_cast<float*>(s_nan + 2 * AP_TILE * kUnits);   // [2][128]
  float* s_kf = s_qf + 2 * AP_TILE;    // [ring][8]: factor of 16 tokens each, -1 where their page is invalid
  int* s_vb = reinterpret_cast<int*>(s_kf + AP_RING * 8);  // [ring][8]: scale byte of V of 16 tokens each, or -1
  float* s_one = reinterpret_cast<float*>(s_vb + AP_RING * 8);  // [8]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_one + 8);
  uint64_t *k_full = bars, *k_empty = bars + AP_K_STAGES, *kf_full = bars + 2 * AP_K_STAGES;
  uint64_t* r_full = kf_full + AP_RING;  // [2]
  uint64_t* r_empty = r_full + 2;        // [2]
  uint64_t* v_full = r_full + 4;         // [2]
  uint64_t* v_empty = v_full + 2;        // [2]
  uint64_t* q_full = v_full + 4;         // [2]
  uint64_t* s_full = v_full + 6;         // [2]
  uint64_t* p_full = v_full + 8;         // [2]
  uint64_t* o_full = v_full + 10;        // [2]
  uint64_t* drained = v_full + 12;
  int* s_has_nan = reinterpret_cast<int*>(v_full + 13);  // [2] 1 + the last tile of the stage with a NaN value
  int* s_bad = s_has_nan + 2;                            // [ring] some page of the tile is invalid
  volatile int* s_abort = s_bad + AP_RING;
  uint32_t* s_tmem = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(s_abort + 1));
  int* s_plan = reinterpret_cast<int*>(s_tmem + 1);      // longest sequence and its length, shortest
  static_assert(8 * (2 * AP_K_STAGES + AP_RING + 17) + 4 * (2 + AP_RING + 2 + 3) <= 512, "small arrays");

  if (warp == AP_WARP_LOAD && lane == 0) {
    *s_abort = 0;
    for (int i = 0; i < AP_K_STAGES; ++i) mbar_init(k_full + i, 1), mbar_init(k_empty + i, 1);
    for (int i = 0; i < AP_RING; ++i) mbar_init(kf_full + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(v_full + i, 4), mbar_init(v_empty + i, 1), mbar_init(q_full + i, 4);
      mbar_init(s_full + i, 1), mbar_init(p_full + i, 4), mbar_init(o_full + i, 1);
      mbar_init(r_full + i, 1), mbar_init(r_empty + i, 4);
      s_has_nan[i] = 0;
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    for (int i = 0; i < 8; ++i) s_one[i] = 1.f;
  } else if (warp == AP_WARP_MMA) {
    tmem_alloc(s_tmem, 512);
    tmem_relinquish();
    tc_fence_before();
  } else if (warp == 0) {
    // the longest sequence (the first of them), whose table shows the prefix's pages
    int most = -1, at = 0, least = 0x7fffffff;
    for (int b = lane; b < a.B; b += 32) {
      const int n = attn_length(a, b);
      if (n > most) most = n, at = b;
      if (n > 0) least = min(least, n);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int n = __shfl_xor_sync(0xffffffffu, most, o), b = __shfl_xor_sync(0xffffffffu, at, o);
      if (n > most || (n == most && b < at)) most = n, at = b;
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    if (lane == 0) s_plan[0] = at, s_plan[1] = most, s_plan[2] = least;
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // tokens [0, shared) that count, tiles of them, and this CTA's share of all units' tiles
  const int lead = s_plan[0];
  const int shared = min(prefix_tokens(t.prefix, t.reach, t.page_shift), s_plan[1]);
  AttnPrefixPlan plan;
  plan.tile0 = attn_first(max(s_plan[2] - a.Sq, 0), a.window) / AP_TILE;
  plan.tiles = max((shared + AP_TILE - 1) / AP_TILE - plan.tile0, 0);
  const int units = a.Hkv * t.row_blocks;
  const int total = units * plan.tiles;
  const int ctas = min((int)gridDim.x, max(1, total / 2));
  AttnShares shares;
  shares.each = plan.each = total / ctas;
  shares.more = plan.more = total - plan.each * ctas;
  const bool idle = (int)blockIdx.x >= ctas;
  const int begin = idle ? 0 : shares.first(blockIdx.x), end = idle ? 0 : shares.first(blockIdx.x + 1);
  if (blockIdx.x == 0 && tid == 0) *reinterpret_cast<AttnPrefixPlan*>(t.plan) = plan;

  // Bounded wait; once one gave up, none waits and nothing more is issued, but
  // every role still runs its loop to the end.
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
  // tiles of a piece of n that group w takes
  auto tiles_of = [](int n, int w) { return kTwo ? n : (n - w + 1) / 2; };

  if (warp < AP_WARP_V) {
    // ---- softmax: a row a thread ---------------------------------------------
    take_registers<AP_REGS_SOFTMAX>();
    const int w = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)quarter << 21);
    const uint32_t t_s = lanes + w * AP_TILE, t_o = lanes + 2 * AP_TILE + w * kD;
    uint8_t* my_q = s_q + w * 2 * Shape::kQTerm;
    int count = 0;             // tiles of this CTA before the piece
    uint32_t s_phase = 0, o_phase = 0;
    for (int pos = begin; pos < end;) {
      const int unit = pos / plan.tiles, j0 = pos - unit * plan.tiles, n = min(plan.tiles - j0, end - pos);
      const int h = unit / t.row_blocks, r0 = (unit - h * t.row_blocks) * (kTwo ? 2 * AP_TILE : AP_TILE) + (kTwo ? w * AP_TILE : 0);
      const int mine = tiles_of(n, w);
      // q of this warp's rows, eight lanes a row, as two terms
      {
        constexpr int kPer = kD / 8;  // values of a lane
#pragma unroll 2
        for (int base = 0; base < 32; base += 4) {
          const int r = quarter * 32 + base + (lane >> 3), j = lane & 7, rr = r0 + r;
          const int s = rr / G, g = rr - s * G, b = s / a.Sq, i = s - b * a.Sq;
          const __nv_bfloat16* src =
              a.q + (long long)b * a.q_bs + (long long)i * a.q_ts + (long long)(h * G + g) * a.q_hs + j * kPer;
          uint32_t raw[kPer / 2];
#pragma unroll
          for (int c = 0; c < kPer / 8; ++c) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (rr < rows) {
              if (t.q_wide) {
                v = __ldg(reinterpret_cast<const uint4*>(src) + c);
              } else {
                uint32_t e[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) e[k] = __bfloat16_as_ushort(src[c * 8 + k]);
                v = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
              }
            }
            raw[4 * c] = v.x, raw[4 * c + 1] = v.y, raw[4 * c + 2] = v.z, raw[4 * c + 3] = v.w;
          }
          uint32_t most = 0u;  // largest finite magnitude, as fp32 bits
          bool infinite = false;
#pragma unroll
          for (int k = 0; k < kPer / 2; ++k) {
            const uint32_t lo = raw[k] & 0x7fffu, hi = raw[k] >> 16 & 0x7fffu;
            if (lo < 0x7f80u) most = max(most, lo << 16); else infinite = true;
            if (hi < 0x7f80u) most = max(most, hi << 16); else infinite = true;
          }
          if (infinite) {  // an infinite q makes its whole row NaN
#pragma unroll
            for (int k = 0; k < kPer / 2; ++k) {
              if ((raw[k] & 0x7fffu) >= 0x7f80u) raw[k] |= 0x7fffu;
              if ((raw[k] >> 16 & 0x7fffu) >= 0x7f80u) raw[k] |= 0x7fff0000u;
            }
          }
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
          const int byte = scale_byte(most);
          const float inv1 = exp2_int(127 - byte);
          const f32x2 inv = pack2(inv1, inv1);
          uint32_t hi[kPer / 4], lo[kPer / 4];
#pragma unroll
          for (int k = 0; k < kPer / 2; ++k) {
            const f32x2 x = mul2(pack2(bf_lo(raw[k]), bf_hi(raw[k])), inv);
            const uint32_t h2 = __nv_cvt_float2_to_fp8x2(unpack2(x), __NV_SATFINITE, __NV_E4M3);
            const float2 back = e4m3x2_to_f32(h2);
            const f32x2 rest = fma2(pack2(back.x, back.y), pack2(-1.f, -1.f), x);
            const uint32_t l2 = __nv_cvt_float2_to_fp8x2(unpack2(rest), __NV_SATFINITE, __NV_E4M3);
            hi[k / 2] = k % 2 ? hi[k / 2] | h2 << 16 : h2;
            lo[k / 2] = k % 2 ? lo[k / 2] | l2 << 16 : l2;
          }
          if constexpr (kD == 128) {
            uint8_t* to = my_q + r * kD + ((j ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(to + Shape::kQTerm) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
            uint8_t* to = my_q + r * kD + (((j >> 1) ^ ((r >> 1) & 3)) << 4) + (j & 1) * 8;
            *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
            *reinterpret_cast<uint2*>(to + Shape::kQTerm) = make_uint2(lo[0], lo[1]);
          }
          if (j == 0) s_qf[w * AP_TILE + r] = exp2_int(byte - 127) * a.scale_log2;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full + w);
      }
      const float qf = s_qf[w * AP_TILE + row];
      // tokens that the row sees: [lo, hi]
      int lo = 0, hi = shared - 1;  // a row past the last: all, for no one
      if (r0 + row < rows) {
        const int s = (r0 + row) / G, b = s / a.Sq, last = attn_length(a, b) - a.Sq + (s - b * a.Sq);
        lo = attn_first(last, a.window);
        hi = min(last, shared - 1);
      }
      float M = AT_NONE;
      f32x2 l2[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)};
      uint32_t poison[kD / 32];
#pragma unroll
      for (int i = 0; i < kD / 32; ++i) poison[i] = 0u;

      for (int i = 0; i < mine; ++i) {
        const int j = kTwo ? i : 2 * i + w;  // tile of the piece
        const int tile = count + j, ring = tile % AP_RING, vs = tile & 1;
        const int key0 = (plan.tile0 + j0 + j) * AP_TILE;
        wait(kf_full + ring, (uint32_t)(tile / AP_RING) & 1u);
        wait(s_full + w, s_phase);
        s_phase ^= 1u;
        tc_fence_after();
        const bool sees = hi >= key0 && lo < key0 + AP_TILE && hi >= lo;
        // A score times f(16 tokens) is its exponent of 2.
        const float* kf = s_kf + ring * 8;
        float row_f = qf;
        auto factor = [&](int group) {  // finite, so that a score of 0 stays 0
          float f = row_f * kf[group];
          if (fabsf(f) == INFINITY) f = copysignf(0x1p127f, f);
          return f;
        };
        if (!__all_sync(0xffffffffu, lo <= key0 && hi >= key0 + AP_TILE - 1) || s_bad[ring] != 0) {
          // masked: the exponents take the scores' place
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t v[16];
            tmem_ld_x16(t_s + c * 16, v);
            tmem_wait_ld();
            const float f = factor(c);
            const int first = kf[c] < 0.f ? 0x7fffffff : lo;  // an invalid page: no token seen
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int key = key0 + c * 16 + e;
              v[e] = key >= first && key <= hi ? __float_as_uint(__uint_as_float(v[e]) * f) : 0xff800000u;
            }
            tmem_st_x16(t_s + c * 16, v);
          }
          tmem_wait_st();
          kf = s_one, row_f = 1.f;
        }
        uint32_t p[64];
        f32x2 sum[2];
        bool move = __any_sync(0xffffffffu, sees && M == AT_NONE), moved = false;
        while (true) {
          if (move) {
            float high = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t v[16];
              tmem_ld_x16(t_s + c * 16, v);
              tmem_wait_ld();
              const float f = factor(c);
#pragma unroll
              for (int e = 0; e < 16; ++e) high = fmaxf(high, __uint_as_float(v[e]) * f);
            }
            const float to = fmaxf(M, high), f = ex2_approx(M - to);
            M = to;
            l2[0] = mul2(l2[0], pack2(f, f));
            l2[1] = mul2(l2[1], pack2(f, f));
            if (i > 0 && __any_sync(0xffffffffu, f != 1.f)) {  // the products before this tile's are done
#pragma unroll 1
              for (int c = 0; c < kD; c += 16) {
                uint32_t o[16];
                tmem_ld_x16(t_o + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st_x16(t_o + c, o);
              }
              tmem_wait_st();
            }
            moved = true;
          }
          const float m = M == AT_NONE ? 0.f : M;
          const f32x2 minus = pack2(-m, -m);
          float top = -INFINITY;
          sum[0] = sum[1] = pack2(0.f, 0.f);
          uint32_t v[2][32];
          tmem_ld_x32(t_s, v[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_wait_ld(v[c & 1]);
            if (c < 3) tmem_ld_x32(t_s + c * 32 + 32, v[(c + 1) & 1]);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float f1 = factor(2 * c + half);
              const f32x2 f = pack2(f1, f1);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int col = half * 16 + 2 * e;
                const f32x2 s2 = pack2(__uint_as_float(v[c & 1][col]), __uint_as_float(v[c & 1][col + 1]));
                const float2 y = unpack2(fma2(s2, f, minus));
                top = max3(top, y.x, y.y);
                const float2 z = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                sum[e & 1] = add2(sum[e & 1], pack2(z.x, z.y));
                p[c * 16 + half * 8 + e] = pack_bf16(z.x, z.y);
              }
            }
          }
          if (moved) break;
          move = __any_sync(0xffffffffu, top > AP_ROOM);
          if (!move) break;
        }
        l2[0] = add2(l2[0], sum[0]);
        l2[1] = add2(l2[1], sum[1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st_x16(t_s + c * 16, p + c * 16);
        tmem_wait_st();
        wait(v_full + vs, (uint32_t)(tile >> 1) & 1u);
        if (s_has_nan[vs] == tile + 1) {
          for (int k = max(lo - key0, 0); k <= min(hi - key0, AP_TILE - 1); ++k) {
            const uint16_t* bits = s_nan + (vs * AP_TILE + k) * kUnits;
#pragma unroll
            for (int u = 0; u < kUnits; ++u) poison[u / 2] |= (uint32_t)bits[u] << (16 * (u & 1));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + w);
      }
      // ---- the piece's O, reference and sum to its slot --------------------------
      float* slot = t.slots + (size_t)(2 * (blockIdx.x + unit) + w) * Shape::kSlotFloats;
      const float2 la = unpack2(add2(l2[0], l2[1]));
      __stcg(slot + AP_TILE * kD + row, M);
      __stcg(slot + AP_TILE * (kD + 1) + row, la.x + la.y);
      if (mine > 0) {
        wait(o_full + w, o_phase);
        o_phase ^= 1u;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kD; c += 32) {
          uint32_t o[32];
          tmem_ld_x32(t_o + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float4 y;
            float* f = &y.x;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              f[k] = poison[c / 32] >> (e + k) & 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float(o[e + k]);
            __stcg(reinterpret_cast<float4*>(slot) + (c + e) / 4 * AP_TILE + row, y);
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      count += n;
      pos += n;
    }
  } else if (warp < AP_WARP_LOAD) {
    // ---- V widened to bf16 -----------------------------------------------------
    // Lane pairs of eight take half of two neighbouring rows each, so that a
    // quarter warp's loads and swizzled stores lie in eight different banks' groups.
    give_registers<AP_REGS_V>();
    const int id = tid - AP_WARP_V * 32;
    constexpr int kPass = 128 / kUnits;  // rows of a pass
    const int pass_row = kUnits == 8 ? (id >> 4) * 2 + ((id >> 2) & 1) : id >> 2;
    const int u = kUnits == 8 ? (id & 3) | ((((id >> 2) & 1) ^ ((id >> 3) & 1)) << 2) : id & 3;
    int tile = 0;
    for (int pos = begin; pos < end;) {
      const int unit = pos / plan.tiles, j0 = pos - unit * plan.tiles, n = min(plan.tiles - j0, end - pos);
      for (int j = 0; j < n; ++j, ++tile) {
        const int vs = tile & 1, live = shared - (plan.tile0 + j0 + j) * AP_TILE;  // rows of the prefix
        const uint32_t parity = (uint32_t)(tile >> 1) & 1u;
        wait(r_full + vs, parity);
        wait(v_empty + vs, parity ^ 1u);
        const int* scales = s_vb + tile % AP_RING * 8;
        const uint8_t* src = s_raw + vs * Shape::kKBytes + u * 16;
        uint8_t* dst = s_v + vs * Shape::kVBytes + (u >> 2) * (AP_TILE * 128);
#pragma unroll 2
        for (int i = 0; i < kUnits; ++i) {
          const int r = i * kPass + pass_row, s = scales[r >> 4];
          uint4 raw = *reinterpret_cast<const uint4*>(src + r * kD);
          if (r >= live || s < 0) raw = make_uint4(0u, 0u, 0u, 0u);
          uint32_t mask = 0u, b[8];
          // NaN values are taken out and noted: 0 times NaN would reach rows that do not see them
          if (s == 255) {
            raw = make_uint4(0u, 0u, 0u, 0u);
            mask = r < live ? 0xffffu : 0u;
          }
          if (e4m3x16_to_bf16(raw, b)) {
            uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t m = ((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bit 7 of each NaN's byte
              w[e] &= ~((m >> 7) * 0xffu);
              mask |= ((m >> 7 & 1u) | (m >> 14 & 2u) | (m >> 21 & 4u) | (m >> 28 & 8u)) << (4 * e);
            }
            e4m3x16_to_bf16(make_uint4(w[0], w[1], w[2], w[3]), b);
          }
          if (mask) s_has_nan[vs] = tile + 1;
          s_nan[(vs * AP_TILE + r) * kUnits + u] = (uint16_t)mask;
          // 2^(s - 7) makes up for the codes' 2^-120, in two factors where it is no bf16
          const int scale = s == 255 || s < 0 ? 127 : s;
          const uint32_t one = (uint32_t)(min(scale, 134) + 120) << 7, m1 = one | one << 16;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const __nv_bfloat162 y =
                __hmul2(*reinterpret_cast<const __nv_bfloat162*>(b + e), *reinterpret_cast<const __nv_bfloat162*>(&m1));
            b[e] = *reinterpret_cast<const uint32_t*>(&y);
          }
          if (scale > 134) {
            const uint32_t two = (uint32_t)(scale - 7) << 7, m2 = two | two << 16;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(b + e),
                                               *reinterpret_cast<const __nv_bfloat162*>(&m2));
              b[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
          uint8_t* at = dst + r * 128;
          const int c = 2 * (u & 3), sw = r & 7;
          *reinterpret_cast<uint4*>(at + ((c ^ sw) << 4)) = make_uint4(b[0], b[1], b[2], b[3]);
          *reinterpret_cast<uint4*>(at + (((c + 1) ^ sw) << 4)) = make_uint4(b[4], b[5], b[6], b[7]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(v_full + vs);
          mbar_arrive(r_empty + vs);
        }
      }
      pos += n;
    }
  } else if (warp == AP_WARP_LOAD) {
    // ---- pages of K and V, and their scales ------------------------------------
    give_registers<AP_REGS_REST>();
    const int per_tile = AP_TILE >> t.page_shift;
    const uint64_t policy = l2_policy_evict_first();
    const int32_t* table = a.table + (size_t)lead * a.table_stride;
    int tile = 0;
    for (int pos = begin; pos < end;) {
      const int unit = pos / plan.tiles, j0 = pos - unit * plan.tiles, n = min(plan.tiles - j0, end - pos);
      const int h = unit / t.row_blocks;
      // pages of 32 columns at a time, one batch ahead
      const int c0 = (plan.tile0 + j0) * per_tile, stop = min(c0 + n * per_tile, (shared + (1 << t.page_shift) - 1) >> t.page_shift);
      auto page_at = [&](int col) {
        const int pid = col < stop ? __ldg(table + col) : -1;
        return pid >= 0 && pid < a.pages ? pid : -1;
      };
      int batch = c0, used = 0;
      int pid = page_at(batch + lane), pid_next = page_at(batch + 32 + lane);
      int kb = 0, vb = -1;
      if (pid >= 0) {
        kb = __ldg(a.ks + (size_t)pid * a.Hkv + h);
        vb = __ldg(a.vs + (size_t)pid * a.Hkv + h);
      }
      for (int j = 0; j < n; ++j, ++tile) {
        if (used == 32) {
          used = 0;
          batch += 32;
          pid = pid_next;
          kb = 0, vb = -1;
          if (pid >= 0) {
            kb = __ldg(a.ks + (size_t)pid * a.Hkv + h);
            vb = __ldg(a.vs + (size_t)pid * a.Hkv + h);
          }
          pid_next = page_at(batch + 32 + lane);
        }
        const int col = batch + lane, stage = tile % AP_K_STAGES, ring = tile % AP_RING, rs = tile & 1;
        const bool mine = lane >= used && lane < used + per_tile, needed = mine && col < stop;
        const uint32_t bad = __ballot_sync(0xffffffffu, needed && pid < 0);
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, needed && pid >= 0)) * (uint32_t)(kD << t.page_shift);
        if (bad && lane == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
        const int row = needed && pid >= 0 ? (pid * a.Hkv + h) << t.page_shift : -1;
        int at[AT_MAX_PAGES];
#pragma unroll
        for (int p = 0; p < AT_MAX_PAGES; ++p) {
          const int r = __shfl_sync(0xffffffffu, row, (used + p) & 31);
          at[p] = p < per_tile ? r : -1;
        }
        auto issue = [&](uint8_t* to, const CUtensorMap* map, uint64_t* bar) {
          if (lane == 0) mbar_expect_tx(bar, bytes);
          __syncwarp();
          if (elect_one()) {
#pragma unroll
            for (int p = 0; p < AT_MAX_PAGES; ++p)
              if (at[p] >= 0) tma_load_2d(to + (p << t.page_shift) * kD, map, 0, at[p], bar, policy);
          }
          __syncwarp();
        };
        if (__all_sync(0xffffffffu, wait(k_empty + stage, ((uint32_t)(tile / AP_K_STAGES) & 1u) ^ 1u))) {
          issue(s_k + stage * Shape::kKBytes, &tm_k, k_full + stage);
          // tokens past the prefix are masked by their number
          const float f = needed && pid < 0 ? -1.f : ue8m0_to_f32((uint32_t)kb);
          const int each = 8 / per_tile;  // groups of 16 tokens of a page
          if (mine) {
            for (int e = 0; e < each; ++e) {
              s_kf[ring * 8 + (lane - used) * each + e] = f;
              s_vb[ring * 8 + (lane - used) * each + e] = vb;
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
        used += per_tile;
      }
      pos += n;
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0) {
      for (int i = max(0, tile - AP_K_STAGES); i < tile; ++i)
        mbar_wait(k_full + i % AP_K_STAGES, (uint32_t)(i / AP_K_STAGES) & 1u);
      for (int i = max(0, tile - 2); i < tile; ++i) mbar_wait(r_full + (i & 1), (uint32_t)(i >> 1) & 1u);
    }
    __syncwarp();
  } else if (warp == AP_WARP_MMA) {
    // ---- products ----------------------------------------------------------------
    give_registers<AP_REGS_REST>();
    constexpr uint32_t kIdS = tc_idesc_e4m3(AP_TILE, AP_TILE, false, false);
    constexpr uint32_t kIdO = tc_idesc_bf16(AP_TILE, kD) | 1u << 16;  // V lies with its values side by side
    const uint64_t d_q = tc_desc(smem_u32(s_q), 16, kAtom, kSwz), d_k = tc_desc(smem_u32(s_k), 16, kAtom, kSwz);
    const uint64_t d_v = tc_desc(smem_u32(s_v), AP_TILE * 128, 1024, 2);
    int count = 0;
    uint32_t q_phase = 0, p_phase = 0;
    auto scores = [&](int tile, int w, bool last_of_tile, bool ok) {
      const int stage = tile % AP_K_STAGES;
      ok = wait(k_full + stage, (uint32_t)(tile / AP_K_STAGES) & 1u) && ok;
      tc_fence_after();
      if (__all_sync(0xffffffffu, ok) && elect_one()) {
        const uint64_t k = d_k + (uint32_t)(stage * Shape::kKBytes / 16);
        const uint64_t q = d_q + (uint32_t)(w * 2 * Shape::kQTerm / 16);
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int s = 0; s < kD / 32; ++s)
            tc_mma_f8(tmem + w * AP_TILE, q + term * (Shape::kQTerm / 16) + 2 * s, k + 2 * s, kIdS, term + s > 0);
        tc_commit(s_full + w);
        if (last_of_tile) tc_commit(k_empty + stage);
      }
      __syncwarp();
    };
    for (int pos = begin; pos < end;) {
      const int unit = pos / plan.tiles, j0 = pos - unit * plan.tiles, n = min(plan.tiles - j0, end - pos);
      for (int w = 0; w < 2; ++w) {
        const bool ok = wait(q_full + w, q_phase);
        if (tiles_of(n, w) > 0) scores(count + (kTwo ? 0 : w), w, !kTwo || w == 1, ok);
      }
      q_phase ^= 1u;
      for (int i = 0; i < tiles_of(n, 0); ++i) {
        for (int w = 0; w < 2; ++w) {
          const int mine = tiles_of(n, w);
          if (i >= mine) continue;
          const int tile = count + (kTwo ? i : 2 * i + w), vs = tile & 1;
          bool ok = wait(p_full + w, p_phase >> w & 1u);
          p_phase ^= 1u << w;
          ok = wait(v_full + vs, (uint32_t)(tile >> 1) & 1u) && ok;
          tc_fence_after();
          if (__all_sync(0xffffffffu, ok) && elect_one()) {
            const uint64_t v = d_v + (uint32_t)(vs * Shape::kVBytes / 16);
#pragma unroll
            for (int s = 0; s < AP_TILE / 16; ++s)
              tc_mma_bf16_ts(tmem + 2 * AP_TILE + w * kD, tmem + w * AP_TILE + 8 * s, v + s * 128, kIdO, i > 0 || s > 0);
            if (!kTwo || w == 1) tc_commit(v_empty + vs);
            if (i == mine - 1) tc_commit(o_full + w);
          }
          __syncwarp();
          if (i + 1 < mine) scores(count + (kTwo ? i + 1 : 2 * i + 2 + w), w, !kTwo || w == 1, ok);
        }
      }
      count += n;
      pos += n;
    }
    // After an abort let what was issued end before TMEM is freed.
    __syncwarp();
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained);
      mbar_wait(drained, 0);
    }
    __syncwarp();
  } else {
    give_registers<AP_REGS_REST>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == AP_WARP_MMA) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the prefix and the sequences' own parts (fp32 values already
// over their sums, with their log sums): a thread four values of a row, a block 32
// rows of a unit's row tile by 32 values.
template <int kD, bool kTwo>
__global__ void __launch_bounds__(256)
    attn_prefix_join_kernel(const AttnPrefixArgs t, const float* own, const float* own_lse) {
  using Shape = AttnPrefixShape<kD>;
  const AttnArgs& a = t.a;
  const AttnPrefixPlan plan = *reinterpret_cast<const AttnPrefixPlan*>(t.plan);
  const int lane = threadIdx.x & 31, quad = blockIdx.y * 8 + (threadIdx.x >> 5);
  constexpr int kTiles = kTwo ? 2 : 1;
  const int tile = blockIdx.x >> 2, sub = blockIdx.x & 3;          // row tile of all, 32 rows of it
  const int unit = tile / kTiles, half = tile - unit * kTiles, row = sub * 32 + lane;
  const int G = a.Hq / a.Hkv, rows = a.B * a.Sq * G;
  const int h = unit / t.row_blocks, rr = (unit - h * t.row_blocks) * kTiles * AP_TILE + half * AP_TILE + row;
  if (rr >= rows) return;
  const size_t at = (size_t)(rr / G) * a.Hq + h * G + rr % G;  // row of the output
  float4 y = __ldcg(reinterpret_cast<const float4*>(own + at * kD) + quad);
  const float lse = __ldcg(own_lse + at);
  // (a NaN log sum is a part whose values are NaN)
  float M = lse == -INFINITY ? AT_NONE : lse * 1.4426950408889634f, sum = lse == -INFINITY ? 0.f : 1.f;
  if (plan.tiles > 0) {
    AttnShares shares;
    shares.each = plan.each, shares.more = plan.more;
    const int ca = shares.cta_of(unit * plan.tiles), cz = shares.cta_of(unit * plan.tiles + plan.tiles - 1);
    const int each = kTwo ? 1 : 2, pieces = (cz - ca + 1) * each;
    constexpr int kBatch = 4;
    for (int p0 = 0; p0 < pieces; p0 += kBatch) {
      float m[kBatch], l[kBatch];
      float4 v[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int p = min(p0 + e, pieces - 1);
        const float* s = t.slots + (size_t)(2 * (ca + p / each + unit) + (kTwo ? half : p % each)) * Shape::kSlotFloats;
        m[e] = __ldcg(s + AP_TILE * kD + row);
        l[e] = __ldcg(s + AP_TILE * (kD + 1) + row);
        v[e] = __ldcg(reinterpret_cast<const float4*>(s) + quad * AP_TILE + row);
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (p0 + e >= pieces || (m[e] == AT_NONE && l[e] == 0.f)) continue;  // no token seen: O may be anything
        const float to = fmaxf(M, m[e]), f = ex2_approx(M - to), w = ex2_approx(m[e] - to);
        M = to;
        sum = fmaf(l[e], w, sum * f);
        y.x = fmaf(v[e].x, w, y.x * f), y.y = fmaf(v[e].y, w, y.y * f);
        y.z = fmaf(v[e].z, w, y.z * f), y.w = fmaf(v[e].w, w, y.w * f);
      }
    }
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(a.out + at * kD + 4 * quad) = make_uint2(pack_bf16(y.x * f, y.y * f), pack_bf16(y.z * f, y.w * f));
  if (a.lse && quad == 0) a.lse[at] = sum == 0.f ? -INFINITY : M * 0.6931471805599453f + logf(sum);
}

}  // namespace wdb

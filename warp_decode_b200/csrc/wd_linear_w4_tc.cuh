// Projection with 4-bit weights on the tensor cores (the formula and the packed
// layout: wd_linear_w4.cuh), sm_100a.
//
// A block: 128 output rows of up to 64 tokens over a share of k, in steps of 128 k.
// Eight warps load codes, several steps ahead in registers, and turn them into bf16
// whole numbers (less their zero points, exactly) in the swizzled layout of the
// products, in two groups that take every second step; x comes through TMA in the same
// layout.  A group's sum is an accumulator of its own in TMEM, and four warps add it,
// times its scale, to the block's sums in registers while the next is made: nothing is
// rounded before the end.  The blocks of a cluster share k and join their sums over
// distributed shared memory, in rank order.
//
// Codes do not come through TMA: the first copy waits some 4000 clocks for its
// descriptor. x does, though all blocks read the same x: copied 16 bytes a lane it
// arrived at 7 bytes a clock (64 tokens of 4096 to 9216: 36 us).
//
// Measured (B200): 64 tokens of 4096 to 9216, and 16 of 8192 to 4096 with zero points, 20.5
// us, 16 steps a block of ~750 clocks: eight matrix instructions take 450 of them, the
// conversion of a step 600 in each of its two groups.  More tokens read and convert the
// codes again for every 64: 128 of 4096 to 9216 35 us (cold), 320 86, 1024 217, 4096 847.
#pragma once

#include "wd_linear_w4.cuh"

namespace wdb {

constexpr int W4T_ROWS = 128;
constexpr int W4T_THREADS = 448;     // 2 x 4 warps convert, 4 add up, one loads x, one issues products
constexpr int W4T_ADD = 8, W4T_LOAD = 12, W4T_MMA = 13;  // first warps of the roles
constexpr int W4T_X = 4, W4T_W = 4;  // stages of x and of bf16 codes

template <int kN>
struct W4TcShape {
  static constexpr int kXBytes = kN * 256, kWBytes = W4T_ROWS * 256;
  static constexpr int kOffW = W4T_X * kXBytes;
  static constexpr int kOffBar = kOffW + W4T_W * kWBytes;
  static constexpr int kSmem = kOffBar + 256 + 1024;  // + alignment slack
};

// kN: tokens of the block, rounded up to 16, 32 or 64.  kSums: groups of a step.
template <int kN, int kSums, int kScale>
__global__ void __launch_bounds__(W4T_THREADS, 1)
    linear_w4_tc_kernel(const LinearW4Args a, const __grid_constant__ CUtensorMap tm_x) {
  using Shape = W4TcShape<kN>;
  constexpr int kTmem = 2 * kSums * kN < 32 ? 32 : 2 * kSums * kN;  // columns: two steps' sums
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)cluster_ctarank(), ranks = gridDim.x;
  const int n0 = blockIdx.y * W4T_ROWS, t0 = blockIdx.z * kN;
  const int first = (int)((long long)a.blocks * rank / ranks), steps = (int)((long long)a.blocks * (rank + 1) / ranks) - first;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_x = smem;                  // [stages][2][kN][64]
  uint8_t* s_w = smem + Shape::kOffW;   // [stages][2][128][64]
  uint64_t* x_full = reinterpret_cast<uint64_t*>(smem + Shape::kOffBar);
  uint64_t* x_empty = x_full + W4T_X;
  uint64_t* w_full = x_empty + W4T_X;
  uint64_t* w_empty = w_full + W4T_W;
  uint64_t* sum_full = w_empty + W4T_W;   // [2]
  uint64_t* sum_empty = sum_full + 2;     // [2]
  uint64_t* drained = sum_empty + 2;
  volatile int* s_abort = reinterpret_cast<volatile int*>(drained + 1);
  uint32_t* s_tmem = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(s_abort + 1));
  static_assert(8 * (2 * W4T_X + 2 * W4T_W + 5) + 8 <= 256, "barriers");
  static_assert(W4T_ROWS * kN * 4 <= W4T_W * Shape::kWBytes, "the sums take the place of the codes");

  // ---- codes: four 16-byte units of a step a thread, of steps group, group + 2, ...  ----
  constexpr int kUnits = 4, kAhead = 2;
  const int group = warp >> 2, in_group = tid & 127, t4 = in_group & 3, row0 = in_group >> 2;
  uint4 raw[kAhead][kUnits];
  auto load = [&](uint4 (&to)[kUnits], int step) {
    if (step >= steps) return;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const size_t r = min(n0 + row0 + 32 * u, a.N - 1);
      to[u] = __ldcs(reinterpret_cast<const uint4*>(a.w + (r * a.blocks + first + step) * 64) + t4);
    }
  };
  if (warp < W4T_ADD) {  // before anything else
#pragma unroll
    for (int d = 0; d < kAhead; ++d) load(raw[d], group + 2 * d);
  }

  auto load_x = [&](int step) {
    mbar_arrive_expect_tx(x_full + step % W4T_X, Shape::kXBytes);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      tma_load_2d(s_x + step % W4T_X * Shape::kXBytes + h * kN * 128, &tm_x, (first + step) * 128 + h * 64, t0,
                  x_full + step % W4T_X, l2_policy_evict_last());
  };
  if (warp == W4T_LOAD && lane == 0) {
    prefetch_tensormap(&tm_x);
    *s_abort = 0;
    for (int i = 0; i < W4T_X; ++i) mbar_init(x_full + i, 1), mbar_init(x_empty + i, 1);
    for (int i = 0; i < W4T_W; ++i) mbar_init(w_full + i, 4), mbar_init(w_empty + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(sum_full + i, 1), mbar_init(sum_empty + i, 4);
    mbar_init(drained, 1);
    fence_mbar_init();
    for (int i = 0; i < min(steps, W4T_X); ++i) load_x(i);
  } else if (warp == W4T_MMA) {
    tmem_alloc(s_tmem, kTmem);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;

  // Bounded wait of a whole warp; once one gave up, none waits and nothing more is issued.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return wait_on(bar, parity, s_abort, nullptr);
  };

  float acc[kN];
  if (warp < W4T_ADD) {
    // zero points of a step's groups, loaded a step ahead and left as they come
    uint32_t z[kUnits][kSums];
    auto zeros_of = [&](int step) {
      if (step >= steps) return;
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const uint8_t* p = a.zero + (size_t)min(n0 + row0 + 32 * u, a.N - 1) * a.groups + (first + step) * kSums;
#pragma unroll
        for (int j = 0; j < kSums; ++j)
          if ((first + step) * kSums + j < a.groups) z[u][j] = __ldg(p + j);
      }
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int j = 0; j < kSums; ++j) z[u][j] = 8u;
    if (a.zero) zeros_of(group);
    auto convert = [&](uint4 (&codes)[kUnits], int i) {
      const int ws = i % W4T_W;
      wait(w_empty + ws, ((uint32_t)(i / W4T_W) & 1u) ^ 1u);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int r = row0 + 32 * u;
        uint8_t* to = s_w + ws * Shape::kWBytes + r * 128;
        const uint32_t word[4] = {codes[u].x, codes[u].y, codes[u].z, codes[u].w};
        __nv_bfloat162 z128[kSums];
#pragma unroll
        for (int j = 0; j < kSums; ++j)
          z128[j] = __float2bfloat162_rn(128.f + (float)min(z[u][j], 127u));
#pragma unroll
        for (int s = 0; s < 4; ++s) {  // k = 32 s + 8 t4 + 0..7
          const __nv_bfloat162 zs = z128[s * kSums / 4];
          *reinterpret_cast<uint4*>(to + (s >> 1) * (W4T_ROWS * 128) + (((4 * (s & 1) + t4) ^ (r & 7)) << 4)) =
              make_uint4(w4_pair(word[s], 0, zs), w4_pair(word[s], 1, zs), w4_pair(word[s], 2, zs),
                         w4_pair(word[s], 3, zs));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(w_full + ws);
      load(codes, i + 2 * kAhead);
      if (a.zero) zeros_of(i + 2);
    };
#pragma unroll 1
    for (int i = group; i < steps; i += 2 * kAhead) {
#pragma unroll
      for (int d = 0; d < kAhead; ++d)
        if (i + 2 * d < steps) convert(raw[d], i + 2 * d);
    }
  } else if (warp < W4T_LOAD) {
    // ---- groups' sums, times their scales ------------------------------------------
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const size_t scales = (size_t)min(n0 + row, a.N - 1) * a.groups;
#pragma unroll
    for (int c = 0; c < kN; ++c) acc[c] = 0.f;
    // scales, loaded three steps ahead and left as they come
    constexpr int kAheadS = 4;
    using Raw = std::conditional_t<kScale == W4_F32, float, uint16_t>;
    Raw f[kAheadS][kSums];
    auto scales_of = [&](int step, Raw (&to)[kSums]) {
#pragma unroll
      for (int j = 0; j < kSums; ++j) {
        const int g = (first + step) * kSums + j;
        to[j] = 0;
        if (step < steps && g < a.groups) to[j] = __ldg(static_cast<const Raw*>(a.scale) + scales + g);
      }
    };
#pragma unroll
    for (int d = 0; d < kAheadS; ++d) scales_of(d, f[d]);
    auto add = [&](int i, Raw (&scale)[kSums]) {
      const int b = i & 1;
      wait(sum_full + b, (uint32_t)(i >> 1) & 1u);
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < kSums; ++j) {
        if ((first + i) * kSums + j < a.groups) {  // (no group there: no scale)
          const float factor = w4_value<kScale>(scale[j]);
#pragma unroll
          for (int c = 0; c < kN; c += 16) {
            uint32_t v[16];
            tmem_ld_x16(lanes + (b * kSums + j) * kN + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(v[e]), factor, acc[c + e]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_empty + b);
      scales_of(i + kAheadS, scale);
    };
#pragma unroll 1
    for (int i = 0; i < steps; i += kAheadS) {
#pragma unroll
      for (int d = 0; d < kAheadS; ++d)
        if (i + d < steps) add(i + d, f[d]);
    }
  } else if (warp == W4T_LOAD) {
    // ---- x: zeros past its end and past the last token --------------------------------
#pragma unroll 1
    for (int i = W4T_X; i < steps; ++i) {
      const bool ok = wait(x_empty + i % W4T_X, ((uint32_t)(i / W4T_X) & 1u) ^ 1u);
      if (__all_sync(0xffffffffu, ok) && lane == 0) load_x(i);
      __syncwarp();
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0)
      for (int i = max(0, steps - W4T_X); i < steps; ++i) mbar_wait(x_full + i % W4T_X, (uint32_t)(i / W4T_X) & 1u);
    __syncwarp();
  } else {
    // ---- products ----------------------------------------------------------------------
    constexpr uint32_t kId = tc_idesc_bf16(W4T_ROWS, kN);
    const uint64_t d_w = tc_desc_sw128(smem_u32(s_w)), d_x = tc_desc_sw128(smem_u32(s_x));
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const int ws = i % W4T_W, xs = i % W4T_X, b = i & 1;
      bool ok = wait(sum_empty + b, ((uint32_t)(i >> 1) & 1u) ^ 1u);
      ok = wait(x_full + xs, (uint32_t)(i / W4T_X) & 1u) && ok;
      ok = wait(w_full + ws, (uint32_t)(i / W4T_W) & 1u) && ok;
      tc_fence_after();
      if (__all_sync(0xffffffffu, ok) && elect_one()) {
        const uint64_t w = d_w + (uint32_t)(ws * Shape::kWBytes / 16), x = d_x + (uint32_t)(xs * Shape::kXBytes / 16);
#pragma unroll
        for (int s = 0; s < 8; ++s) {  // 16 k each
          constexpr int kPer = 8 / kSums;
          const uint32_t at = (uint32_t)(s >> 2), in = (uint32_t)(2 * (s & 3));
          tc_mma_bf16(tmem + (b * kSums + s / kPer) * kN, w + at * (W4T_ROWS * 128 / 16) + in, x + at * (kN * 128 / 16) + in,
                      kId, s % kPer > 0);
        }
        tc_commit(w_empty + ws);
        tc_commit(x_empty + xs);
        tc_commit(sum_full + b);
      }
      __syncwarp();
    }
    // After an abort let what was issued end before TMEM is freed.
    if (__any_sync(0xffffffffu, *s_abort != 0) && elect_one()) {
      tc_commit(drained);
      mbar_wait(drained, 0);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == W4T_MMA) tmem_dealloc(tmem, kTmem);

  // sums as [token][row], in the place of the codes; every product has read them
  float* s_sum = reinterpret_cast<float*>(s_w);
  if (warp >= W4T_ADD && warp < W4T_LOAD) {
    const int row = (warp & 3) * 32 + lane;
#pragma unroll
    for (int c = 0; c < kN; ++c) s_sum[c * W4T_ROWS + row] = acc[c];
  }
  if (ranks > 1)
    cluster_sync();
  else
    __syncthreads();
  // four rows of a token a thread
  const bool wide = (a.o_ts | a.N) % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0;
  const int tokens = min(kN, a.T - t0);
  for (int e = tid + rank * W4T_THREADS; e < tokens * (W4T_ROWS / 4); e += ranks * W4T_THREADS) {
    const int t = e / (W4T_ROWS / 4), r = e % (W4T_ROWS / 4) * 4;
    if (n0 + r >= a.N) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ranks > 1) {
      float4 v[W4_MAX_SPLIT];
#pragma unroll
      for (int i = 0; i < W4_MAX_SPLIT; ++i)
        if (i < ranks) v[i] = dsmem_ld_f32x4(dsmem_addr(s_sum + t * W4T_ROWS + r, i));
#pragma unroll
      for (int i = 0; i < W4_MAX_SPLIT; ++i)
        if (i < ranks) sum.x += v[i].x, sum.y += v[i].y, sum.z += v[i].z, sum.w += v[i].w;
    } else {
      sum = *reinterpret_cast<const float4*>(s_sum + t * W4T_ROWS + r);
    }
    __nv_bfloat16* out = a.out + (t0 + t) * a.o_ts + n0 + r;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
    if (wide) {
      *reinterpret_cast<uint2*>(out) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      out[0] = lo.x;
      if (n0 + r + 1 < a.N) out[1] = lo.y;
      if (n0 + r + 2 < a.N) out[2] = hi.x;
      if (n0 + r + 3 < a.N) out[3] = hi.y;
    }
  }
  if (ranks > 1) cluster_sync();
}

}  // namespace wdb

// Projection with 4-bit weights on the tensor cores (the formula and the packed
// layout: wd_linear_w4.cuh), sm_100a.
//
// A block: 128 output rows of up to 64 tokens over a share of k, in steps of 128 k.
// Codes come through TMA as they are packed; eight warps turn them into bf16 whole
// numbers (less their zero points, exactly) in the swizzled layout of the products;
// x comes through TMA in the same layout.  A group's sum is an accumulator of its own
// in TMEM, and four warps add it, times its scale, to the block's sums in registers
// while the next is made: nothing is rounded before the end.  The blocks of a cluster
// share k and join their sums over distributed shared memory, in rank order.
#pragma once

#include "wd_linear_w4.cuh"

namespace wdb {

constexpr int W4T_ROWS = 128;
constexpr int W4T_THREADS = 448;     // 8 warps convert, 4 add up, one loads, one issues products
constexpr int W4T_ADD = 8, W4T_LOAD = 12, W4T_MMA = 13;  // first warps of the roles
constexpr int W4T_RAW = 8, W4T_X = 4, W4T_W = 3;         // stages: packed codes, x, bf16 codes

template <int kN>
struct W4TcShape {
  static constexpr int kRawBytes = W4T_ROWS * 64, kXBytes = kN * 256, kWBytes = W4T_ROWS * 256;
  static constexpr int kOffW = W4T_X * kXBytes, kOffRaw = kOffW + W4T_W * kWBytes;
  static constexpr int kOffBar = kOffRaw + W4T_RAW * kRawBytes;
  static constexpr int kSmem = kOffBar + 512 + 1024;  // + alignment slack
};

// kN: tokens of the block, rounded up to 16, 32 or 64.  kSums: groups of a step.
template <int kN, int kSums, int kScale>
__global__ void __launch_bounds__(W4T_THREADS, 1)
    linear_w4_tc_kernel(const LinearW4Args a, uint32_t* status, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_x) {
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
  uint8_t* s_raw = smem + Shape::kOffRaw;
  uint64_t* raw_full = reinterpret_cast<uint64_t*>(smem + Shape::kOffBar);
  uint64_t* raw_empty = raw_full + W4T_RAW;
  uint64_t* x_full = raw_empty + W4T_RAW;
  uint64_t* x_empty = x_full + W4T_X;
  uint64_t* w_full = x_empty + W4T_X;
  uint64_t* w_empty = w_full + W4T_W;
  uint64_t* sum_full = w_empty + W4T_W;   // [2]
  uint64_t* sum_empty = sum_full + 2;     // [2]
  uint64_t* drained = sum_empty + 2;
  volatile int* s_abort = reinterpret_cast<volatile int*>(drained + 1);
  uint32_t* s_tmem = const_cast<uint32_t*>(reinterpret_cast<volatile uint32_t*>(s_abort + 1));
  static_assert(8 * (2 * W4T_RAW + 2 * W4T_X + 2 * W4T_W + 5) + 8 <= 512, "barriers");
  static_assert(W4T_ROWS * kN * 4 <= W4T_W * Shape::kWBytes, "the sums take the place of the codes");

  if (warp == W4T_LOAD && lane == 0) {
    *s_abort = 0;
    for (int i = 0; i < W4T_RAW; ++i) mbar_init(raw_full + i, 1), mbar_init(raw_empty + i, 8);
    for (int i = 0; i < W4T_X; ++i) mbar_init(x_full + i, 1), mbar_init(x_empty + i, 1);
    for (int i = 0; i < W4T_W; ++i) mbar_init(w_full + i, 8), mbar_init(w_empty + i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(sum_full + i, 1), mbar_init(sum_empty + i, 4);
    mbar_init(drained, 1);
    fence_mbar_init();
    prefetch_tensormap(&tm_w);
    prefetch_tensormap(&tm_x);
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
    bool ok = mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    const uint64_t begin = globaltimer_ns();
    for (uint32_t it = 1; !(ok = mbar_try_wait(bar, parity)); ++it) {
      if ((it & 31u) == 0) {
        if (*s_abort) break;
        if (globaltimer_ns() - begin > WD_WAIT_LIMIT_NS) {
          *s_abort = 1;
          raise_status(status, WD_STATUS_WAIT_TIMEOUT);
          break;
        }
      }
    }
    __syncwarp();
    return ok;
  };

  float acc[kN];
  if (warp < W4T_ADD) {
    // ---- codes to bf16: two 16-byte units of a step a thread ----------------------
    const int row = tid >> 2, t4 = tid & 3;  // and row + 64
    const int groups_of[2] = {min(n0 + row, a.N - 1), min(n0 + row + 64, a.N - 1)};
    // zero points of a step's groups, a byte each, 8 without them
    auto zeros_of = [&](int step, uint32_t (&z)[2]) {
      z[0] = z[1] = 0x08080808u;
      if (!a.zero || step >= steps) return;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint8_t* p = a.zero + (size_t)groups_of[u] * a.groups + (first + step) * kSums;
        z[u] = 0u;
#pragma unroll
        for (int j = 0; j < kSums; ++j)
          if ((first + step) * kSums + j < a.groups) z[u] |= (uint32_t)__ldg(p + j) << (8 * j);
      }
    };
    uint32_t z[2];
    zeros_of(0, z);
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const int rs = i % W4T_RAW, ws = i % W4T_W;
      uint32_t next[2];
      zeros_of(i + 1, next);
      wait(raw_full + rs, (uint32_t)(i / W4T_RAW) & 1u);
      uint4 raw[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        raw[u] = *reinterpret_cast<const uint4*>(s_raw + rs * Shape::kRawBytes + (row + 64 * u) * 64 + t4 * 16);
      __syncwarp();
      if (lane == 0) mbar_arrive(raw_empty + rs);
      wait(w_empty + ws, ((uint32_t)(i / W4T_W) & 1u) ^ 1u);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int r = row + 64 * u;
        uint8_t* to = s_w + ws * Shape::kWBytes + r * 128;
        const uint32_t word[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {  // k = 32 s + 8 t4 + 0..7
          const uint32_t zero = z[u] >> (8 * (s * kSums / 4)) & 0xffu;
          const __nv_bfloat162 z128 = __float2bfloat162_rn(128.f + (float)min(zero, 127u));
          *reinterpret_cast<uint4*>(to + (s >> 1) * (W4T_ROWS * 128) + (((4 * (s & 1) + t4) ^ (r & 7)) << 4)) =
              make_uint4(w4_pair(word[s], 0, z128), w4_pair(word[s], 1, z128), w4_pair(word[s], 2, z128),
                         w4_pair(word[s], 3, z128));
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(w_full + ws);
      z[0] = next[0], z[1] = next[1];
    }
  } else if (warp < W4T_LOAD) {
    // ---- groups' sums, times their scales ------------------------------------------
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const size_t scales = (size_t)min(n0 + row, a.N - 1) * a.groups;
#pragma unroll
    for (int c = 0; c < kN; ++c) acc[c] = 0.f;
    auto scales_of = [&](int step, float (&f)[kSums]) {
#pragma unroll
      for (int j = 0; j < kSums; ++j) {
        const int g = (first + step) * kSums + j;
        f[j] = step < steps && g < a.groups ? w4_scale<kScale>(a.scale, scales + g) : 0.f;
      }
    };
    float f[kSums];
    scales_of(0, f);
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const int b = i & 1;
      float next[kSums];
      scales_of(i + 1, next);
      wait(sum_full + b, (uint32_t)(i >> 1) & 1u);
      tc_fence_after();
#pragma unroll
      for (int j = 0; j < kSums; ++j) {
        if ((first + i) * kSums + j < a.groups) {  // (no group there: no scale, and its products are not made)
#pragma unroll
          for (int c = 0; c < kN; c += 16) {
            uint32_t v[16];
            tmem_ld_x16(lanes + (b * kSums + j) * kN + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(__uint_as_float(v[e]), f[j], acc[c + e]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_empty + b);
#pragma unroll
      for (int j = 0; j < kSums; ++j) f[j] = next[j];
    }
  } else if (warp == W4T_LOAD) {
    // ---- packed codes and x ------------------------------------------------------------
    const uint64_t once = l2_policy_evict_first(), keep = l2_policy_evict_last();
#pragma unroll 1
    for (int i = 0; i < steps + W4T_RAW - W4T_X; ++i) {
      // codes run ahead of x by as much as their ring is longer
      const int j = i - (W4T_RAW - W4T_X);
      if (i < steps) {
        const int rs = i % W4T_RAW;
        const bool ok = wait(raw_empty + rs, ((uint32_t)(i / W4T_RAW) & 1u) ^ 1u);
        if (__all_sync(0xffffffffu, ok) && elect_one()) {
          mbar_arrive_expect_tx(raw_full + rs, Shape::kRawBytes);
          tma_load_2d(s_raw + rs * Shape::kRawBytes, &tm_w, (first + i) * 64, n0, raw_full + rs, once);
        }
        __syncwarp();
      }
      if (j >= 0) {
        const int xs = j % W4T_X;
        const bool ok = wait(x_empty + xs, ((uint32_t)(j / W4T_X) & 1u) ^ 1u);
        if (__all_sync(0xffffffffu, ok) && elect_one()) {
          mbar_arrive_expect_tx(x_full + xs, Shape::kXBytes);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tma_load_2d(s_x + xs * Shape::kXBytes + h * kN * 128, &tm_x, (first + j) * 128 + h * 64, t0, x_full + xs, keep);
        }
        __syncwarp();
      }
    }
    // After an abort let every issued copy land before the CTA can exit.
    if (*s_abort && lane == 0) {
      for (int i = max(0, steps - W4T_RAW); i < steps; ++i)
        mbar_wait(raw_full + i % W4T_RAW, (uint32_t)(i / W4T_RAW) & 1u);
      for (int i = max(0, steps - W4T_X); i < steps; ++i) mbar_wait(x_full + i % W4T_X, (uint32_t)(i / W4T_X) & 1u);
    }
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
  // two rows a thread
  for (int e = tid + rank * W4T_THREADS; e < kN * (W4T_ROWS / 2); e += ranks * W4T_THREADS) {
    const int t = e / (W4T_ROWS / 2), r = e % (W4T_ROWS / 2) * 2;
    if (t0 + t >= a.T || n0 + r >= a.N) continue;
    float2 sum = *reinterpret_cast<const float2*>(s_sum + t * W4T_ROWS + r);
    if (ranks > 1) {
      sum = make_float2(0.f, 0.f);
      for (int i = 0; i < ranks; ++i) {
        const uint32_t at = dsmem_addr(s_sum + t * W4T_ROWS + r, i);
        sum.x += dsmem_ld_f32(at), sum.y += dsmem_ld_f32(at + 4);
      }
    }
    __nv_bfloat16* out = a.out + (t0 + t) * a.o_ts + n0 + r;
    out[0] = __float2bfloat16_rn(sum.x);
    if (n0 + r + 1 < a.N) out[1] = __float2bfloat16_rn(sum.y);
  }
  if (ranks > 1) cluster_sync();
}

}  // namespace wdb

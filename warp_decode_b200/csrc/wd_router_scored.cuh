// Expert choice from router logits, sm_100a: softmax or sigmoid scores, a
// balance bias, expert groups, top-k, renormalised weights.  Extends the
// plain softmax router of wd_router.cuh; the reference has no router.
//
// One warp per token; lane l keeps `per` consecutive experts from l * per on
// as 32-bit keys whose unsigned order is the order of the choice values, and
// the best two of them.  A top-k step is two warp reductions in hardware
// (largest key, then the lowest expert that has it); only a lane that loses
// its second best looks through its experts again.  Key 0 marks what is not
// up for choice: it lies below the key of -infinity.
//
// Bound by instructions: 16384 x 256 logits with 4 of 8 groups read 17.8 MB
// (2.7 us of HBM) and take 19.2 us, about 800 instructions a token: 250 for its
// scores (exp, an exactly rounded reciprocal), the rest for the choice.  With
// experts strided over the lanes and groups through shared memory it took 25.0,
// with a rescan at every step 30.7.
#pragma once

#include "wd_common.cuh"

namespace wdb {

constexpr int RS_WARPS = 4;
constexpr int RS_MAX_E = 1024;
constexpr int RS_MAX_K = 32;

struct RouterScoredArgs {
  const void* logits;  // [T, E] bf16 or fp32
  const float* bias;   // [E] or null
  int32_t* ids;        // [T, K]
  float* weights;      // [T, K]
  int T, E, K;
  int sigmoid, n_group, topk_group, group_top, renormalize;
  float weight_scale;
  int per;        // experts of a lane: ceil(E / 32)
  int size;       // experts of a group
  int group_lanes;  // lanes of a group where groups are whole lanes (kWhole)
  uint32_t group_magic;  // ceil(2^21 / size): expert / size = expert * magic >> 21
};

// Unsigned order of the keys = order of the floats (-infinity .. +infinity);
// -0 counts as +0, as it does in a comparison.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// NaN: score 0, below every number.
__device__ __forceinline__ float router_number(float x) { return x != x ? -INFINITY : x; }

template <bool kFp32>
__device__ __forceinline__ float router_logit(const void* logits, size_t at) {
  return router_number(kFp32 ? __ldg(reinterpret_cast<const float*>(logits) + at)
                             : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(logits)[at]));
}

// 1 / (1 + exp(-x)) with every operation rounded once, so that the order of
// two scores does not depend on how a compiler contracts them.
__device__ __forceinline__ float sigmoid_f32(float x) { return __frcp_rn(__fadd_rn(1.f, expf(-x))); }

// kPer: room for a lane's experts.  kVector: E = 32 kPer and rows of whole
// 16-byte units.  kWhole: a group is a power of two of whole lanes (or all are
// one group), so its rank is found by shuffles; otherwise through shared memory.
template <int kPer, bool kFp32, bool kVector, bool kWhole>
__global__ void __launch_bounds__(RS_WARPS * 32) moe_router_scored_kernel(const RouterScoredArgs a) {
  constexpr uint32_t kAll = 0xffffffffu;
  // choice values of a token, one word of padding per 32 so that lanes that
  // walk groups of 32 experts hit different banks
  __shared__ float s_choice[kWhole ? 1 : RS_WARPS][kWhole ? 1 : kPer * 33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (int)blockIdx.x * RS_WARPS + warp;
  if (t >= a.T) return;  // whole warps leave together
  const int E = a.E, K = a.K, per = kVector ? kPer : a.per, e0 = lane * per;
  const int mine = max(0, min(per, E - e0));  // experts of this lane
  const size_t row = (size_t)t * E;
  const bool by_score = a.bias != nullptr || a.group_top == 2;

  float c[kPer];
  if constexpr (kVector && kFp32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.logits) + row + e0);
#pragma unroll
    for (int q = 0; q < kPer; q += 4) {
      const float4 v = __ldg(p + q / 4);
      c[q] = router_number(v.x), c[q + 1] = router_number(v.y);
      c[q + 2] = router_number(v.z), c[q + 3] = router_number(v.w);
    }
  } else if constexpr (kVector) {
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.logits) + row + e0);
#pragma unroll
    for (int q = 0; q < kPer; q += 8) {
      float v[8];
      unpack_bf16x8(__ldg(p + q / 8), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) c[q + i] = router_number(v[i]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < kPer; ++q) c[q] = q < mine ? router_logit<kFp32>(a.logits, row + e0 + q) : -INFINITY;
  }
  // softmax statistics, where scores of unchosen experts matter; with a logit of
  // +infinity the sum is NaN, and so are the scores and the weights
  float top = 0.f, sum = 1.f;
  if (!a.sigmoid && (by_score || !a.renormalize)) {
    top = c[0];
#pragma unroll
    for (int q = 1; q < kPer; ++q) top = fmaxf(top, c[q]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    if (!(top > -INFINITY)) top = 0.f;  // every logit -infinity or NaN
    sum = 0.f;
#pragma unroll
    for (int q = 0; q < kPer; ++q) sum += expf(c[q] - top);
    sum = warp_sum(sum);
  }
  if (by_score) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      float s = a.sigmoid ? sigmoid_f32(c[q]) : (sum != 0.f ? expf(c[q] - top) / sum : 0.f);
      if (a.bias) s = __fadd_rn(s, __ldg(a.bias + (kVector ? e0 + q : min(e0 + q, E - 1))));
      c[q] = router_number(s);
    }
  }

  // this lane's keys, its best and second best
  uint32_t key[kPer];
  uint32_t best = 0u, best_at = kAll, next = 0u, next_at = kAll;
  auto rank_mine = [&](auto up) {
    best = next = 0u;
    best_at = next_at = kAll;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int e = e0 + q;
      key[q] = (kVector || q < mine) && up(e) ? order_key(c[q]) : 0u;
      const bool first = key[q] > best, second = key[q] > next;
      next_at = first ? best_at : second ? e : next_at;
      next = first ? best : second ? key[q] : next;
      best_at = first ? e : best_at;
      best = first ? key[q] : best;
    }
  };
  if (kWhole || a.n_group == 1) rank_mine([](int) { return true; });

  if (a.n_group > 1) {
    // a group's rank in every lane of its `per_group` lanes
    int per_group, g;
    float rank;
    if constexpr (kWhole) {
      per_group = a.group_lanes;
      g = lane / per_group;
      uint32_t b0 = best, b1 = next;
      for (int o = per_group / 2; o > 0; o >>= 1) {
        const uint32_t o0 = __shfl_xor_sync(kAll, b0, o), o1 = __shfl_xor_sync(kAll, b1, o);
        b1 = max(min(b0, o0), max(b1, o1));
        b0 = max(b0, o0);
      }
      rank = key_value(b0);
      if (a.group_top == 2 && a.size > 1) rank = __fadd_rn(rank, key_value(b1));
    } else {
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const int e = e0 + q;
        if (q < mine) s_choice[warp][e + (e >> 5)] = c[q];
      }
      __syncwarp();
      // a power of two of lanes per group; each finds its two largest values
      per_group = 1;
      while (per_group * 2 * a.n_group <= 32) per_group *= 2;
      g = lane / per_group;
      float b0 = -INFINITY, b1 = -INFINITY;
      if (g < a.n_group) {
        for (int j = lane % per_group; j < a.size; j += per_group) {
          const int e = g * a.size + j;
          const float v = s_choice[warp][e + (e >> 5)];
          b1 = fmaxf(b1, fminf(b0, v));
          b0 = fmaxf(b0, v);
        }
      }
      for (int o = per_group / 2; o > 0; o >>= 1) {
        const float o0 = __shfl_xor_sync(kAll, b0, o), o1 = __shfl_xor_sync(kAll, b1, o);
        b1 = fmaxf(fminf(b0, o0), fmaxf(b1, o1));
        b0 = fmaxf(b0, o0);
      }
      rank = b0;
      if (a.group_top == 2 && a.size > 1) rank = __fadd_rn(b0, b1);
    }
    const uint32_t mine_rank = order_key(rank);
    int ahead = 0;  // groups that go before this lane's
    for (int h = 0; h < a.n_group; ++h) {
      const uint32_t other = __shfl_sync(kAll, mine_rank, h * per_group);
      ahead += other > mine_rank || (other == mine_rank && h < g);
    }
    const bool in = g < a.n_group && ahead < a.topk_group;
    if constexpr (kWhole) {
      if (!in) {
        best = next = 0u;
        best_at = next_at = kAll;
      }
    } else {
      const uint32_t lanes_in = __ballot_sync(kAll, in);
      rank_mine([&](int e) { return (lanes_in >> (((e * a.group_magic) >> 21) * per_group)) & 1u; });
    }
  }

  int id = 0;  // lane k keeps the k-th chosen expert
  bool known = true;  // next is the best of what is left after best
  for (int k = 0; k < K; ++k) {
    const uint32_t most = __reduce_max_sync(kAll, best);
    const uint32_t at = __reduce_min_sync(kAll, best == most ? best_at : kAll);
    if (lane == k) id = (int)at;
    if (best_at == at) {
      if (known) {
        best = next;
        best_at = next_at;
        known = false;
      } else {  // the best of the experts behind the one taken
        const uint32_t taken = best;
        best = 0u;
        best_at = kAll;
#pragma unroll
        for (int q = 0; q < kPer; ++q) {
          const uint32_t e = e0 + q;
          const bool left = key[q] < taken || (key[q] == taken && e > at);
          if (left && key[q] > best) best = key[q], best_at = e;
        }
      }
    }
  }

  // Weights from the chosen logits (still in L1).  A softmax over the chosen
  // alone is taken around their own maximum, so it cannot underflow to 0 / 0.
  const float x = lane < K ? router_logit<kFp32>(a.logits, row + id) : -INFINITY;
  float w = 0.f;
  if (a.sigmoid) {
    w = lane < K ? sigmoid_f32(x) : 0.f;
  } else {
    if (a.renormalize) {
      top = x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      if (!(top > -INFINITY)) top = 0.f;
      if (sum == sum) sum = 1.f;
    }
    w = lane < K && sum != 0.f ? expf(x - top) / sum : 0.f;
  }
  if (a.renormalize) {
    const float den = warp_sum(w);
    w = den != 0.f ? w / den : 1.f / (float)K;
  }
  if (lane < K) {
    a.ids[(size_t)t * K + lane] = id;
    a.weights[(size_t)t * K + lane] = w * a.weight_scale;
  }
}

}  // namespace wdb

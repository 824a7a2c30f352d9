// Expert choice from router logits, sm_100a: softmax or sigmoid scores, a
// balance bias, expert groups, top-k, renormalised weights.  Extends the
// plain softmax router of wd_router.cuh; the reference has no router.
//
// One warp per token; lane l keeps the experts l, l + 32, ... as 32-bit keys
// whose unsigned order is the order of the choice values, so a top-k step is
// two warp reductions in hardware (largest key, then the lowest expert that
// has it).  Key 0 marks what is not up for choice: it lies below the key of
// -infinity.
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
  int logits_fp32, sigmoid, n_group, topk_group, group_top, renormalize;
  float weight_scale;
  uint32_t group_magic;  // ceil(2^21 / experts of a group): expert / size = expert * magic >> 21
};

// Unsigned order of the keys = order of the floats (-infinity .. +infinity);
// -0 counts as +0, as it does in a comparison.
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float router_logit(const RouterScoredArgs& a, size_t at) {
  float x = a.logits_fp32 ? reinterpret_cast<const float*>(a.logits)[at]
                          : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.logits)[at]);
  return x != x ? -INFINITY : x;  // NaN: score 0, below every number
}

// 1 / (1 + exp(-x)) with every operation rounded once, so that the order of
// two scores does not depend on how a compiler contracts them.
__device__ __forceinline__ float sigmoid_f32(float x) { return __frcp_rn(__fadd_rn(1.f, expf(-x))); }

// kPer: experts per lane (E <= 32 * kPer).
template <int kPer>
__global__ void __launch_bounds__(RS_WARPS * 32) moe_router_scored_kernel(const RouterScoredArgs a) {
  constexpr uint32_t kAll = 0xffffffffu;
  // choice values of a token, one word of padding per 32 so that lanes that
  // walk groups of 32 experts hit different banks
  __shared__ float s_choice[RS_WARPS][kPer * 33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (int)blockIdx.x * RS_WARPS + warp;
  if (t >= a.T) return;  // whole warps leave together
  const int E = a.E, K = a.K;
  const size_t row = (size_t)t * E;
  const bool by_score = a.bias != nullptr || a.group_top == 2;

  float c[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int e = lane + 32 * q;
    c[q] = e < E ? router_logit(a, row + e) : -INFINITY;
  }
  // softmax statistics, where scores of unchosen experts matter
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
      float s = a.sigmoid ? sigmoid_f32(c[q]) : (sum > 0.f ? expf(c[q] - top) / sum : 0.f);
      if (a.bias) s = __fadd_rn(s, __ldg(a.bias + min(lane + 32 * q, E - 1)));
      c[q] = s != s ? -INFINITY : s;
    }
  }

  uint32_t kept = kAll;  // bit g: group g stands for choice
  const int size = E / a.n_group;
  if (a.n_group > 1) {
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      const int e = lane + 32 * q;
      if (e < E) s_choice[warp][e + (e >> 5)] = c[q];
    }
    __syncwarp();
    // a power of two of lanes per group; each finds its two largest values
    int per = 1;
    while (per * 2 * a.n_group <= 32) per *= 2;
    const int g = lane / per;
    float b0 = -INFINITY, b1 = -INFINITY;
    if (g < a.n_group) {
      for (int j = lane % per; j < size; j += per) {
        const int e = g * size + j;
        const float v = s_choice[warp][e + (e >> 5)];
        b1 = fmaxf(b1, fminf(b0, v));
        b0 = fmaxf(b0, v);
      }
    }
    for (int o = per / 2; o > 0; o >>= 1) {
      const float o0 = __shfl_xor_sync(kAll, b0, o), o1 = __shfl_xor_sync(kAll, b1, o);
      b1 = fmaxf(fminf(b0, o0), fmaxf(b1, o1));
      b0 = fmaxf(b0, o0);
    }
    float rank = b0;
    if (a.group_top == 2 && size > 1) rank = __fadd_rn(b0, b1);
    const uint32_t mine = order_key(rank);
    int ahead = 0;  // groups that go before mine
    for (int h = 0; h < a.n_group; ++h) {
      const uint32_t other = __shfl_sync(kAll, mine, h * per);
      ahead += other > mine || (other == mine && h < g);
    }
    const bool in = g < a.n_group && lane % per == 0 && ahead < a.topk_group;
    const uint32_t leaders = __ballot_sync(kAll, in);
    kept = 0u;
    for (int h = 0; h < a.n_group; ++h) kept |= ((leaders >> (h * per)) & 1u) << h;
  }

  // Each lane's best and second best; a lane whose best is taken moves its
  // second up, and only one that was taken twice looks through its experts.
  uint32_t key[kPer];
  uint32_t best = 0u, best_at = kAll, next = 0u, next_at = kAll;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int e = lane + 32 * q;
    const bool up = e < E && ((kept >> ((e * a.group_magic) >> 21)) & 1u);
    key[q] = up ? order_key(c[q]) : 0u;
    const bool first = key[q] > best, second = key[q] > next;
    next_at = first ? best_at : second ? e : next_at;
    next = first ? best : second ? key[q] : next;
    best_at = first ? e : best_at;
    best = first ? key[q] : best;
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
          const uint32_t e = lane + 32 * q;
          const bool left = key[q] < taken || (key[q] == taken && e > at);
          if (left && key[q] > best) best = key[q], best_at = e;
        }
      }
    }
  }

  // Weights from the chosen logits (still in L1).  A softmax over the chosen
  // alone is taken around their own maximum, so it cannot underflow to 0 / 0.
  const float x = lane < K ? router_logit(a, row + id) : -INFINITY;
  float w = 0.f;
  if (a.sigmoid) {
    w = lane < K ? sigmoid_f32(x) : 0.f;
  } else {
    if (a.renormalize) {
      top = x;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
      if (!(top > -INFINITY)) top = 0.f;
      sum = 1.f;
    }
    w = lane < K && sum > 0.f ? expf(x - top) / sum : 0.f;
  }
  if (a.renormalize) {
    const float den = warp_sum(w);
    w = den > 0.f ? w / den : 1.f / (float)K;
  }
  if (lane < K) {
    a.ids[(size_t)t * K + lane] = id;
    a.weights[(size_t)t * K + lane] = w * a.weight_scale;
  }
}

}  // namespace wdb

// Attention of a few query tokens per sequence over the FP8 paged cache, on
// the CUDA cores: any head size, one launch, no workspace.  Head sizes 64 and
// 128 run on the tensor cores instead (wd_attn_fp8_tc.cuh).
//
// A block takes up to ATTN_ROWS query rows that share a key head.  A warp walks
// every eighth token, ATTN_AHEAD of them at a time; a lane holds four or eight
// of the head's values (of q, scaled, and of the output), so a token is one
// coalesced read of its codes and a warp sum per row.  Running maximum and sum
// per warp (online softmax: where the maximum rises by x, what was summed so
// far is multiplied by 2^-x), joined over the warps at the end.  Bound by
// latency (look-up, codes and warp sums in turn, no split of a long sequence):
// 16 sequences of 1000 tokens, 32 heads over 4 of 256 values 117 us, 0.28 TB/s;
// with a token at a time 157.
#pragma once

#include "wd_common.cuh"
#include "wd_kv_fp8.cuh"

namespace wdb {

constexpr int ATTN_ROWS = 4;
constexpr int ATTN_WARPS = 8;
constexpr int ATTN_AHEAD = 4;

struct AttnArgs {
  const __nv_bfloat16* q;
  long long q_bs, q_ts, q_hs;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *table, *seq_lens;
  __nv_bfloat16* out;
  float* lse;
  uint32_t* status;
  int table_stride, B, Sq, Hq, Hkv, D, page, pages, window;
  float scale_log2;  // softmax_scale * log2(e)
};

// Length of a sequence; a negative one is none.
__device__ __forceinline__ int attn_length(const AttnArgs& a, int b) { return max(__ldg(a.seq_lens + b), 0); }

// First token that a row sees whose last one is `last`; without a difference that
// could pass 32 bits.
__device__ __forceinline__ int attn_first(int last, int window) {
  return window > 0 && last >= window ? last - window + 1 : 0;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__global__ void __launch_bounds__(ATTN_WARPS * 32) attn_fp8_simt_kernel(const AttnArgs a) {
  __shared__ float s_m[ATTN_WARPS][ATTN_ROWS], s_l[ATTN_WARPS][ATTN_ROWS];
  __shared__ float s_o[ATTN_WARPS][KV_MAX_D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.Hq / a.Hkv, rows_all = a.Sq * G;
  const int chunks = (rows_all + ATTN_ROWS - 1) / ATTN_ROWS;
  int u = blockIdx.x;
  const int r0 = (u % chunks) * ATTN_ROWS;
  u /= chunks;
  const int h = u % a.Hkv, b = u / a.Hkv;
  const int len = attn_length(a, b);
  const int reach = (int)min((long long)a.table_stride * a.page, 0x7fffffffll - 128);
  const int n4 = a.D / 4;
  const bool has[2] = {lane < n4, lane + 32 < n4};

  float q[ATTN_ROWS][8], o[ATTN_ROWS][8], m[ATTN_ROWS], l[ATTN_ROWS];
  int hi[ATTN_ROWS], lo[ATTN_ROWS];  // tokens that a row sees: [lo, hi]
  int from = 0x7fffffff, to = -1;
#pragma unroll
  for (int r = 0; r < ATTN_ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    const int row = r0 + r, i = row / G, head = h * G + row % G;
    const bool on = row < rows_all;
    hi[r] = on ? min(len - a.Sq + i, len - 1) : -1;
    lo[r] = attn_first(hi[r], a.window);
    if (hi[r] >= reach) {  // tokens past the table's last column
      if (threadIdx.x == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
      hi[r] = reach - 1;
    }
    if (hi[r] >= lo[r]) {
      from = min(from, lo[r]);
      to = max(to, hi[r]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      o[r][j] = 0.f;
      const int d = 4 * (lane + 32 * (j / 4)) + j % 4;
      q[r][j] = on && has[j / 4] ? __bfloat162float(a.q[(long long)b * a.q_bs + (long long)i * a.q_ts +
                                                       (long long)head * a.q_hs + d]) * a.scale_log2
                                 : 0.f;
      // an infinite q makes its row NaN, as on the tensor cores: scores that are all
      // -infinity would pass for keys that are not seen
      if (fabsf(q[r][j]) == INFINITY) q[r][j] = __uint_as_float(0x7fc00000u);
    }
  }
  if (to < 0) from = 0;  // no row sees a token: the loop below must not start at INT_MAX + warp
  for (int t0 = from + warp; t0 <= to; t0 += ATTN_WARPS * ATTN_AHEAD) {
    // ATTN_AHEAD tokens' pages, then all their scales and codes in flight together
    uint32_t kw[ATTN_AHEAD][2], vw[ATTN_AHEAD][2];
    float ks[ATTN_AHEAD], vs[ATTN_AHEAD];
    int pid[ATTN_AHEAD];
#pragma unroll
    for (int u = 0; u < ATTN_AHEAD; ++u) {
      const int t = t0 + u * ATTN_WARPS;
      pid[u] = -1;
      if (t > to) continue;
      pid[u] = __ldg(a.table + (size_t)b * a.table_stride + t / a.page);
      if (pid[u] < 0 || pid[u] >= a.pages) {
        pid[u] = -1;
        if (lane == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
      }
    }
#pragma unroll
    for (int u = 0; u < ATTN_AHEAD; ++u) {
      const size_t ph = (size_t)max(pid[u], 0) * a.Hkv + h;
      const size_t off = (ph * a.page + (t0 + u * ATTN_WARPS) % a.page) * a.D;
      ks[u] = vs[u] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) kw[u][half] = vw[u][half] = 0u;
      if (pid[u] < 0) continue;
      ks[u] = ue8m0_to_f32(__ldg(a.ks + ph));
      vs[u] = ue8m0_to_f32(__ldg(a.vs + ph));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!has[half]) continue;
        kw[u][half] = __ldg(reinterpret_cast<const uint32_t*>(a.kc + off) + lane + 32 * half);
        vw[u][half] = __ldg(reinterpret_cast<const uint32_t*>(a.vc + off) + lane + 32 * half);
      }
    }
    // all scores, so that their sums over the lanes overlap
    float x[ATTN_AHEAD][ATTN_ROWS];
#pragma unroll
    for (int u = 0; u < ATTN_AHEAD; ++u) {
      float k[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float2 k0 = e4m3x2_to_f32(kw[u][half] & 0xffffu), k1 = e4m3x2_to_f32(kw[u][half] >> 16);
        k[4 * half] = k0.x, k[4 * half + 1] = k0.y, k[4 * half + 2] = k1.x, k[4 * half + 3] = k1.y;
      }
#pragma unroll
      for (int r = 0; r < ATTN_ROWS; ++r) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(q[r][j], k[j], sum);
        x[u][r] = sum;
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int u = 0; u < ATTN_AHEAD; ++u)
#pragma unroll
        for (int r = 0; r < ATTN_ROWS; ++r) x[u][r] += __shfl_xor_sync(0xffffffffu, x[u][r], off);
    // weights of a row's unseen tokens are 0; its maximum rises once for all
    uint32_t seen = 0u;
#pragma unroll
    for (int r = 0; r < ATTN_ROWS; ++r) {
      float top = m[r];
#pragma unroll
      for (int u = 0; u < ATTN_AHEAD; ++u) {
        const int t = t0 + u * ATTN_WARPS;
        const bool sees = pid[u] >= 0 && t >= lo[r] && t <= hi[r];
        seen |= (uint32_t)sees << (u * ATTN_ROWS + r);
        x[u][r] = sees ? x[u][r] * ks[u] : -INFINITY;
        top = fmaxf(top, x[u][r]);
      }
      const float f = m[r] == top ? 1.f : ex2_approx(m[r] - top);
      m[r] = top;
      l[r] *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[r][j] *= f;
#pragma unroll
      for (int u = 0; u < ATTN_AHEAD; ++u) {
        // a score of -infinity (or none above it yet) weighs nothing; NaN stays
        x[u][r] = x[u][r] == -INFINITY ? 0.f : ex2_approx(x[u][r] - top);
        l[r] += x[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < ATTN_AHEAD; ++u) {
      float v[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float2 v0 = e4m3x2_to_f32(vw[u][half] & 0xffffu), v1 = e4m3x2_to_f32(vw[u][half] >> 16);
        v[4 * half] = v0.x, v[4 * half + 1] = v0.y, v[4 * half + 2] = v1.x, v[4 * half + 3] = v1.y;
      }
#pragma unroll
      for (int r = 0; r < ATTN_ROWS; ++r) {
        if (!((seen >> (u * ATTN_ROWS + r)) & 1u)) continue;  // 0 times NaN; the same in every lane
        const float pv = x[u][r] * vs[u];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[r][j] = fmaf(pv, v[j], o[r][j]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ATTN_ROWS; ++r)
    if (lane == 0) s_m[warp][r] = m[r], s_l[warp][r] = l[r];
#pragma unroll
  for (int r = 0; r < ATTN_ROWS; ++r) {
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < ATTN_WARPS; ++w) top = fmaxf(top, s_m[w][r]);
    const float f = m[r] == -INFINITY ? 1.f : ex2_approx(m[r] - top);  // l = o = 0 (or NaN) at -infinity
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (has[j / 4]) s_o[warp][4 * (lane + 32 * (j / 4)) + j % 4] = o[r][j] * f;
    __syncthreads();
    const int row = r0 + r, i = row / G, head = h * G + row % G;
    if (row >= rows_all) continue;
    float den = 0.f;
    for (int w = 0; w < ATTN_WARPS; ++w)
      den += s_l[w][r] * (s_m[w][r] == -INFINITY ? 1.f : ex2_approx(s_m[w][r] - top));
    const size_t at = ((size_t)b * a.Sq + i) * a.Hq + head;
    for (int d = threadIdx.x; d < a.D; d += ATTN_WARPS * 32) {
      float y = 0.f;
      for (int w = 0; w < ATTN_WARPS; ++w) y += s_o[w][d];
      a.out[at * a.D + d] = __float2bfloat16_rn(den == 0.f ? 0.f : y / den);
    }
    if (a.lse && threadIdx.x == 0)
      a.lse[at] = den == 0.f ? -INFINITY : (top == -INFINITY ? 0.f : top * 0.6931471805599453f) + logf(den);
  }
}

}  // namespace wdb

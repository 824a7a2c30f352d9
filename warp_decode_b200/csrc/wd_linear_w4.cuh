// Projection of a few tokens with 4-bit weights, sm_100a:
//   out[t, n] = sum_k x[t, k] (code[n, k] - zero[n, k / g]) scale[n, k / g]
// No counterpart in the reference.
//
// Codes become bf16 by bits (128 + code is bf16 0x4300 | code), the zero point is
// taken off there, exactly, and the whole numbers meet x in matrix instructions;
// a group's scale multiplies its fp32 sum, so nothing is rounded before the end.
//
// A row's codes lie in blocks of 128 (64 bytes): word 4 t + s of a block holds
// the codes of k = 32 s + 8 t + 0..7, the even ones in the low half.  Lane 4 g + t
// of a warp so reads 16 bytes of row g that are its operands of eight matrix
// instructions (sixteen k each, four of them this lane's), two for each 32 k, with
// x as it lies in memory: the order of k within a product is the same on both
// sides.  No shuffle, no shared memory before the sums.
//
// Measured (B200): one token, 4096 to 9216 (19 MB) 13.9 us, where a kernel that only
// reads those bytes cold takes 12.3; 4096 to 512 6.2, as a launch that does nothing.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "wd_tc.cuh"

namespace wdb {

constexpr int W4_WARPS = 8;      // of a block, each its share of k
constexpr int W4_MAX_SPLIT = 8;  // blocks of a cluster that share k

struct LinearW4Args {
  const __nv_bfloat16* x;
  const uint8_t* w;
  const void* scale;
  const uint8_t* zero;  // or NULL: 8
  __nv_bfloat16* out;
  long long x_ts, o_ts;  // token strides
  int T, N, K, blocks;   // blocks of 128 k
  int groups;            // of a row
  int x_wide;            // x's rows are 16-byte aligned
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two codes (bits 0..3 and 16..19 of `word` >> 4 j) less their zero point, as bf16.
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int j, __nv_bfloat162 zero128) {
  const uint32_t c = ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), zero128);
  return *reinterpret_cast<const uint32_t*>(&v);
}

enum W4ScaleType { W4_BF16 = 0, W4_F16 = 1, W4_F32 = 2 };

template <int kScale, typename Raw>
__device__ __forceinline__ float w4_value(Raw raw) {
  if constexpr (kScale == W4_F32)
    return raw;
  else if constexpr (kScale == W4_F16)
    return __half2float(__ushort_as_half(raw));
  else
    return __uint_as_float((uint32_t)raw << 16);
}

template <int kScale>
__device__ __forceinline__ float w4_scale(const void* p, size_t at) {
  if constexpr (kScale == W4_F32)
    return __ldg(static_cast<const float*>(p) + at);
  else
    return w4_value<kScale>(__ldg(static_cast<const uint16_t*>(p) + at));
}

// A block: 16 kRows output rows of up to 8 kTokens tokens, k split over its warps
// and over the blocks of its cluster; sums joined in that order.
template <int kRows, int kTokens, int kGroup, int kScale>
__global__ void __launch_bounds__(W4_WARPS * 32) linear_w4_kernel(const LinearW4Args a) {
  constexpr int kR = 16 * kRows, kT = 8 * kTokens;
  __shared__ float s_sum[W4_WARPS][kT][kR + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int rank = (int)cluster_ctarank(), ranks = gridDim.x;
  const int n0 = blockIdx.y * kR, t0 = blockIdx.z * kT;
  const int parts = ranks * W4_WARPS, part = rank * W4_WARPS + warp;
  const int first = (int)((long long)a.blocks * part / parts), last = (int)((long long)a.blocks * (part + 1) / parts);

  float acc[kRows][kTokens][4];
#pragma unroll
  for (int m = 0; m < kRows; ++m)
#pragma unroll
    for (int n = 0; n < kTokens; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;

  int row[kRows][2];
#pragma unroll
  for (int m = 0; m < kRows; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h) row[m][h] = min(n0 + m * 16 + h * 8 + g, a.N - 1);  // rows past the last: its copy
  const __nv_bfloat16* x[kTokens];
  bool live[kTokens];
#pragma unroll
  for (int n = 0; n < kTokens; ++n) {
    live[n] = t0 + n * 8 + g < a.T;
    x[n] = a.x + (long long)(live[n] ? t0 + n * 8 + g : 0) * a.x_ts + 8 * t4;
  }
  auto codes = [&](int m, int h, int b) {
    return __ldcs(reinterpret_cast<const uint4*>(a.w + ((size_t)row[m][h] * a.blocks + b) * 64) + t4);
  };
#pragma unroll 2
  for (int b = first; b < last; ++b) {
    uint4 w[kRows][2];
#pragma unroll
    for (int m = 0; m < kRows; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) w[m][h] = codes(m, h, b);
    float part_sum[kRows][kTokens][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = b * 128 + s * 32;
      if (k >= a.K) break;  // K is a multiple of 32
      constexpr int kSteps = kGroup / 32;
      const int group = (b * 128) / kGroup + s / kSteps;
      uint4 xv[kTokens];
#pragma unroll
      for (int n = 0; n < kTokens; ++n) {
        xv[n] = make_uint4(0u, 0u, 0u, 0u);
        if (live[n]) {
          if (a.x_wide) {
            xv[n] = __ldg(reinterpret_cast<const uint4*>(x[n] + k));
          } else {
            uint32_t v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __bfloat16_as_ushort(x[n][k + i]);
            xv[n] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
          }
        }
      }
      if (s % kSteps == 0) {
#pragma unroll
        for (int m = 0; m < kRows; ++m)
#pragma unroll
          for (int n = 0; n < kTokens; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) part_sum[m][n][i] = 0.f;
      }
#pragma unroll
      for (int m = 0; m < kRows; ++m) {
        __nv_bfloat162 z[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float zero = a.zero ? (float)__ldg(a.zero + (size_t)row[m][h] * a.groups + group) : 8.f;
          z[h] = __float2bfloat162_rn(128.f + fminf(zero, 127.f));
        }
        const uint32_t w0[4] = {w[m][0].x, w[m][0].y, w[m][0].z, w[m][0].w};
        const uint32_t w1[4] = {w[m][1].x, w[m][1].y, w[m][1].z, w[m][1].w};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t f[4] = {w4_pair(w0[s], 2 * half, z[0]), w4_pair(w1[s], 2 * half, z[1]),
                                 w4_pair(w0[s], 2 * half + 1, z[0]), w4_pair(w1[s], 2 * half + 1, z[1])};
#pragma unroll
          for (int n = 0; n < kTokens; ++n)
            mma_bf16(part_sum[m][n], f, half ? xv[n].z : xv[n].x, half ? xv[n].w : xv[n].y);
        }
      }
      if (s % kSteps == kSteps - 1 || k + 32 >= a.K) {
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
          const float f0 = w4_scale<kScale>(a.scale, (size_t)row[m][0] * a.groups + group);
          const float f1 = w4_scale<kScale>(a.scale, (size_t)row[m][1] * a.groups + group);
#pragma unroll
          for (int n = 0; n < kTokens; ++n) {
            acc[m][n][0] = fmaf(part_sum[m][n][0], f0, acc[m][n][0]);
            acc[m][n][1] = fmaf(part_sum[m][n][1], f0, acc[m][n][1]);
            acc[m][n][2] = fmaf(part_sum[m][n][2], f1, acc[m][n][2]);
            acc[m][n][3] = fmaf(part_sum[m][n][3], f1, acc[m][n][3]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kRows; ++m)
#pragma unroll
    for (int n = 0; n < kTokens; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s_sum[warp][n * 8 + 2 * t4 + (i & 1)][m * 16 + g + 8 * (i >> 1)] = acc[m][n][i];
  __syncthreads();
  // this block's sums into its first warp's place, then a share of all blocks' sums
  for (int e = threadIdx.x; e < kT * kR; e += W4_WARPS * 32) {
    const int t = e / kR, n = e % kR;
    float sum = s_sum[0][t][n];
#pragma unroll
    for (int i = 1; i < W4_WARPS; ++i) sum += s_sum[i][t][n];
    if (ranks > 1)
      s_sum[0][t][n] = sum;
    else if (t0 + t < a.T && n0 + n < a.N)
      a.out[(t0 + t) * a.o_ts + n0 + n] = __float2bfloat16_rn(sum);
  }
  if (ranks > 1) {
    cluster_sync();
    for (int e = threadIdx.x + rank * W4_WARPS * 32; e < kT * kR; e += ranks * W4_WARPS * 32) {
      const int t = e / kR, n = e % kR;
      if (t0 + t >= a.T || n0 + n >= a.N) continue;
      float sum = 0.f;
      for (int i = 0; i < ranks; ++i) sum += dsmem_ld_f32(dsmem_addr(&s_sum[0][t][n], i));
      a.out[(t0 + t) * a.o_ts + n0 + n] = __float2bfloat16_rn(sum);
    }
    cluster_sync();
  }
}

}  // namespace wdb

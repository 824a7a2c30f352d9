// The step between two blocks of a decoder layer, sm_100a: a block's output,
// normed if asked, gated onto the scaled residual stream, and the norm before
// the next block, in one pass over the row.  No counterpart in the reference.
//
//   z = y                                     or  y rsqrt(mean y^2 + eps) post_weight
//   r' = residual_scale r + gate z
//   x = r' rsqrt(mean r'^2 + eps) norm_weight
//
// A row stays in the registers of its threads from the loads to both stores, so
// y and r are read once and r' and x written once: bound by HBM where there are
// many rows, by one round of loads and the block's sums where there are few.
// The second norm takes r' before it is rounded.
//
// Many long rows: blocks that stay, as many as an SM has threads for, and copy their next rows to
// shared memory while they work on one (block_norm_stream_kernel): 8192 rows of 4096
// with both norms and a channel gate 53.0 us, 5.1 TB/s (cold 55, a block a row 64); 1999
// rows on an fp32 residual 20.9 us, 4.7 TB/s.  Rows off the 16-byte grid go value by value,
// a block a row: 2000 of 4096 39 us cold, 21 on the grid.  Few rows take what a launch takes: 64 rows of
// 7168 6 us.
#pragma once

#include "wd_common.cuh"
#include "wd_qk_rope.cuh"

namespace wdb {

constexpr int BN_MAX_THREADS = 1024;
constexpr int BN_MAX_H = 16384;  // 1024 threads of two units of eight values
constexpr int BN_MAX_STAGES = 4;
constexpr int BN_WARP_ROWS = 4;  // rows of a block whose rows are a warp each

struct BlockNormArgs {
  const __nv_bfloat16* y;
  const void *r, *gate, *norm_w, *post_w;  // gate, post_w: or NULL
  __nv_bfloat16* x;
  void* r_out;
  long long y_ts, r_ts, g_ts, x_ts, ro_ts;  // token strides
  int T, H;
  int weight_fp32, gate_fp32, gate_per_token;  // gate_per_token: one value a token
  float scale, eps;
  int stages;  // of block_norm_stream_kernel: rows in shared memory
};

// Eight consecutive values (kVector, 16-byte aligned) or eight a block apart.
template <bool kVector, bool kFp32>
__device__ __forceinline__ void bn_load(const void* p, int at, int step, int H, float (&v)[8]) {
  if constexpr (kVector) {
    if constexpr (kFp32) {
      const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
      const float4 a = s[0], b = s[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at), v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = at + i * step;
      v[i] = 0.f;
      if (e < H) {
        if constexpr (kFp32)
          v[i] = static_cast<const float*>(p)[e];
        else
          v[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
      }
    }
  }
}

template <bool kVector, bool kFp32>
__device__ __forceinline__ void bn_store(void* p, int at, int step, int H, const float (&v)[8]) {
  if constexpr (kVector) {
    if constexpr (kFp32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&two);
      }
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int e = at + i * step;
      if (e >= H) continue;
      if constexpr (kFp32)
        static_cast<float*>(p)[e] = v[i];
      else
        static_cast<__nv_bfloat16*>(p)[e] = __float2bfloat16_rn(v[i]);
    }
  }
}

// A channel's factor, in either of two types.
template <bool kVector>
__device__ __forceinline__ void bn_load_as(int fp32, const void* p, int at, int step, int H, float (&v)[8]) {
  if (fp32)
    bn_load<kVector, true>(p, at, step, H, v);
  else
    bn_load<kVector, false>(p, at, step, H, v);
}

// Sum over the row's threads: a warp, or the block (every thread calls it).
template <bool kWarp>
__device__ __forceinline__ float bn_row_sum(float v, float* s_part) {
  v = warp_sum(v);
  if constexpr (!kWarp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) s_part[warp] = v;
    __syncthreads();
    v = warp_sum(lane < warps ? s_part[lane] : 0.f);
  }
  return v;
}

// A row in the registers of its threads: z and res hold y and r, and sums are kWarp's or
// the block's; `first` and `second` are rooms for them.
template <int kUnits, bool kVector, bool kFp32, bool kWarp>
__device__ __forceinline__ void bn_row(const BlockNormArgs& a, long long t, int lane, int lanes, float (&z)[kUnits][8],
                                       float (&res)[kUnits][8], float* first, float* second) {
  const float inv_h = 1.f / (float)a.H;
  const int size = kFp32 ? 4 : 2, step = kVector ? 1 : lanes;
  auto at = [&](int u) { return kVector ? (u * lanes + lane) * 8 : u * lanes * 8 + lane; };
  if (a.post_w) {
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(z[u][i], z[u][i], sum);
    const float f = rsqrtf(fmaf(bn_row_sum<kWarp>(sum, first), inv_h, a.eps));
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (at(u) >= a.H) continue;
      float w[8];
      bn_load_as<kVector>(a.weight_fp32, a.post_w, at(u), step, a.H, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[u][i] = z[u][i] * f * w[i];
    }
  }
  if (a.gate) {
    const char* gate = static_cast<const char*>(a.gate) + t * a.g_ts * (a.gate_fp32 ? 4 : 2);
    if (a.gate_per_token) {
      const float g = a.gate_fp32 ? *reinterpret_cast<const float*>(gate)
                                  : __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(gate));
#pragma unroll
      for (int u = 0; u < kUnits; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) z[u][i] *= g;
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (at(u) >= a.H) continue;
        float g[8];
        bn_load_as<kVector>(a.gate_fp32, gate, at(u), step, a.H, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[u][i] *= g[i];
      }
    }
  }
  float sum = 0.f;
  char* ro = static_cast<char*>(a.r_out) + t * a.ro_ts * size;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    if (at(u) >= a.H) continue;  // (an infinite token gate would make NaN of what lies past the row)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      res[u][i] = fmaf(res[u][i], a.scale, z[u][i]);
      if (kVector || at(u) + i * step < a.H) sum = fmaf(res[u][i], res[u][i], sum);
    }
    bn_store<kVector, kFp32>(ro, at(u), step, a.H, res[u]);
  }
  const float f = rsqrtf(fmaf(bn_row_sum<kWarp>(sum, second), inv_h, a.eps));
  __nv_bfloat16* x = a.x + t * a.x_ts;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    if (at(u) >= a.H) continue;
    float w[8];
    bn_load_as<kVector>(a.weight_fp32, a.norm_w, at(u), step, a.H, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = res[u][i] * f * w[i];
    bn_store<kVector, false>(x, at(u), step, a.H, w);
  }
}

// kUnits units of eight values a thread; kWarp: a row is a warp's, else a block's.
template <int kUnits, bool kVector, bool kFp32, bool kWarp>
__global__ void __launch_bounds__(kWarp ? 32 * BN_WARP_ROWS : BN_MAX_THREADS)
    block_norm_kernel(const BlockNormArgs a) {
  __shared__ float s_part[2][32];
  const int lane = kWarp ? threadIdx.x & 31 : threadIdx.x, lanes = kWarp ? 32 : blockDim.x;
  const int t = kWarp ? blockIdx.x * BN_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  if (kWarp && t >= a.T) return;
  const __nv_bfloat16* y = a.y + t * a.y_ts;
  const int size = kFp32 ? 4 : 2;
  const char* r = static_cast<const char*>(a.r) + t * a.r_ts * size;
  // unit u of a thread: eight values from `at(u)`, `step` apart
  const int step = kVector ? 1 : lanes;
  auto at = [&](int u) { return kVector ? (u * lanes + lane) * 8 : u * lanes * 8 + lane; };

  float z[kUnits][8], res[kUnits][8];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    if (at(u) < a.H) {
      bn_load<kVector, false>(y, at(u), step, a.H, z[u]);
      bn_load<kVector, kFp32>(r, at(u), step, a.H, res[u]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[u][i] = res[u][i] = 0.f;
    }
  }
  bn_row<kUnits, kVector, kFp32, kWarp>(a, t, lane, lanes, z, res, s_part[0], s_part[1]);
}

// Rows blockIdx.x, blockIdx.x + gridDim.x, ...: `stages` of them on their way at once.
// A thread has the same channels of every row, so the channels' factors stay in its
// registers: those of z (post_weight and a gate of channels, as one product) in fp32,
// norm_weight as it is stored (one in fp32 is read again for every row). Read for
// every row, the three cost as much as the row itself (8192 rows of 4096: norm alone 50
// us, with post_weight 60, and a gate 72).
template <bool kFp32, bool kWeightFp32>
__global__ void __launch_bounds__(512) block_norm_stream_kernel(const BlockNormArgs a) {
  constexpr int kUnits = 4;
  __shared__ float s_part[4][32];
  __shared__ uint64_t s_full[BN_MAX_STAGES];
  extern __shared__ uint4 s_rows[];  // [stages]: y, r
  const int tid = threadIdx.x, size = kFp32 ? 4 : 2;
  const uint32_t y_bytes = 2u * a.H, row_bytes = y_bytes + (uint32_t)size * a.H;
  const bool channel_gate = a.gate && !a.gate_per_token && a.g_ts == 0, row_gate = a.gate && !channel_gate;
  uint8_t* rows = reinterpret_cast<uint8_t*>(s_rows);
  auto load = [&](long long t, int stage) {  // by one thread
    uint8_t* to = rows + (size_t)stage * row_bytes;
    mbar_arrive_expect_tx(s_full + stage, row_bytes);
    bulk_g2s_big(to, a.y + t * a.y_ts, y_bytes, s_full + stage, l2_policy_evict_first());
    bulk_g2s_big(to + y_bytes, static_cast<const char*>(a.r) + t * a.r_ts * size, row_bytes - y_bytes, s_full + stage,
                 l2_policy_evict_first());
  };
  if (tid == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(s_full + i, 1);
    fence_mbar_init();
    for (int i = 0; i < a.stages; ++i) {
      const long long t = blockIdx.x + (long long)i * gridDim.x;
      if (t < a.T) load(t, i);
    }
  }
  auto at = [&](int u) { return (u * (int)blockDim.x + tid) * 8; };
  auto pairs = [](const float (&v)[8], f32x2 (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = pack2(v[2 * i], v[2 * i + 1]);
  };
  f32x2 c[kUnits][4];
  uint4 w[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float p[8], g[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = g[i] = 1.f;
    w[u] = make_uint4(0u, 0u, 0u, 0u);
    if (at(u) < a.H) {
      if (a.post_w) bn_load<true, kWeightFp32>(a.post_w, at(u), 1, a.H, p);
      if (channel_gate) bn_load_as<true>(a.gate_fp32, a.gate, at(u), 1, a.H, g);
      if (!kWeightFp32) w[u] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.norm_w) + at(u));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] *= g[i];
    pairs(p, c[u]);
  }
  __syncthreads();
  const float inv_h = 1.f / (float)a.H;
  const f32x2 scale = pack2(a.scale, a.scale);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x) {
    if (!mbar_wait(s_full + stage, phase) && tid == 0) raise_status(nullptr, WD_STATUS_WAIT_TIMEOUT);
    const uint8_t* from = rows + (size_t)stage * row_bytes;
    f32x2 res[kUnits][4], zero = pack2(0.f, 0.f), sum = zero;
    float f = 1.f;
    if (a.post_w) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        if (at(u) >= a.H) continue;
        float y[8];
        f32x2 y2[4];
        bn_load<true, false>(from, at(u), 1, a.H, y);
        pairs(y, y2);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum = fma2(y2[i], y2[i], sum);
      }
      f = rsqrtf(fmaf(bn_row_sum<false>(unpack2(sum).x + unpack2(sum).y, s_part[turn]), inv_h, a.eps));
    }
    const char* gate = static_cast<const char*>(a.gate) + (row_gate ? t * a.g_ts * (a.gate_fp32 ? 4 : 2) : 0);
    if (row_gate && a.gate_per_token)
      f *= a.gate_fp32 ? *reinterpret_cast<const float*>(gate)
                       : __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(gate));
    const f32x2 f2 = pack2(f, f);
    char* ro = static_cast<char*>(a.r_out) + t * a.ro_ts * size;
    sum = zero;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (at(u) >= a.H) continue;
      float y[8], r[8];
      f32x2 y2[4], r2[4];
      bn_load<true, false>(from, at(u), 1, a.H, y);
      bn_load<true, kFp32>(from + y_bytes, at(u), 1, a.H, r);
      pairs(y, y2);
      pairs(r, r2);
#pragma unroll
      for (int i = 0; i < 4; ++i) y2[i] = mul2(mul2(y2[i], f2), c[u][i]);
      if (row_gate && !a.gate_per_token) {
        float g[8];
        f32x2 g2[4];
        bn_load_as<true>(a.gate_fp32, gate, at(u), 1, a.H, g);
        pairs(g, g2);
#pragma unroll
        for (int i = 0; i < 4; ++i) y2[i] = mul2(y2[i], g2[i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        res[u][i] = fma2(r2[i], scale, y2[i]);
        sum = fma2(res[u][i], res[u][i], sum);
        r[2 * i] = unpack2(res[u][i]).x, r[2 * i + 1] = unpack2(res[u][i]).y;
      }
      bn_store<true, kFp32>(ro, at(u), 1, a.H, r);
    }
    const float fx = rsqrtf(fmaf(bn_row_sum<false>(unpack2(sum).x + unpack2(sum).y, s_part[turn + 1]), inv_h, a.eps));
    const long long next = t + (long long)a.stages * gridDim.x;
    if (tid == 0 && next < a.T) {  // every thread has read the row
      fence_proxy_async_smem();
      load(next, stage);
    }
    const f32x2 fx2 = pack2(fx, fx);
    __nv_bfloat16* x = a.x + t * a.x_ts;
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      if (at(u) >= a.H) continue;
      float v[8];
      if constexpr (kWeightFp32)
        bn_load<true, true>(a.norm_w, at(u), 1, a.H, v);
      else
        unpack_bf16x8(w[u], v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 o = unpack2(mul2(mul2(res[u][i], fx2), pack2(v[2 * i], v[2 * i + 1])));
        v[2 * i] = o.x, v[2 * i + 1] = o.y;
      }
      bn_store<true, false>(x, at(u), 1, a.H, v);
    }
    turn ^= 2;  // rooms of their own for the sums of consecutive rows
    if (++stage == a.stages) stage = 0, phase ^= 1u;
  }
}

}  // namespace wdb

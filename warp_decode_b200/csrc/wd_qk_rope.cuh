// RMS norm of every query and key head with the position rotation in the same
// pass, sm_100a.  No counterpart in the reference.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)
//
// Bound by memory: each value is read and written once.  A row (one head of
// one token) belongs to a group of lanes, each holding values that rotate with
// each other, so the pairs of both conventions meet inside a lane and the only
// exchange is the sum of squares.
#pragma once

#include "wd_common.cuh"

namespace wdb {

constexpr int QK_THREADS = 256;
constexpr int QK_MAX_D = 256;

struct QkRopeArgs {
  const __nv_bfloat16 *q, *k;
  __nv_bfloat16 *qo, *ko;
  long long q_ts, q_hs, k_ts, k_hs, qo_ts, qo_hs, ko_ts, ko_hs;
  const void *qw, *kw;
  const int32_t* pos;
  const float* cos_sin;
  uint32_t* status;
  int T, Hq, Hkv, D, rot, max_pos;
  int weight_fp32, interleaved;
  int lanes;  // lanes of a row: a power of two
  float eps;
};

template <int kV>
struct Chunk {
  float v[kV];
};

template <int kV>
__device__ __forceinline__ Chunk<kV> load_bf16(const __nv_bfloat16* p) {
  Chunk<kV> c;
  if constexpr (kV == 8) {
    unpack_bf16x8(*reinterpret_cast<const uint4*>(p), c.v);
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) c.v[i] = __bfloat162float(p[i]);
  }
  return c;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int kV>
__device__ __forceinline__ Chunk<kV> load_f32(const float* p) {
  Chunk<kV> c;
  if constexpr (kV == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    c.v[0] = a.x; c.v[1] = a.y; c.v[2] = a.z; c.v[3] = a.w;
    c.v[4] = b.x; c.v[5] = b.y; c.v[6] = b.z; c.v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) c.v[i] = __ldg(p + i);
  }
  return c;
}

template <int kV>
__device__ __forceinline__ Chunk<kV> load_weight(const void* w, int fp32, int at) {
  if (fp32) return load_f32<kV>(reinterpret_cast<const float*>(w) + at);
  return load_bf16<kV>(reinterpret_cast<const __nv_bfloat16*>(w) + at);
}

// Packed pairs of fp32 (sm_100 multiplies and adds two at once).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The wide form: 16-byte accesses, where D and every address are multiples of
// 8 values and the rotated halves of 8 (rot of 16).  A lane holds two chunks
// of 8 values and, for all its rows, two factors of each value, so that a row
// costs two products a value and one with its norm:
//   out_j = inv * (x_j A_j + x_partner(j) B_j),  A = w cos, B = -+ w_partner sin
// kHeads: heads of one kind (queries or keys) that a lane group takes, loaded
// together.  Bound by HBM's mixed reads and writes and the loads in flight (two
// blocks of 100 registers a thread): 8192 tokens of 36 heads of 128 values (155
// MB) 34.3 us, 4.5 TB/s; one head at a time in scalar arithmetic took 57.7,
// four 46.1; eight heads a group of lanes of half the width 37.0.
template <int kHeads, bool kInterleaved>
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_wide_kernel(const QkRopeArgs a) {
  const int per_block = QK_THREADS / a.lanes;
  const int sub = threadIdx.x % a.lanes;
  const int q_parts = (a.Hq + kHeads - 1) / kHeads, parts = q_parts + (a.Hkv + kHeads - 1) / kHeads;
  const long long group = (long long)blockIdx.x * per_block + threadIdx.x / a.lanes;
  const int t = (int)(group / parts), part = (int)(group - (long long)t * parts);
  const bool is_q = part < q_parts, live = t < a.T;  // idle lanes stay for the shuffles
  const int h0 = (is_q ? part : part - q_parts) * kHeads, heads = live ? min(kHeads, (is_q ? a.Hq : a.Hkv) - h0) : 0;
  const int half = a.rot / 2;
  const bool on0 = sub * 16 < a.D, turns = sub * 8 < half;
  const int at0 = turns && !kInterleaved ? sub * 8 : sub * 16;
  const int at1 = turns && !kInterleaved ? half + sub * 8 : sub * 16 + 8;
  const bool on1 = on0 && at1 < a.D;
  int pos = 0;  // its load flies while the rows' do
  if (live) pos = a.pos[t];
  const __nv_bfloat16* src = is_q ? a.q + (size_t)t * a.q_ts + (size_t)h0 * a.q_hs
                                  : a.k + (size_t)t * a.k_ts + (size_t)h0 * a.k_hs;
  const size_t src_hs = is_q ? a.q_hs : a.k_hs;
  uint4 raw0[kHeads], raw1[kHeads];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    raw0[k] = raw1[k] = make_uint4(0u, 0u, 0u, 0u);
    if (k < heads && on0) raw0[k] = *reinterpret_cast<const uint4*>(src + k * src_hs + at0);
    if (k < heads && on1) raw1[k] = *reinterpret_cast<const uint4*>(src + k * src_hs + at1);
  }
  const bool good = pos >= 0 && pos < a.max_pos;
  if (live && !good && sub == 0) raise_status(a.status, WD_STATUS_BAD_POSITION);
  // the factors of this lane's values
  f32x2 A0[4], A1[4], B0[4], B1[4];
  {
    const void* w = is_q ? a.qw : a.kw;
    Chunk<8> w0{}, w1{}, c{}, s{};
    if (heads > 0 && on0) w0 = load_weight<8>(w, a.weight_fp32, at0);
    if (heads > 0 && on1) w1 = load_weight<8>(w, a.weight_fp32, at1);
    if (turns && good && heads > 0) {
      const float* angle = a.cos_sin + (size_t)pos * a.rot + sub * 8;
      c = load_f32<8>(angle);
      s = load_f32<8>(angle + half);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!turns) {
        A0[i] = pack2(w0.v[2 * i], w0.v[2 * i + 1]);
        A1[i] = pack2(w1.v[2 * i], w1.v[2 * i + 1]);
        B0[i] = B1[i] = pack2(0.f, 0.f);
      } else if (kInterleaved) {  // pair i of each chunk, angles i and 4 + i
        A0[i] = pack2(w0.v[2 * i] * c.v[i], w0.v[2 * i + 1] * c.v[i]);
        B0[i] = pack2(-w0.v[2 * i + 1] * s.v[i], w0.v[2 * i] * s.v[i]);
        A1[i] = pack2(w1.v[2 * i] * c.v[4 + i], w1.v[2 * i + 1] * c.v[4 + i]);
        B1[i] = pack2(-w1.v[2 * i + 1] * s.v[4 + i], w1.v[2 * i] * s.v[4 + i]);
      } else {
        A0[i] = pack2(w0.v[2 * i] * c.v[2 * i], w0.v[2 * i + 1] * c.v[2 * i + 1]);
        B0[i] = pack2(-w1.v[2 * i] * s.v[2 * i], -w1.v[2 * i + 1] * s.v[2 * i + 1]);
        A1[i] = pack2(w1.v[2 * i] * c.v[2 * i], w1.v[2 * i + 1] * c.v[2 * i + 1]);
        B1[i] = pack2(w0.v[2 * i] * s.v[2 * i], w0.v[2 * i + 1] * s.v[2 * i + 1]);
      }
    }
  }
  __nv_bfloat16* dst = is_q ? a.qo + (size_t)t * a.qo_ts + (size_t)h0 * a.qo_hs
                            : a.ko + (size_t)t * a.ko_ts + (size_t)h0 * a.ko_hs;
  const size_t dst_hs = is_q ? a.qo_hs : a.ko_hs;
  const float over_d = 1.f / (float)a.D;
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {  // the same count in every lane of the warp
    f32x2 x0[4], x1[4], ss2 = pack2(0.f, 0.f);
    const uint32_t r0[4] = {raw0[k].x, raw0[k].y, raw0[k].z, raw0[k].w};
    const uint32_t r1[4] = {raw1[k].x, raw1[k].y, raw1[k].z, raw1[k].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x0[i] = pack2(bf_lo(r0[i]), bf_hi(r0[i]));
      x1[i] = pack2(bf_lo(r1[i]), bf_hi(r1[i]));
      ss2 = fma2(x0[i], x0[i], ss2);
      ss2 = fma2(x1[i], x1[i], ss2);
    }
    float ss = unpack2(ss2).x + unpack2(ss2).y;
    for (int o = a.lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (k >= heads || !on0) continue;
    const float inv1 = rsqrtf(ss * over_d + a.eps);
    const f32x2 inv = pack2(inv1, inv1);
    uint32_t o0[4], o1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 y0 = mul2(x0[i], A0[i]), y1 = mul2(x1[i], A1[i]);
      if (turns) {
        const float2 u = unpack2(x0[i]), v = unpack2(x1[i]);
        y0 = fma2(kInterleaved ? pack2(u.y, u.x) : x1[i], B0[i], y0);
        y1 = fma2(kInterleaved ? pack2(v.y, v.x) : x0[i], B1[i], y1);
      }
      const float2 u = unpack2(mul2(y0, inv)), v = unpack2(mul2(y1, inv));
      o0[i] = good ? pack_bf16(u.x, u.y) : 0u;
      o1[i] = good ? pack_bf16(v.x, v.y) : 0u;
    }
    *reinterpret_cast<uint4*>(dst + k * dst_hs + at0) = make_uint4(o0[0], o0[1], o0[2], o0[3]);
    if (on1) *reinterpret_cast<uint4*>(dst + k * dst_hs + at1) = make_uint4(o1[0], o1[1], o1[2], o1[3]);
  }
}

// Every other layout, a value at a time: rows off the 16-byte grid, odd sizes.
// A row has 32 lanes at most, a lane kSlots pairs that turn with each other.
constexpr int QK_SLOTS = 4;
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(const QkRopeArgs a) {
  const int per_block = QK_THREADS / a.lanes;
  const int sub = threadIdx.x % a.lanes;
  const int H = a.Hq + a.Hkv;
  const long long group = (long long)blockIdx.x * per_block + threadIdx.x / a.lanes;
  const int t = (int)(group / H), h = (int)(group - (long long)t * H);
  const bool live = t < a.T, is_q = h < a.Hq;  // idle lanes stay for the shuffles
  const int hh = is_q ? h : h - a.Hq, half = a.rot / 2;
  const int pos = live ? a.pos[t] : 0;
  const bool good = pos >= 0 && pos < a.max_pos;
  if (live && !good && sub == 0) raise_status(a.status, WD_STATUS_BAD_POSITION);
  const __nv_bfloat16* src = is_q ? a.q + (size_t)t * a.q_ts + (size_t)hh * a.q_hs
                                  : a.k + (size_t)t * a.k_ts + (size_t)hh * a.k_hs;
  float x[QK_SLOTS], y[QK_SLOTS], ss = 0.f;
#pragma unroll
  for (int i = 0; i < QK_SLOTS; ++i) {
    const int c = sub + i * a.lanes;  // pair
    const bool split = c < half && !a.interleaved;
    x[i] = y[i] = 0.f;
    if (live && c < a.D / 2) {
      x[i] = __bfloat162float(src[split ? c : 2 * c]);
      y[i] = __bfloat162float(src[split ? half + c : 2 * c + 1]);
    }
    ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
  }
  for (int o = a.lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (!live) return;
  const float inv = rsqrtf(ss / (float)a.D + a.eps);
  const void* w = is_q ? a.qw : a.kw;
  __nv_bfloat16* dst = is_q ? a.qo + (size_t)t * a.qo_ts + (size_t)hh * a.qo_hs
                            : a.ko + (size_t)t * a.ko_ts + (size_t)hh * a.ko_hs;
#pragma unroll
  for (int i = 0; i < QK_SLOTS; ++i) {
    const int c = sub + i * a.lanes;
    if (c >= a.D / 2) continue;
    const bool split = c < half && !a.interleaved;
    const int at0 = split ? c : 2 * c, at1 = split ? half + c : 2 * c + 1;
    float u = x[i] * inv * load_weight<1>(w, a.weight_fp32, at0).v[0];
    float v = y[i] * inv * load_weight<1>(w, a.weight_fp32, at1).v[0];
    if (c < half && good) {
      const float cs = __ldg(a.cos_sin + (size_t)pos * a.rot + c);
      const float sn = __ldg(a.cos_sin + (size_t)pos * a.rot + half + c);
      const float uu = u * cs - v * sn;
      v = v * cs + u * sn;
      u = uu;
    }
    dst[at0] = __float2bfloat16_rn(good ? u : 0.f);
    dst[at1] = __float2bfloat16_rn(good ? v : 0.f);
  }
}

}  // namespace wdb

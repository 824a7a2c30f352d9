// RMS norm of every query and key head with the position rotation in the same
// pass, sm_100a.  No counterpart in the reference.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;   (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin)
//
// Bound by memory: each value is read and written once.  A row (one head of
// one token) belongs to a group of lanes, each holding two chunks of kV
// values that rotate with each other, so the pairs of both conventions meet
// inside a lane and the only exchange is the sum of squares.
#pragma once

#include "wd_common.cuh"

namespace wdb {

constexpr int QK_THREADS = 256;
constexpr int QK_MAX_D = 256;
constexpr int QK_MANY = 4;  // heads of a lane group in a call with many rows

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
  int heads;  // heads that one lane group takes of its token (kHeads)
  float eps;
};

template <int kV>
struct Chunk {
  float v[kV];
};

// kV bf16 values as they are.
template <int kV>
struct Raw {
  __nv_bfloat16 v[kV];
};
template <>
struct Raw<8> {
  uint4 v;
};
template <int kV>
__device__ __forceinline__ Raw<kV> load_raw(const __nv_bfloat16* p) {
  return *reinterpret_cast<const Raw<kV>*>(p);
}
__device__ __forceinline__ Chunk<8> widen_raw(const Raw<8>& r) {
  Chunk<8> c;
  unpack_bf16x8(r.v, c.v);
  return c;
}
__device__ __forceinline__ Chunk<1> widen_raw(const Raw<1>& r) {
  Chunk<1> c;
  c.v[0] = __bfloat162float(r.v[0]);
  return c;
}

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
__device__ __forceinline__ void store_bf16(__nv_bfloat16* p, const Chunk<kV>& c) {
  if constexpr (kV == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(c.v[0], c.v[1]), pack_bf16(c.v[2], c.v[3]), pack_bf16(c.v[4], c.v[5]),
                   pack_bf16(c.v[6], c.v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i) p[i] = __float2bfloat16_rn(c.v[i]);
  }
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

// kV = 8 (16-byte accesses) where D - rot, the rotated halves and every
// address are multiples of 8 values; kV = 1 for everything else.  kSlots: chunk
// pairs of a lane; kV = 8 has at most 16 pairs in a row, one per lane.  kHeads:
// heads that a lane group takes, loaded together.
template <int kV, int kSlots, int kHeads>
__global__ void __launch_bounds__(QK_THREADS) qk_norm_rope_kernel(const QkRopeArgs a) {
  const int per_block = QK_THREADS / a.lanes;
  const int sub = threadIdx.x % a.lanes;
  const int H = a.Hq + a.Hkv;
  const int parts = (H + kHeads - 1) / kHeads;
  const long long group = (long long)blockIdx.x * per_block + threadIdx.x / a.lanes;
  const int t = (int)(group / parts);
  const int h0 = (int)(group % parts) * kHeads;
  const bool live = t < a.T;  // idle lanes stay for the shuffles
  const int half = a.rot / 2;
  const int pairs = (a.D + 2 * kV - 1) / (2 * kV);

  int pos = 0;  // its load flies while the rows' do
  if (live) pos = a.pos[t];
  // where this lane's chunks lie
  int at0[kSlots], at1[kSlots];
  bool on0[kSlots], on1[kSlots], turns[kSlots];
  Chunk<kV> cs[kSlots], sn[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    const int c = sub + i * a.lanes;
    const int rotated = half / kV;  // chunk pairs that turn
    turns[i] = c < rotated;
    on0[i] = live && c < pairs;
    if (turns[i] && !a.interleaved) {
      at0[i] = c * kV;
      at1[i] = half + c * kV;
    } else if (kV == 1 || !turns[i]) {
      at0[i] = 2 * c * kV;
      at1[i] = at0[i] + kV;
    } else {
      at0[i] = 2 * c * kV;  // interleaved: 2 kV consecutive values, kV pairs
      at1[i] = at0[i] + kV;
    }
    on1[i] = on0[i] && at1[i] < a.D;
  }

  Raw<kV> raw0[kHeads][kSlots], raw1[kHeads][kSlots];
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {
    const int h = h0 + k;
    const __nv_bfloat16* src = h < a.Hq ? a.q + (size_t)t * a.q_ts + (size_t)h * a.q_hs
                                        : a.k + (size_t)t * a.k_ts + (size_t)(h - a.Hq) * a.k_hs;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (h < H && on0[i]) raw0[k][i] = load_raw<kV>(src + at0[i]);
      if (h < H && on1[i]) raw1[k][i] = load_raw<kV>(src + at1[i]);
    }
  }
  const bool good = pos >= 0 && pos < a.max_pos;
  if (live && !good && sub == 0) raise_status(a.status, WD_STATUS_BAD_POSITION);
#pragma unroll
  for (int i = 0; i < kSlots; ++i) {
    if (on0[i] && turns[i] && good) {
      const float* angle = a.cos_sin + (size_t)pos * a.rot + (sub + i * a.lanes) * kV;
      cs[i] = load_f32<kV>(angle);
      sn[i] = load_f32<kV>(angle + half);
    }
  }
#pragma unroll
  for (int k = 0; k < kHeads; ++k) {  // the same count in every lane of the warp
    const int h = h0 + k;
    const bool row = live && h < H;
    const bool is_q = h < a.Hq;
    const int hh = is_q ? h : h - a.Hq;
    Chunk<kV> x0[kSlots], x1[kSlots];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (row && on0[i]) x0[i] = widen_raw(raw0[k][i]);
      if (row && on1[i]) x1[i] = widen_raw(raw1[k][i]);
    }
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (row && on0[i]) {
#pragma unroll
        for (int j = 0; j < kV; ++j) ss = fmaf(x0[i].v[j], x0[i].v[j], ss);
      }
      if (row && on1[i]) {
#pragma unroll
        for (int j = 0; j < kV; ++j) ss = fmaf(x1[i].v[j], x1[i].v[j], ss);
      }
    }
    for (int o = a.lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss / (float)a.D + a.eps);
    if (!row) continue;
    const void* w = is_q ? a.qw : a.kw;
    __nv_bfloat16* dst = is_q ? a.qo + (size_t)t * a.qo_ts + (size_t)hh * a.qo_hs
                              : a.ko + (size_t)t * a.ko_ts + (size_t)hh * a.ko_hs;
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (!on0[i]) continue;
      const Chunk<kV> w0 = load_weight<kV>(w, a.weight_fp32, at0[i]);
#pragma unroll
      for (int j = 0; j < kV; ++j) x0[i].v[j] = good ? x0[i].v[j] * inv * w0.v[j] : 0.f;
      if (on1[i]) {
        const Chunk<kV> w1 = load_weight<kV>(w, a.weight_fp32, at1[i]);
#pragma unroll
        for (int j = 0; j < kV; ++j) x1[i].v[j] = good ? x1[i].v[j] * inv * w1.v[j] : 0.f;
      }
      if (turns[i] && good) {
        if (kV > 1 && a.interleaved) {
#pragma unroll
          for (int j = 0; j < kV / 2; ++j) {  // pairs inside each chunk
            float y = x0[i].v[2 * j], z = x0[i].v[2 * j + 1];
            x0[i].v[2 * j] = y * cs[i].v[j] - z * sn[i].v[j];
            x0[i].v[2 * j + 1] = z * cs[i].v[j] + y * sn[i].v[j];
            y = x1[i].v[2 * j], z = x1[i].v[2 * j + 1];
            x1[i].v[2 * j] = y * cs[i].v[kV / 2 + j] - z * sn[i].v[kV / 2 + j];
            x1[i].v[2 * j + 1] = z * cs[i].v[kV / 2 + j] + y * sn[i].v[kV / 2 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const float y = x0[i].v[j], z = x1[i].v[j];
            x0[i].v[j] = y * cs[i].v[j] - z * sn[i].v[j];
            x1[i].v[j] = z * cs[i].v[j] + y * sn[i].v[j];
          }
        }
      }
      store_bf16<kV>(dst + at0[i], x0[i]);
      if (on1[i]) store_bf16<kV>(dst + at1[i], x1[i]);
    }
  }
}

}  // namespace wdb

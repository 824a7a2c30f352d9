// FP8 paged key/value cache, sm_100a: quantise new tokens as they are written,
// read a range of tokens back.  No counterpart in the reference.
//
// A page of one head has one scale, 2^e.  With a power of two the codes of an
// E4M3 page lose nothing against any other scale (the format is a float one),
// a page whose scale rises is rounded again without error except where codes
// fall below E4M3's normal range, and attention can fold the scale into its
// exponents.  e is the least integer with amax <= 448 * 2^e, found exactly
// from the bits of amax: amax = m * 2^x with m in [1, 2), and 448 = 1.75 * 2^8,
// so e = x - 8 for m <= 1.75, else x - 7.
#pragma once

#include <cuda_fp8.h>

#include "wd_common.cuh"
#include "wd_qk_rope.cuh"

namespace wdb {

constexpr int KV_MAX_D = 256;
constexpr int KV_WRITE_THREADS = 256;
constexpr int KV_READ_THREADS = 256;
constexpr int KV_READ_EACH = 4;

struct KvWriteArgs {
  const __nv_bfloat16* x[2];       // keys, values
  long long bs[2], ts[2], hs[2];   // batch, token and head strides
  uint8_t* cache[2];
  uint8_t* scale[2];
  const int32_t *table, *start, *lens;
  uint32_t* status;
  int table_stride, S, H, D, page_shift, pages;
  int rows;             // rows that the block's threads hold at once
  uint32_t unit_magic;  // thread / units of a row = thread * unit_magic >> 21
};

struct KvReadArgs {
  const uint8_t* cache[2];
  const uint8_t* scale[2];
  const int32_t *table, *start, *lens;
  __nv_bfloat16* out[2];
  uint32_t* status;
  int table_stride, R, H, D, page_shift, pages;
  int span_shift;       // log2 of the tokens of a block, at most a page
  int units, rows;      // units of a pass: `rows` whole rows, or part of one
  uint32_t unit_magic;  // thread / units = thread * unit_magic >> 21
  uint32_t vec_magic;   // unit / (D / 16) = unit * vec_magic >> 21, for units below 1024 D / 16
};

// Scale byte of a page whose largest finite magnitude has the fp32 bits `u`.
__device__ __forceinline__ int scale_byte(uint32_t u) {
  if (u == 0u) return 1;
  if (u < 0x00800000u) return 1;  // below 2^-126
  const int x = (int)(u >> 23) - 127;
  const int e = (u & 0x007fffffu) <= 0x00600000u ? x - 8 : x - 7;
  return min(max(e + 127, 1), 254);
}
// 2^n as fp32 for -149 <= n <= 127.
__device__ __forceinline__ float exp2_int(int n) {
  return n >= -126 ? __uint_as_float((uint32_t)(n + 127) << 23) : __uint_as_float(1u << (n + 149));
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The tokens of one (sequence, touched page, head) of keys or of values, kV
// values at a time.  kKeep > 0: a thread has at most kKeep units and keeps them
// between the maximum and the rounding.  Grid: sequences, touched pages,
// 2 x heads.  Bound by HBM and, in small calls, by four dependent look-ups:
// 12 k tokens of 4 heads of 128 values (38 MB) about 11 us, 3.4 TB/s; with
// divisions by sizes and a scalar maximum it took 16.8.
template <int kV, int kKeep>
__global__ void __launch_bounds__(KV_WRITE_THREADS) kv_write_fp8_kernel(const KvWriteArgs a) {
  __shared__ uint32_t s_amax[KV_WRITE_THREADS / 32];
  const int b = blockIdx.x, which = blockIdx.z & 1, h = blockIdx.z >> 1;
  const int start = a.start[b];
  int len = a.lens ? a.lens[b] : a.S;
  len = min(max(len, 0), a.S);
  if (start < 0) {
    if (threadIdx.x == 0 && len > 0) raise_status(a.status, WD_STATUS_BAD_POSITION);
    return;
  }
  const long long end = (long long)start + len;
  const int col = (start >> a.page_shift) + blockIdx.y;
  const long long p0 = (long long)col << a.page_shift;  // first position of the page
  if (len == 0 || p0 >= end) return;
  // its load flies while the tokens' do
  const int pid = col < a.table_stride ? a.table[(size_t)b * a.table_stride + col] : -1;
  const int first = (int)max(0ll, (long long)start - p0);                   // rows [0, first): earlier tokens
  const int last = (int)min(1ll << a.page_shift, end - p0);                 // rows [first, last): new ones
  // a thread: one unit of kV values of every a.rows-th row
  const int vecs = a.D / kV, row0 = (int)((threadIdx.x * a.unit_magic) >> 21), d0 = (threadIdx.x - row0 * vecs) * kV;
  const int rows = row0 < a.rows ? last - first : 0;  // threads past whole rows have none
  const long long ts = which ? a.ts[1] : a.ts[0];
  const __nv_bfloat16* x = (which ? a.x[1] : a.x[0]) + (long long)b * (which ? a.bs[1] : a.bs[0]) +
                           (long long)h * (which ? a.hs[1] : a.hs[0]) + (p0 + first - start) * ts;
  x += d0;
  __nv_bfloat162 most2 = __floats2bfloat162_rn(0.f, 0.f);  // the largest magnitudes; NaN is passed over
  auto widen = [&](uint32_t two) { most2 = __hmax2(most2, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&two))); };
  uint4 kept[kKeep > 0 ? kKeep : 1];
  if constexpr (kKeep > 0) {
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      const int r = row0 + k * a.rows;
      kept[k] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) kept[k] = *reinterpret_cast<const uint4*>(x + (long long)r * ts);
    }
#pragma unroll
    for (int k = 0; k < kKeep; ++k) widen(kept[k].x), widen(kept[k].y), widen(kept[k].z), widen(kept[k].w);
  } else {
    for (int r = row0; r < rows; r += a.rows) {
      if constexpr (kV == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(x + (long long)r * ts);
        widen(v.x), widen(v.y), widen(v.z), widen(v.w);
      } else {
        widen(*reinterpret_cast<const uint16_t*>(x + (long long)r * ts));
      }
    }
  }
  const uint32_t two = *reinterpret_cast<const uint32_t*>(&most2);
  uint32_t most = max(two & 0xffffu, two >> 16) << 16;  // as fp32 bits
  if (most >= 0x7f800000u) {  // an infinity: once more without any
    most = 0u;
    for (int r = row0; r < rows; r += a.rows)
      for (int j = 0; j < kV; ++j) {
        const uint32_t u = (uint32_t)(reinterpret_cast<const uint16_t*>(x + (long long)r * ts)[j] & 0x7fffu) << 16;
        if (u < 0x7f800000u) most = max(most, u);
      }
  }
  if (pid < 0 || pid >= a.pages) {  // the whole block
    if (threadIdx.x == 0) raise_status(a.status, WD_STATUS_BAD_PAGE);
    return;
  }
  uint8_t* page = (which ? a.cache[1] : a.cache[0]) + (((size_t)pid * a.H + h) << a.page_shift) * a.D;
  uint8_t* scale = (which ? a.scale[1] : a.scale[0]) + (size_t)pid * a.H + h;
  const int was = first > 0 ? *scale : 0;

  most = __reduce_max_sync(0xffffffffu, most);
  if (blockDim.x > 32) {
    if ((threadIdx.x & 31) == 0) s_amax[threadIdx.x >> 5] = most;
    __syncthreads();
    most = 0u;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) most = max(most, s_amax[i]);
  }
  const int now = max(scale_byte(most), was);
  __syncwarp();  // every lane has read the old scale (the block barrier covers larger blocks)
  if (threadIdx.x == 0 && now != was) *scale = (uint8_t)now;

  const float inv = exp2_int(127 - now);
  uint8_t* page0 = page;
  page += first * a.D + d0;
  auto store = [&](int r, const Chunk<kV>& c) {
    uint8_t* out = page + r * a.D;
    if constexpr (kV == 8) {
      *reinterpret_cast<uint2*>(out) =
          make_uint2(e4m3x4(c.v[0] * inv, c.v[1] * inv, c.v[2] * inv, c.v[3] * inv),
                     e4m3x4(c.v[4] * inv, c.v[5] * inv, c.v[6] * inv, c.v[7] * inv));
    } else {
      *out = (uint8_t)__nv_cvt_float_to_fp8(c.v[0] * inv, __NV_SATFINITE, __NV_E4M3);
    }
  };
  if constexpr (kKeep > 0) {
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
      const int r = row0 + k * a.rows;
      Chunk<kV> c;
      unpack_bf16x8(kept[k], c.v);
      if (r < rows) store(r, c);
    }
  } else {
    for (int r = row0; r < rows; r += a.rows) store(r, load_bf16<kV>(x + (long long)r * ts));
  }
  if (first > 0 && now > was) {  // the earlier codes at the larger scale
    const float down = exp2_int(max(was - now, -149));
    for (int i = threadIdx.x; i < first * a.D / 4; i += blockDim.x) {
      uint32_t* at = reinterpret_cast<uint32_t*>(page0) + i;
      const float2 lo = e4m3x2_to_f32(*at & 0xffffu), hi = e4m3x2_to_f32(*at >> 16);
      *at = e4m3x4(lo.x * down, lo.y * down, hi.x * down, hi.y * down);
    }
  }
}

// A block: the tokens of one page of a sequence, or an aligned part of them,
// keys (blockIdx.z 0) or values (1): the page is looked up once; a thread: one unit of 16 values (one
// head, one scale) of every a.rows-th token, KV_READ_EACH loads in flight.
// Grid: sequences, touched spans, 2.  Bound by HBM: 12 k tokens of 4 heads of
// 128 values (46 MB) about 11 us, 4.2 TB/s; with a look-up and divisions for
// every unit it took 17.4.
__global__ void __launch_bounds__(KV_READ_THREADS) kv_read_fp8_kernel(const KvReadArgs a) {
  const int b = blockIdx.x, which = blockIdx.z;
  const int start = a.start[b], len = min(a.lens ? a.lens[b] : a.R, a.R);
  const int vecs = a.D / 16, per_row = a.H * vecs, page = 1 << a.page_shift;
  // rows [r0, r1) of the output lie on this span (of a negative start as if it
  // were 0: they are zeros)
  const int s0 = max(start, 0);
  const long long p0 = ((long long)(s0 >> a.span_shift) + blockIdx.y) << a.span_shift;
  const int r0 = (int)max(0ll, p0 - s0);
  const int r1 = (int)min((long long)a.R, p0 + (1ll << a.span_shift) - s0);
  if (r0 >= r1) return;
  const int col = (int)(p0 >> a.page_shift);
  int pid = -1;
  if (r0 < len) {
    if (start >= 0 && col < a.table_stride) pid = __ldg(a.table + (size_t)b * a.table_stride + col);
    if (pid < 0 || pid >= a.pages) {
      pid = -1;
      if (threadIdx.x == 0) raise_status(a.status, start < 0 ? WD_STATUS_BAD_POSITION : WD_STATUS_BAD_PAGE);
    }
  }
  const int live = pid >= 0 ? min(r1, len) : r0;  // rows [live, r1) are zeros
  const int row = (int)((threadIdx.x * a.unit_magic) >> 21);
  if (row >= a.rows) return;  // threads past whole rows
  uint4* out = reinterpret_cast<uint4*>(which ? a.out[1] : a.out[0]) + (size_t)b * a.R * per_row * 2;
  for (int e = threadIdx.x - row * a.units; e < per_row; e += a.units) {
    const int h = (int)((e * a.vec_magic) >> 21);
    const size_t ph = (size_t)max(pid, 0) * a.H + h;
    const float f = pid >= 0 ? ue8m0_to_f32(__ldg((which ? a.scale[1] : a.scale[0]) + ph)) : 0.f;
    const uint4* src = reinterpret_cast<const uint4*>(which ? a.cache[1] : a.cache[0]) +
                       (ph << a.page_shift) * vecs + (e - h * vecs);
    for (int r = r0 + row; r < r1; r += a.rows * KV_READ_EACH) {
      uint4 codes[KV_READ_EACH];
#pragma unroll
      for (int k = 0; k < KV_READ_EACH; ++k) {
        const int rr = r + k * a.rows;
        codes[k] = make_uint4(0u, 0u, 0u, 0u);
        if (rr < live) codes[k] = __ldg(src + (size_t)(((uint32_t)s0 + rr) & (page - 1)) * vecs);
      }
#pragma unroll
      for (int k = 0; k < KV_READ_EACH; ++k) {
        const int rr = r + k * a.rows;
        if (rr >= r1) break;
        const float g = rr < live ? f : 0.f;
        const uint32_t cw[4] = {codes[k].x, codes[k].y, codes[k].z, codes[k].w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 lo = e4m3x2_to_f32(cw[j] & 0xffffu), hi = e4m3x2_to_f32(cw[j] >> 16);
          o[2 * j] = pack_bf16(lo.x * g, lo.y * g);
          o[2 * j + 1] = pack_bf16(hi.x * g, hi.y * g);
        }
        uint4* to = out + ((size_t)rr * per_row + e) * 2;
        to[0] = make_uint4(o[0], o[1], o[2], o[3]);
        to[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
}

}  // namespace wdb

// C ABI of the operators around the MoE FFN (include/warp_decode_layer.h):
// argument checks, launch geometry and dispatch.  A translation unit and a
// library of its own, so the FFN library's exports stay as they are.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <string>

#include "warp_decode_layer.h"

#include "wd_attn_fp8.cuh"
#include "wd_attn_fp8_tc.cuh"
#include "wd_kv_fp8.cuh"
#include "wd_qk_rope.cuh"
#include "wd_router_scored.cuh"

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* msg) {
  g_last_error = msg;
  return code;
}

std::atomic<unsigned long long> g_launches{0};

// Result of the launch just made.
int launched(const char* what) {
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) {
    g_last_error = std::string(what) + ": " + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return WD_OK;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr long long kMaxBlocks = 0x7fffffffll;

// i / n = i * magic21(n) >> 21 for 0 <= i < 1024 n, i < 2^21 / n
uint32_t magic21(int n) { return (uint32_t)(((1 << 21) + n - 1) / n); }

int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

// Checks shared by the three cache entry points.
int check_cache(int B, int Hkv, int D, int page, int pages, int table_stride) {
  if (B < 0) return fail(WD_ERR_SHAPE, "B must be >= 0");
  if (Hkv < 1) return fail(WD_ERR_SHAPE, "Hkv must be >= 1");
  if (page != 16 && page != 32 && page != 64 && page != 128)
    return fail(WD_ERR_UNSUPPORTED, "page must be 16, 32, 64 or 128 tokens");
  if (D < 16 || D % 16 != 0) return fail(WD_ERR_SHAPE, "D must be a positive multiple of 16");
  if (D > wdb::KV_MAX_D) return fail(WD_ERR_UNSUPPORTED, "D must be <= 256");
  if (pages < 0 || table_stride < 0) return fail(WD_ERR_SHAPE, "pages and table_stride must be >= 0");
  return WD_OK;
}

int check_cache_pointers(const void* kc, const void* ks, const void* vc, const void* vs,
                         const void* table, int table_stride, const void* lens) {
  if (!kc || !ks || !vc || !vs || (!table && table_stride > 0) || !lens)
    return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(kc, 16) || !aligned(vc, 16))
    return fail(WD_ERR_ALIGNMENT, "the caches must be 16-byte aligned");
  if (!aligned(table, 4) || !aligned(lens, 4))
    return fail(WD_ERR_ALIGNMENT, "int32 tensors must be 4-byte aligned");
  return WD_OK;
}

// cuTensorMapEncodeTiled from the driver, resolved once through the runtime.
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<EncodeTiledFn>(nullptr);
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

constexpr int kMaxDevices = 64;

// SM count of the current device, looked up once per device.
int sm_count(int* out) {
  static std::atomic<int> known[kMaxDevices];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) return fail(WD_ERR_CUDA, "device index out of range");
  int n = err == cudaSuccess ? known[dev].load(std::memory_order_relaxed) : 0;
  if (err == cudaSuccess && n == 0) {
    err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    if (err == cudaSuccess) known[dev].store(n, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    g_last_error = std::string("device: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  *out = n;
  return WD_OK;
}

// Columns (query rows of one key head) per tensor-core unit.
int attn_columns(long long rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

bool attn_on_tensor_cores(int D) { return D == 64 || D == 128; }

int attn_ctas(int sms) { return std::min(sms, wdb::AT_MAX_CTAS); }  // one per SM

size_t attn_workspace(int sms, int D, int columns) {
  const size_t slot = (size_t)(columns * D + 5 * columns) * 4;  // AttnTcShape::kSlotFloats
  return wdb::AT_COUNTERS + (columns == 64 ? 2 : 4) * (size_t)attn_ctas(sms) * slot;  // kSlots of two pieces
}

template <int kD, int kN>
int launch_attn_tc(const wdb::AttnTcArgs& t, const CUtensorMap& k, const CUtensorMap& v, int ctas,
                   cudaStream_t s) {
  using Shape = wdb::AttnTcShape<kD, kN>;
  static std::atomic<unsigned long long> ready{0};  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && !((ready.load(std::memory_order_relaxed) >> dev) & 1ull)) {
    err = cudaFuncSetAttribute(wdb::attn_fp8_tc_kernel<kD, kN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               Shape::kSmem);
    if (err == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    g_last_error = std::string("attn_decode_fp8 set-up: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  // Cooperative: CTAs that share a unit wait for one another at its end.
  cudaLaunchAttribute coop;
  coop.id = cudaLaunchAttributeCooperative;
  coop.val.cooperative = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(wdb::AT_THREADS);
  cfg.dynamicSmemBytes = Shape::kSmem;
  cfg.stream = s;
  cfg.attrs = &coop;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, wdb::attn_fp8_tc_kernel<kD, kN>, t, k, v);
  if (err != cudaSuccess) {
    cudaGetLastError();
    g_last_error = std::string("attn_decode_fp8: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  return launched("attn_decode_fp8");
}

// Experts per lane: the least room that holds ceil(E / 32).
template <bool kFp32, bool kVector, bool kWhole>
void launch_router(const wdb::RouterScoredArgs& a, cudaStream_t s) {
  auto kernel = wdb::moe_router_scored_kernel<32, kFp32, kVector, kWhole>;
  if (a.per <= 1 && !kVector)
    kernel = wdb::moe_router_scored_kernel<1, kFp32, false, kWhole>;
  else if (a.per <= 4 && (!kVector || kFp32))
    kernel = wdb::moe_router_scored_kernel<4, kFp32, kVector && kFp32, kWhole>;
  else if (a.per <= 8)
    kernel = wdb::moe_router_scored_kernel<8, kFp32, kVector, kWhole>;
  else if (a.per <= 16)
    kernel = wdb::moe_router_scored_kernel<16, kFp32, kVector, kWhole>;
  kernel<<<(a.T + wdb::RS_WARPS - 1) / wdb::RS_WARPS, wdb::RS_WARPS * 32, 0, s>>>(a);
}

}  // namespace

extern "C" {

const char* wd_layer_last_error_message(void) { return g_last_error.c_str(); }

unsigned long long wd_layer_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

int wd_layer_status_read(uint32_t* value, int clear) {
  if (!value) return fail(WD_ERR_NULL_POINTER, "value is NULL");
  cudaError_t err = cudaMemcpyFromSymbol(value, wdb::g_wd_status, sizeof(uint32_t));
  if (err == cudaSuccess && clear && *value != 0u) {
    const uint32_t zero = 0u;
    err = cudaMemcpyToSymbol(wdb::g_wd_status, &zero, sizeof(uint32_t));
  }
  if (err != cudaSuccess) {
    g_last_error = std::string("status: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  return WD_OK;
}

int wd_moe_router_scored_topk(const void* logits, int logits_fp32, const float* bias,
                              int32_t* topk_ids, float* topk_weights, int T, int E, int topk,
                              int scoring, int n_group, int topk_group, int group_top,
                              int renormalize, float weight_scale, void* stream) {
  if (T < 0) return fail(WD_ERR_SHAPE, "T must be >= 0");
  if (E < 1) return fail(WD_ERR_SHAPE, "E (number of experts) must be >= 1");
  if (E > wdb::RS_MAX_E) return fail(WD_ERR_UNSUPPORTED, "E must be <= 1024");
  if (topk < 1) return fail(WD_ERR_SHAPE, "topk must be >= 1");
  if (topk > wdb::RS_MAX_K) return fail(WD_ERR_UNSUPPORTED, "topk must be <= 32");
  if (scoring != 0 && scoring != 1) return fail(WD_ERR_SHAPE, "scoring must be 0 (softmax) or 1 (sigmoid)");
  if (n_group < 1 || E % n_group != 0) return fail(WD_ERR_SHAPE, "n_group must divide E");
  if (n_group > 32) return fail(WD_ERR_UNSUPPORTED, "n_group must be <= 32");
  if (topk_group < 1 || topk_group > n_group)
    return fail(WD_ERR_SHAPE, "topk_group must be between 1 and n_group");
  if (group_top != 1 && group_top != 2) return fail(WD_ERR_SHAPE, "group_top must be 1 or 2");
  if (topk > E / n_group * topk_group)
    return fail(WD_ERR_SHAPE, "topk exceeds the experts of topk_group groups");
  if (T == 0) return WD_OK;
  if (!logits || !topk_ids || !topk_weights) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(logits, logits_fp32 ? 4 : 2) || !aligned(bias, 4) || !aligned(topk_ids, 4) ||
      !aligned(topk_weights, 4))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer");
  wdb::RouterScoredArgs a{};
  a.logits = logits, a.bias = bias, a.ids = topk_ids, a.weights = topk_weights;
  a.T = T, a.E = E, a.K = topk, a.sigmoid = scoring, a.n_group = n_group, a.topk_group = topk_group;
  a.group_top = group_top, a.renormalize = renormalize ? 1 : 0, a.weight_scale = weight_scale;
  a.per = (E + 31) / 32;
  a.size = E / n_group;
  a.group_magic = magic21(a.size);
  a.group_lanes = a.size / a.per;
  // a lane's experts in whole 16-byte units (all of 4, 8, 16 or 32 of them)
  const int unit = logits_fp32 ? 4 : 8;
  const bool vector = E % 32 == 0 && (a.per & (a.per - 1)) == 0 && a.per >= unit && aligned(logits, 16);
  // groups of a power of two of whole lanes
  const bool whole = n_group == 1 || (a.size % a.per == 0 && (a.group_lanes & (a.group_lanes - 1)) == 0);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto launch = logits_fp32 ? (vector ? (whole ? launch_router<true, true, true> : launch_router<true, true, false>)
                                      : (whole ? launch_router<true, false, true> : launch_router<true, false, false>))
                            : (vector ? (whole ? launch_router<false, true, true> : launch_router<false, true, false>)
                                      : (whole ? launch_router<false, false, true> : launch_router<false, false, false>));
  launch(a, s);
  return launched("moe_router_scored_topk");
}

int wd_qk_norm_rope(const void* q, long long q_token_stride, long long q_head_stride, const void* k,
                    long long k_token_stride, long long k_head_stride, const void* q_weight,
                    const void* k_weight, int weight_fp32, const int32_t* positions,
                    const float* cos_sin, int max_pos, void* q_out, long long qo_token_stride,
                    long long qo_head_stride, void* k_out, long long ko_token_stride,
                    long long ko_head_stride, int T, int Hq, int Hkv, int D, int rot,
                    int interleaved, float eps, uint32_t* status, void* stream) {
  if (T < 0) return fail(WD_ERR_SHAPE, "T must be >= 0");
  if (Hq < 0 || Hkv < 0) return fail(WD_ERR_SHAPE, "Hq and Hkv must be >= 0");
  if (D < 2 || D % 2 != 0) return fail(WD_ERR_SHAPE, "D must be a positive multiple of 2");
  if (D > wdb::QK_MAX_D) return fail(WD_ERR_UNSUPPORTED, "D must be <= 256");
  if (rot < 0 || rot > D || rot % 2 != 0) return fail(WD_ERR_SHAPE, "rot must be even and between 0 and D");
  if (max_pos < 0) return fail(WD_ERR_SHAPE, "max_pos must be >= 0");
  if (T == 0 || Hq + Hkv == 0) return WD_OK;
  if ((Hq > 0 && (!q || !q_out || !q_weight)) || (Hkv > 0 && (!k || !k_out || !k_weight)) || !positions ||
      (rot > 0 && !cos_sin))
    return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  const uintptr_t wa = weight_fp32 ? 4 : 2;
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(q_out, 2) || !aligned(k_out, 2) ||
      !aligned(q_weight, wa) || !aligned(k_weight, wa) || !aligned(positions, 4) || !aligned(cos_sin, 4))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer");
  wdb::QkRopeArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.qo = static_cast<__nv_bfloat16*>(q_out);
  a.ko = static_cast<__nv_bfloat16*>(k_out);
  a.q_ts = q_token_stride, a.q_hs = q_head_stride, a.k_ts = k_token_stride, a.k_hs = k_head_stride;
  a.qo_ts = qo_token_stride, a.qo_hs = qo_head_stride, a.ko_ts = ko_token_stride, a.ko_hs = ko_head_stride;
  a.qw = q_weight, a.kw = k_weight;
  a.pos = positions, a.cos_sin = cos_sin, a.status = status;
  a.T = T, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.rot = rot, a.max_pos = max_pos;
  a.weight_fp32 = weight_fp32 ? 1 : 0, a.interleaved = interleaved ? 1 : 0, a.eps = eps;
  // 16-byte accesses where every row and chunk allows them
  const long long strides = q_token_stride | q_head_stride | k_token_stride | k_head_stride |
                            qo_token_stride | qo_head_stride | ko_token_stride | ko_head_stride;
  const bool wide = D % 8 == 0 && rot % 16 == 0 && strides % 8 == 0 && aligned(q, 16) && aligned(k, 16) &&
                    aligned(q_out, 16) && aligned(k_out, 16) && aligned(q_weight, 16) &&
                    aligned(k_weight, 16) && aligned(cos_sin, 16);
  const int pairs = wide ? (D + 15) / 16 : D / 2;
  a.lanes = 1;
  while (a.lanes < pairs && a.lanes < 32) a.lanes *= 2;
  // Heads a lane group: their loads fly together and share the angles and factors,
  // but the call has fewer groups.  One where that makes no more than three blocks
  // an SM, two where two make no more than two; otherwise four, unless the heads
  // leave a third of such groups empty.  Measured with one, two and four (us):
  //   32 + 4 heads of 128: 256 tokens 3.1, 3.4, 3.8; 512: 4.9, 3.8, 3.9; 1000: 6.9,
  //   6.4, 4.8; 8192: 51.1, 50.0, 34.5.  16 + 2 heads of 64: 1000 tokens 3.2, 3.3,
  //   3.9; 1999: 4.9, 4.0, 4.7; 4000: 7.2, 6.1, 6.4; 8192: 16.4, 12.4, 12.0.
  //   5 + 1 heads of 64: 4000 tokens 3.6, 3.8, 4.6; 8192: 5.7, 6.0, 6.6.
  const long long per_block = wdb::QK_THREADS / a.lanes;
  auto blocks_of = [&](int n) {
    const long long groups = (long long)T * (((long long)Hq + n - 1) / n + ((long long)Hkv + n - 1) / n);
    return (groups + per_block - 1) / per_block;
  };
  int each = 1;
  if (wide) {
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    if (blocks_of(1) > 3 * sms) each = blocks_of(2) <= 2 * sms ? 2 : 4 * blocks_of(4) * 2 <= 3 * blocks_of(1) ? 4 : 1;
  }
  const long long blocks = blocks_of(each);
  if (blocks > kMaxBlocks) return fail(WD_ERR_UNSUPPORTED, "T * heads is too large");
  auto kernel = wdb::qk_norm_rope_kernel;
  if (wide && interleaved)
    kernel = each == 4   ? wdb::qk_norm_rope_wide_kernel<4, true>
             : each == 2 ? wdb::qk_norm_rope_wide_kernel<2, true>
                         : wdb::qk_norm_rope_wide_kernel<1, true>;
  else if (wide)
    kernel = each == 4   ? wdb::qk_norm_rope_wide_kernel<4, false>
             : each == 2 ? wdb::qk_norm_rope_wide_kernel<2, false>
                         : wdb::qk_norm_rope_wide_kernel<1, false>;
  kernel<<<(unsigned)blocks, wdb::QK_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launched("qk_norm_rope");
}

int wd_kv_cache_write_fp8(const void* k, long long k_batch_stride, long long k_token_stride,
                          long long k_head_stride, const void* v, long long v_batch_stride,
                          long long v_token_stride, long long v_head_stride, uint8_t* k_cache,
                          uint8_t* k_scale, uint8_t* v_cache, uint8_t* v_scale,
                          const int32_t* table, int table_stride, const int32_t* start,
                          const int32_t* lens, int B, int S, int Hkv, int D, int page, int pages,
                          uint32_t* status, void* stream) {
  if (int rc = check_cache(B, Hkv, D, page, pages, table_stride)) return rc;
  if (S < 0) return fail(WD_ERR_SHAPE, "S must be >= 0");
  if (B == 0 || S == 0) return WD_OK;
  if (int rc = check_cache_pointers(k_cache, k_scale, v_cache, v_scale, table, table_stride, start)) return rc;
  if (!k || !v) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(k, 2) || !aligned(v, 2) || !aligned(lens, 4))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer");
  wdb::KvWriteArgs a{};
  a.x[0] = static_cast<const __nv_bfloat16*>(k), a.x[1] = static_cast<const __nv_bfloat16*>(v);
  a.bs[0] = k_batch_stride, a.ts[0] = k_token_stride, a.hs[0] = k_head_stride;
  a.bs[1] = v_batch_stride, a.ts[1] = v_token_stride, a.hs[1] = v_head_stride;
  a.cache[0] = k_cache, a.cache[1] = v_cache, a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.table = table, a.start = start, a.lens = lens, a.status = status;
  a.table_stride = table_stride, a.S = S, a.H = Hkv, a.D = D, a.pages = pages;
  a.page_shift = page_shift(page);
  const long long touched = ((long long)S + page - 2) / page + 1;
  if (touched > 65535 || Hkv > 1024)
    return fail(WD_ERR_UNSUPPORTED, "S must be at most 65534 pages of tokens, Hkv <= 1024");
  const long long strides = k_batch_stride | k_token_stride | k_head_stride | v_batch_stride |
                            v_token_stride | v_head_stride;
  const bool wide = strides % 8 == 0 && aligned(k, 16) && aligned(v, 16);
  // Four 16-byte units a thread, kept from the maximum to the rounding, where a
  // page's new tokens have no more (wide); otherwise they are read twice.
  const int per_row = D / (wide ? 8 : 1), most = std::min(S, page);  // units of a row, rows
  const int threads =
      std::min(std::max((most * per_row + 127) / 128 * 32, (per_row + 31) / 32 * 32), wdb::KV_WRITE_THREADS);
  a.rows = threads / per_row;  // of a pass; at least one, for D <= 256
  a.unit_magic = magic21(per_row);
  const dim3 grid((unsigned)B, (unsigned)touched, 2u * (unsigned)Hkv);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (wide && most <= 4 * a.rows)
    wdb::kv_write_fp8_kernel<8, 4><<<grid, threads, 0, s>>>(a);
  else if (wide)
    wdb::kv_write_fp8_kernel<8, 0><<<grid, threads, 0, s>>>(a);
  else
    wdb::kv_write_fp8_kernel<1, 0><<<grid, threads, 0, s>>>(a);
  return launched("kv_cache_write_fp8");
}

int wd_kv_cache_read_fp8(const uint8_t* k_cache, const uint8_t* k_scale, const uint8_t* v_cache,
                         const uint8_t* v_scale, const int32_t* table, int table_stride,
                         const int32_t* start, const int32_t* lens, void* k_out, void* v_out, int B,
                         int R, int Hkv, int D, int page, int pages, uint32_t* status, void* stream) {
  if (int rc = check_cache(B, Hkv, D, page, pages, table_stride)) return rc;
  if (R < 0) return fail(WD_ERR_SHAPE, "R must be >= 0");
  if (B == 0 || R == 0) return WD_OK;
  if (int rc = check_cache_pointers(k_cache, k_scale, v_cache, v_scale, table, table_stride, start)) return rc;
  if (!k_out || !v_out) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(lens, 4))
    return fail(WD_ERR_ALIGNMENT, "the outputs must be 16-byte aligned");
  wdb::KvReadArgs a{};
  a.cache[0] = k_cache, a.cache[1] = v_cache, a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.table = table, a.start = start, a.lens = lens, a.status = status;
  a.out[0] = static_cast<__nv_bfloat16*>(k_out), a.out[1] = static_cast<__nv_bfloat16*>(v_out);
  a.table_stride = table_stride, a.R = R, a.H = Hkv, a.D = D, a.pages = pages;
  a.page_shift = page_shift(page);
  const int per_row = Hkv * (D / 16);
  a.units = std::min(per_row, wdb::KV_READ_THREADS);
  a.rows = wdb::KV_READ_THREADS / a.units;
  a.span_shift = 0;  // tokens whose loads all fly together, within a page
  while (a.span_shift < a.page_shift && (2 << a.span_shift) <= a.rows * wdb::KV_READ_EACH) ++a.span_shift;
  auto spans = [&] { return ((long long)R + (1 << a.span_shift) - 2) / (1 << a.span_shift) + 1; };
  while (a.span_shift < a.page_shift && spans() > 65535) ++a.span_shift;  // of a long read: the grid's limit
  const long long touched = spans();
  if (touched > 65535 || Hkv > 1024)
    return fail(WD_ERR_UNSUPPORTED, "R must be at most 65534 pages of tokens, Hkv <= 1024");
  a.unit_magic = magic21(a.units);
  a.vec_magic = magic21(D / 16);
  wdb::kv_read_fp8_kernel<<<dim3((unsigned)B, (unsigned)touched, 2), wdb::KV_READ_THREADS, 0,
                            static_cast<cudaStream_t>(stream)>>>(a);
  return launched("kv_cache_read_fp8");
}

int wd_attn_decode_fp8_workspace(int B, int Sq, int Hq, int Hkv, int D, size_t* bytes) {
  if (!bytes) return fail(WD_ERR_NULL_POINTER, "bytes is NULL");
  if (B < 0 || Sq < 0 || Hq < 0 || Hkv < 1 || Hq % Hkv != 0 || D < 16 || D % 16 != 0)
    return fail(WD_ERR_SHAPE, "inconsistent sizes");
  *bytes = 0;
  if (B == 0 || Sq == 0 || Hq == 0 || !attn_on_tensor_cores(D)) return WD_OK;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  *bytes = attn_workspace(sms, D, attn_columns((long long)Sq * (Hq / Hkv)));
  return WD_OK;
}

int wd_attn_decode_fp8(const void* q, long long q_batch_stride, long long q_token_stride,
                       long long q_head_stride, const uint8_t* k_cache, const uint8_t* k_scale,
                       const uint8_t* v_cache, const uint8_t* v_scale, const int32_t* table,
                       int table_stride, const int32_t* seq_lens, void* out, float* lse,
                       float softmax_scale, int window, int B, int Sq, int Hq, int Hkv, int D,
                       int page, int pages, void* workspace, size_t workspace_bytes,
                       uint32_t* status, void* stream) {
  if (int rc = check_cache(B, Hkv, D, page, pages, table_stride)) return rc;
  if (Sq < 0) return fail(WD_ERR_SHAPE, "Sq must be >= 0");
  if (Hq < 1 || Hq % Hkv != 0) return fail(WD_ERR_SHAPE, "Hq must be a positive multiple of Hkv");
  if (window < 0) return fail(WD_ERR_SHAPE, "window must be >= 0");
  if (B == 0 || Sq == 0) return WD_OK;
  if (int rc = check_cache_pointers(k_cache, k_scale, v_cache, v_scale, table, table_stride, seq_lens)) return rc;
  if (!q || !out) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(q, 2) || !aligned(out, 16) || !aligned(lse, 4))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer (q 2, out 16, lse 4 bytes)");
  wdb::AttnArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_bs = q_batch_stride, a.q_ts = q_token_stride, a.q_hs = q_head_stride;
  a.kc = k_cache, a.ks = k_scale, a.vc = v_cache, a.vs = v_scale;
  a.table = table, a.seq_lens = seq_lens, a.out = static_cast<__nv_bfloat16*>(out), a.lse = lse;
  a.status = status;
  a.table_stride = table_stride, a.B = B, a.Sq = Sq, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.page = page;
  a.pages = pages, a.window = window;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long long rows = (long long)Sq * (Hq / Hkv), cache_rows = (long long)pages * Hkv * page;
  // the tensor maps take row numbers of 32 bits and a cache of at least a row
  if (attn_on_tensor_cores(D) && cache_rows > 0 && cache_rows <= 0x7fffffffll && rows <= 0x7fffffffll / 2) {
    const int columns = attn_columns(rows);
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    if (!workspace) return fail(WD_ERR_NULL_POINTER, "workspace is NULL");
    if (!aligned(workspace, 16)) return fail(WD_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    if (workspace_bytes < attn_workspace(sms, D, columns))
      return fail(WD_ERR_SHAPE, "workspace is smaller than wd_attn_decode_fp8_workspace says");
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) return fail(WD_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    CUtensorMap tm[2];
    const cuuint64_t dim[2] = {(cuuint64_t)D, (cuuint64_t)cache_rows};
    const cuuint64_t str[1] = {(cuuint64_t)D};
    const cuuint32_t box[2] = {(cuuint32_t)D, (cuuint32_t)page}, ones[2] = {1, 1};
    for (int i = 0; i < 2; ++i) {
      const CUresult cr =
          enc(&tm[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(i ? v_cache : k_cache), dim, str,
              box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
              D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
      if (cr != CUDA_SUCCESS) return fail(WD_ERR_CUDA, "tensor map (cache) encode failed");
    }
    wdb::AttnTcArgs t{};
    t.a = a;
    t.counters = static_cast<uint32_t*>(workspace);
    t.slots = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + wdb::AT_COUNTERS);
    t.chunks = (int)((rows + columns - 1) / columns);
    // Measured (B200, page 64, D 128, us) for least share / unit cost of 2/1, 3/2,
    // 6/4 and 12/8 tiles: 1 x 1000 keys, one key head 10.6, 10.6, 12.9, 11.6;
    // 8 ragged up to 4096 15.6, 15.1, 15.1, 19.0; 64 ragged up to 8192 60.4, 59.1,
    // 58.8, 60.7; 1 x 8192 12.7, 13.4, 14.8, 18.7.  A share holds more than a
    // unit's cost, so that every CTA has a tile.
    t.min_share = 3;
    t.unit_cost = 2;
    t.q_wide = aligned(q, 16) && (q_batch_stride | q_token_stride | q_head_stride) % 8 == 0;
    t.reach = (int)std::min((long long)table_stride * page, 0x7fffffffll - wdb::AT_TILE);
    // tiles are counted in 32 bits; lengths up to the tables' reach
    if ((long long)B * Hkv * t.chunks * (t.reach / wdb::AT_TILE + 1 + t.unit_cost) > 0x7fffffffll)
      return fail(WD_ERR_UNSUPPORTED, "B * Hkv * table_stride * page is too large");
    t.page_shift = page_shift(page);
    const int ctas = attn_ctas(sms);
    if (D == 128) {
      if (columns == 16) return launch_attn_tc<128, 16>(t, tm[0], tm[1], ctas, s);
      if (columns == 32) return launch_attn_tc<128, 32>(t, tm[0], tm[1], ctas, s);
      return launch_attn_tc<128, 64>(t, tm[0], tm[1], ctas, s);
    }
    if (columns == 16) return launch_attn_tc<64, 16>(t, tm[0], tm[1], ctas, s);
    if (columns == 32) return launch_attn_tc<64, 32>(t, tm[0], tm[1], ctas, s);
    return launch_attn_tc<64, 64>(t, tm[0], tm[1], ctas, s);
  }
  const long long chunks = (rows + wdb::ATTN_ROWS - 1) / wdb::ATTN_ROWS;
  const long long blocks = chunks * Hkv * B;
  if (blocks > kMaxBlocks) return fail(WD_ERR_UNSUPPORTED, "B * Sq * Hq is too large");
  wdb::attn_fp8_simt_kernel<<<(unsigned)blocks, wdb::ATTN_WARPS * 32, 0, s>>>(a);
  return launched("attn_decode_fp8");
}

}  // extern "C"

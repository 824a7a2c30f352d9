// Host side shared by the libraries of the operators around the MoE FFN: errors,
// checks of the FP8 cache's arguments, its tensor map, and the launch of attention
// on the CUDA cores.  Each library includes it once.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>

#include "warp_decode_layer.h"

#include "wd_attn_fp8.cuh"
#include "wd_attn_fp8_tc.cuh"
#include "wd_kv_fp8.cuh"

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

bool attn_on_tensor_cores(int D) { return D == 64 || D == 128; }

int attn_ctas(int sms) { return std::min(sms, wdb::AT_MAX_CTAS); }  // one per SM

// Tensor map of the codes of `cache`, a box a page of a head; swizzled as the products
// read it, or as it lies.
int cache_map(const wdb::AttnArgs& a, const uint8_t* cache, CUtensorMap* map, bool swizzled = true) {
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(WD_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dim[2] = {(cuuint64_t)a.D, (cuuint64_t)a.pages * a.Hkv * a.page};
  const cuuint64_t str[1] = {(cuuint64_t)a.D};
  const cuuint32_t box[2] = {(cuuint32_t)a.D, (cuuint32_t)a.page}, ones[2] = {1, 1};
  const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(cache), dim, str, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          !swizzled    ? CU_TENSOR_MAP_SWIZZLE_NONE
                          : a.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                       : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return cr == CUDA_SUCCESS ? WD_OK : fail(WD_ERR_CUDA, "tensor map (cache) encode failed");
}

// Head sizes of the tensor cores; their tensor maps take row numbers of 32 bits and
// a cache of at least a row.
bool attn_fits_tensor_cores(const wdb::AttnArgs& a) {
  const long long rows = (long long)a.Sq * (a.Hq / a.Hkv), cache_rows = (long long)a.pages * a.Hkv * a.page;
  return attn_on_tensor_cores(a.D) && cache_rows > 0 && cache_rows <= 0x7fffffffll && rows <= 0x7fffffffll / 2;
}

bool attn_q_wide(const wdb::AttnArgs& a) { return aligned(a.q, 16) && (a.q_bs | a.q_ts | a.q_hs) % 8 == 0; }

int attn_reach(const wdb::AttnArgs& a) {
  return (int)std::min((long long)a.table_stride * a.page, 0x7fffffffll - wdb::AT_TILE);
}

// On the CUDA cores: any head size; kPrefix: with shared tokens (a.prefix).
template <bool kPrefix>
int attn_simt(const wdb::AttnArgs& a, cudaStream_t s) {
  const long long rows = (long long)a.Sq * (a.Hq / a.Hkv);
  const long long chunks = (rows + wdb::ATTN_ROWS - 1) / wdb::ATTN_ROWS;
  const long long blocks = chunks * a.Hkv * a.B;
  if (blocks > kMaxBlocks) return fail(WD_ERR_UNSUPPORTED, "B * Sq * Hq is too large");
  wdb::attn_fp8_simt_kernel<kPrefix><<<(unsigned)blocks, wdb::ATTN_WARPS * 32, 0, s>>>(a);
  return launched("attn_decode_fp8");
}

}  // namespace

// C ABI of the operators that complete a decoder layer's step
// (include/warp_decode_block.h): argument checks, launch geometry and dispatch.
#include "warp_decode_block.h"

#include "wd_attn_prefix.cuh"
#include "wd_block_norm.cuh"
#include "wd_layer_host.cuh"
#include "wd_linear_w4_tc.cuh"

namespace {

constexpr int kNormSmem = 200 << 10;  // rows on their way in an SM, bytes

// ---- block_norm -------------------------------------------------------------
template <int kUnits, bool kVector>
void launch_norm_block(const wdb::BlockNormArgs& a, bool fp32, cudaStream_t s) {
  const int threads = ((a.H + 8 * kUnits - 1) / (8 * kUnits) + 31) / 32 * 32;
  if (fp32)
    wdb::block_norm_kernel<kUnits, kVector, true, false><<<a.T, threads, 0, s>>>(a);
  else
    wdb::block_norm_kernel<kUnits, kVector, false, false><<<a.T, threads, 0, s>>>(a);
}

// Units of eight values a thread: one, where the row allows.  Measured, one and four:
// 200 x 4096 3.3 and 4.8 us, 4000 x 4096 30 and 38, 16000 x 512 13.5 and 18.5.
template <bool kVector>
void launch_norm(const wdb::BlockNormArgs& a, bool fp32, cudaStream_t s) {
  if (a.H > wdb::BN_MAX_THREADS * 8) return launch_norm_block<2, kVector>(a, fp32, s);
  if (a.H > 256) return launch_norm_block<1, kVector>(a, fp32, s);
  const unsigned blocks = ((unsigned)a.T + wdb::BN_WARP_ROWS - 1) / wdb::BN_WARP_ROWS;
  if (fp32)
    wdb::block_norm_kernel<1, kVector, true, true><<<blocks, 32 * wdb::BN_WARP_ROWS, 0, s>>>(a);
  else
    wdb::block_norm_kernel<1, kVector, false, true><<<blocks, 32 * wdb::BN_WARP_ROWS, 0, s>>>(a);
}

template <bool kFp32, bool kWeightFp32>
int launch_norm_stream(const wdb::BlockNormArgs& a, int threads, int ctas, size_t smem, cudaStream_t s) {
  static std::atomic<unsigned long long> ready{0};  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && !((ready.load(std::memory_order_relaxed) >> dev) & 1ull)) {
    err = cudaFuncSetAttribute(wdb::block_norm_stream_kernel<kFp32, kWeightFp32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kNormSmem);
    if (err == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    g_last_error = std::string("block_norm set-up: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  wdb::block_norm_stream_kernel<kFp32, kWeightFp32><<<ctas, threads, smem, s>>>(a);
  return launched("block_norm");
}

// ---- linear_w4 ----------------------------------------------------------------
template <int kRows, int kTokens, int kGroup, int kScale>
int launch_w4(const wdb::LinearW4Args& a, int split, cudaStream_t s) {
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = split, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(split, (a.N + 16 * kRows - 1) / (16 * kRows), (a.T + 8 * kTokens - 1) / (8 * kTokens));
  cfg.blockDim = dim3(wdb::W4_WARPS * 32);
  cfg.stream = s;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, wdb::linear_w4_kernel<kRows, kTokens, kGroup, kScale>, a);
  if (err != cudaSuccess) {
    cudaGetLastError();
    g_last_error = std::string("linear_w4: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  return launched("linear_w4");
}

template <int kN, int kSums, int kScale>
int launch_w4_tc(const wdb::LinearW4Args& a, const CUtensorMap& x, int sms, cudaStream_t s) {
  using Shape = wdb::W4TcShape<kN>;
  static std::atomic<unsigned long long> ready{0};  // devices whose shared-memory limit is raised
  auto kernel = wdb::linear_w4_tc_kernel<kN, kSums, kScale>;
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && !((ready.load(std::memory_order_relaxed) >> dev) & 1ull)) {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (err == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(wdb::W4T_THREADS);
  cfg.dynamicSmemBytes = Shape::kSmem;
  cfg.stream = s;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  auto split_by = [&](int split) {
    cluster.val.clusterDim.x = split, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
    cfg.gridDim = dim3(split, (a.N + wdb::W4T_ROWS - 1) / wdb::W4T_ROWS, (a.T + kN - 1) / kN);
  };
  // Blocks of a cluster, so that there is about one an SM, as far as each has a step and the
  // clusters all run at once: an SM takes one block, and not every part of the chip has a
  // multiple of eight SMs left (16 tokens of 4096 to 2048: 16 clusters of eight took two
  // turns, 14.2 us, of four 10.2; 2048 to 2048 11.9 and 7.1).
  static std::atomic<int> at_once[kMaxDevices];  // clusters of eight; 0: not asked yet
  const long long tiles = (long long)((a.N + wdb::W4T_ROWS - 1) / wdb::W4T_ROWS) * ((a.T + kN - 1) / kN);
  int split = 1;
  while (split < wdb::W4_MAX_SPLIT && tiles * split * 2 <= sms && split * 2 <= a.blocks) split *= 2;
  if (err == cudaSuccess && split == wdb::W4_MAX_SPLIT) {
    int n = at_once[dev].load(std::memory_order_relaxed);
    if (n == 0) {
      split_by(split);
      err = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (err == cudaSuccess) at_once[dev].store(n = std::max(n, 1), std::memory_order_relaxed);
    }
    if (tiles > n) split /= 2;
  }
  split_by(split);
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&cfg, kernel, a, x);
  if (err != cudaSuccess) {
    cudaGetLastError();
    g_last_error = std::string("linear_w4: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  return launched("linear_w4");
}

template <int kGroup, int kScale>
int launch_w4_tc(const wdb::LinearW4Args& a, cudaStream_t s) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return fail(WD_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const int n = a.T <= 16 ? 16 : a.T <= 32 ? 32 : 64;
  CUtensorMap x;
  const cuuint64_t dim[2] = {(cuuint64_t)a.K, (cuuint64_t)a.T};
  const cuuint64_t str[1] = {(cuuint64_t)a.x_ts * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)n}, ones[2] = {1, 1};
  if (enc(&x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<__nv_bfloat16*>(a.x), dim, str, box, ones,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(WD_ERR_CUDA, "tensor map (x) encode failed");
  constexpr int kSums = 128 / kGroup;
  if (n == 16) return launch_w4_tc<16, kSums, kScale>(a, x, sms, s);
  if (n == 32) return launch_w4_tc<32, kSums, kScale>(a, x, sms, s);
  return launch_w4_tc<64, kSums, kScale>(a, x, sms, s);
}

template <int kGroup, int kScale>
int launch_w4(const wdb::LinearW4Args& a, cudaStream_t s) {
  // Tensor cores fed from shared memory from nine tokens, where a tensor map can take the
  // rows of x. Measured (us a call among others, groups of 128) by matrix instructions on
  // registers, and by these: 16 tokens (9 and 12 within 0.3) of 2048 to 512 5.7, 6.2; to 2048
  // 6.2, 7.1; to 4096 11.5, 7.5; 4096 to 512 6.1, 7.4; to 2048 11.8, 10.2; to 9216 24.1, 16.6;
  // 8192 to 512 11.4, 10.7; to 9216 46.4, 28.9. The first is ahead, by a microsecond, only where N
  // and K are both small. One token (of 4096 to 512, to 9216) 6.1, 8.2; 13.9, 18.4.
  if (a.T > 8 && a.x_wide && a.x_ts >= a.K) return launch_w4_tc<kGroup, kScale>(a, s);
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  // blocks of a cluster, so that there is one an SM, as far as each warp has 128 k
  const int rows = a.T <= 8 ? 16 : 32;
  const long long tiles = (a.N + rows - 1) / rows;
  int split = 1;
  while (split < wdb::W4_MAX_SPLIT && tiles * split < sms && split * 2 * wdb::W4_WARPS <= a.blocks) split *= 2;
  if (a.T <= 8) return launch_w4<1, 1, kGroup, kScale>(a, split, s);
  return launch_w4<2, 4, kGroup, kScale>(a, split, s);
}

template <int kGroup>
int launch_w4(const wdb::LinearW4Args& a, int scale_type, cudaStream_t s) {
  if (scale_type == WD_W4_SCALE_BF16) return launch_w4<kGroup, wdb::W4_BF16>(a, s);
  if (scale_type == WD_W4_SCALE_FP16) return launch_w4<kGroup, wdb::W4_F16>(a, s);
  return launch_w4<kGroup, wdb::W4_F32>(a, s);
}

// ---- attn_decode_fp8_prefix ------------------------------------------------------
// Parts of the workspace, in order.
struct PrefixLayout {
  int row_blocks, own_blocks, own_rows, own_slot;
  bool two;  // prefix units of two row tiles
  size_t plan, own_start, slots, own_slots, bytes;
};

PrefixLayout prefix_layout(int sms, long long B, int Sq, int Hq, int Hkv, int D) {
  PrefixLayout l{};
  const long long own = (long long)Sq * (Hq / Hkv), rows = B * own, tile = wdb::AP_TILE;
  l.two = rows > tile;
  const long long each = l.two ? 2 * tile : tile;
  const long long blocks = (rows + each - 1) / each, own_blocks = (own + tile - 1) / tile;
  l.row_blocks = (int)std::min(blocks, 0x7fffffffll);
  l.own_blocks = (int)std::min(own_blocks, 0x7fffffffll);
  l.own_rows = (int)std::min(own, tile);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  l.plan = wdb::AT_COUNTERS;  // attn_decode_fp8's counters stay zero: the workspace may be its too
  l.own_start = l.plan + wdb::AP_HEADER;
  l.slots = l.own_start + up((size_t)B * 4);
  // a piece's number is its CTA's and its unit's together, and it has a slot for each group
  const size_t ctas = (size_t)attn_ctas(sms), row = (size_t)(D + 4) * 4;
  l.own_slots = l.slots + up(2 * (ctas + (size_t)Hkv * blocks) * tile * row);
  l.own_slot = l.own_rows * (D + 4);  // floats: values are written four at a time
  l.bytes = l.own_slots + 2 * (ctas + (size_t)B * Hkv * own_blocks) * l.own_slot * 4;
  return l;
}

template <int kD>
int launch_prefix(const wdb::AttnPrefixArgs& t, const CUtensorMap (&map)[2], int ctas, cudaStream_t s) {
  using Shape = wdb::AttnPrefixShape<kD>;
  static std::atomic<unsigned long long> ready{0};  // devices whose shared-memory limit is raised
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && !((ready.load(std::memory_order_relaxed) >> dev) & 1ull)) {
    err = cudaFuncSetAttribute(wdb::attn_prefix_kernel<kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (err == cudaSuccess) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    g_last_error = std::string("attn_decode_fp8_prefix set-up: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  wdb::attn_prefix_kernel<kD><<<ctas, wdb::AP_THREADS, Shape::kSmem, s>>>(t, map[0], map[1]);
  if (int rc = launched("attn_decode_fp8_prefix")) return rc;
  const unsigned blocks = (unsigned)(t.a.Hkv * ((t.a.B * t.a.Sq * (t.a.Hq / t.a.Hkv) + 31) / 32));
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks, kD / 32);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, wdb::attn_prefix_join_kernel<kD>, t);
  if (err != cudaSuccess) {
    cudaGetLastError();
    g_last_error = std::string("attn_decode_fp8_prefix join: ") + cudaGetErrorString(err);
    return WD_ERR_CUDA;
  }
  return launched("attn_decode_fp8_prefix join");
}

}  // namespace

extern "C" {

const char* wd_block_last_error_message(void) { return g_last_error.c_str(); }

unsigned long long wd_block_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

int wd_block_status_read(uint32_t* value, int clear) {
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

int wd_block_norm(const void* y, long long y_token_stride, const void* r, long long r_token_stride,
                  int residual_fp32, const void* norm_weight, const void* post_weight, int weight_fp32,
                  const void* gate, long long gate_token_stride, int gate_channel_stride, int gate_fp32,
                  float residual_scale, float eps, void* x, long long x_token_stride, void* residual_out,
                  long long ro_token_stride, int T, int H, void* stream) {
  if (T < 0) return fail(WD_ERR_SHAPE, "T must be >= 0");
  if (H < 1) return fail(WD_ERR_SHAPE, "H must be >= 1");
  if (H > wdb::BN_MAX_H) return fail(WD_ERR_UNSUPPORTED, "H must be <= 16384");
  if (gate && gate_channel_stride != 0 && gate_channel_stride != 1)
    return fail(WD_ERR_SHAPE, "gate_channel_stride must be 0 or 1");
  if (T == 0) return WD_OK;
  if (!y || !r || !norm_weight || !x || !residual_out) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  const uintptr_t ra = residual_fp32 ? 4 : 2, wa = weight_fp32 ? 4 : 2, ga = gate_fp32 ? 4 : 2;
  if (!aligned(y, 2) || !aligned(x, 2) || !aligned(r, ra) || !aligned(residual_out, ra) ||
      !aligned(norm_weight, wa) || !aligned(post_weight, wa) || !aligned(gate, ga))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer");
  wdb::BlockNormArgs a{};
  a.y = static_cast<const __nv_bfloat16*>(y), a.r = r, a.gate = gate, a.norm_w = norm_weight, a.post_w = post_weight;
  a.x = static_cast<__nv_bfloat16*>(x), a.r_out = residual_out;
  a.y_ts = y_token_stride, a.r_ts = r_token_stride, a.g_ts = gate_token_stride;
  a.x_ts = x_token_stride, a.ro_ts = ro_token_stride;
  a.T = T, a.H = H, a.weight_fp32 = weight_fp32 ? 1 : 0, a.gate_fp32 = gate_fp32 ? 1 : 0;
  a.gate_per_token = gate_channel_stride == 0, a.scale = residual_scale, a.eps = eps;
  const long long strides = y_token_stride | r_token_stride | x_token_stride | ro_token_stride |
                            (gate && gate_channel_stride ? gate_token_stride : 0);
  const bool vector = H % 8 == 0 && strides % 8 == 0 && aligned(y, 16) && aligned(r, 16) && aligned(x, 16) &&
                      aligned(residual_out, 16) && aligned(norm_weight, 16) && aligned(post_weight, 16) &&
                      (!gate || gate_channel_stride == 0 || aligned(gate, 16));
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const size_t row = (size_t)H * (2 + ra);
  // Rows copied ahead by blocks that stay, where an SM has enough of them to pay for the
  // blocks' start.  Measured with both weights and the gate, microseconds this way and a
  // block a row: 1200 x 4096 10.6 and 9.9, 2400 x 4096 16.7 and 18.0, 16000 x 4096 97 and
  // 107; 1200 x 2048 6.9 and 5.2, 8000 x 2048 24.9 and 27.8; 4000 x 1024 8.1 and 7.5,
  // 16000 x 1024 24.9 and 26.5.  Wider rows leave an SM two blocks a row at once, so that
  // four rows an SM do: 592 x 7168 9.0 and 10.8, 2400 x 7168 27 and 48.
  const bool many = H > 4096 ? T >= 4 * sms : H >= 1024 && (long long)T * H >= 49152ll * sms;
  if (vector && many && 2 * row <= kNormSmem) {
    // blocks of an SM: its 512 threads of 128 registers, or as many as have two rows on
    // their way each
    const int threads = (H + 1023) / 1024 * 32;
    const int each = (int)std::max<size_t>(1, std::min<size_t>(512 / threads, kNormSmem / (2 * row)));
    a.stages = (int)std::min<size_t>(wdb::BN_MAX_STAGES, kNormSmem / (row * each));
    const size_t smem = row * a.stages;
    const int ctas = std::min((long long)T, (long long)sms * each);
    auto launch = residual_fp32 ? (weight_fp32 ? launch_norm_stream<true, true> : launch_norm_stream<true, false>)
                                : (weight_fp32 ? launch_norm_stream<false, true> : launch_norm_stream<false, false>);
    return launch(a, threads, ctas, smem, static_cast<cudaStream_t>(stream));
  }
  if (vector)
    launch_norm<true>(a, residual_fp32 != 0, static_cast<cudaStream_t>(stream));
  else
    launch_norm<false>(a, residual_fp32 != 0, static_cast<cudaStream_t>(stream));
  return launched("block_norm");
}

int wd_linear_w4(const void* x, long long x_token_stride, const uint8_t* w, const void* scale, int scale_type,
                 const uint8_t* zero, void* out, long long out_token_stride, int T, int N, int K, int group,
                 void* stream) {
  if (T < 0 || N < 0) return fail(WD_ERR_SHAPE, "T and N must be >= 0");
  if (group != 32 && group != 64 && group != 128) return fail(WD_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
  if (K < 1 || K % group != 0) return fail(WD_ERR_SHAPE, "K must be a positive multiple of group");
  if (K > 1 << 30) return fail(WD_ERR_UNSUPPORTED, "K must be <= 2^30");
  if (scale_type < WD_W4_SCALE_BF16 || scale_type > WD_W4_SCALE_FP32)
    return fail(WD_ERR_SHAPE, "scale_type must be 0 (bf16), 1 (fp16) or 2 (fp32)");
  if (T == 0 || N == 0) return WD_OK;
  if (!x || !w || !scale || !out) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(x, 2) || !aligned(out, 2) || !aligned(w, 16) || !aligned(scale, scale_type == WD_W4_SCALE_FP32 ? 4 : 2))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer (w 16 bytes)");
  if ((N + 15) / 16 > 65535 || (T + 7) / 8 > 65535)
    return fail(WD_ERR_UNSUPPORTED, "N must be at most 1048560, T at most 524280");
  wdb::LinearW4Args a{};
  a.x = static_cast<const __nv_bfloat16*>(x), a.w = w, a.scale = scale, a.zero = zero;
  a.out = static_cast<__nv_bfloat16*>(out), a.x_ts = x_token_stride, a.o_ts = out_token_stride;
  a.T = T, a.N = N, a.K = K, a.blocks = (K + 127) / 128, a.groups = K / group;
  a.x_wide = aligned(x, 16) && x_token_stride % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (group == 32) return launch_w4<32>(a, scale_type, s);
  if (group == 64) return launch_w4<64>(a, scale_type, s);
  return launch_w4<128>(a, scale_type, s);
}

int wd_attn_decode_fp8_prefix_workspace(int B, int Sq, int Hq, int Hkv, int D, size_t* bytes) {
  if (!bytes) return fail(WD_ERR_NULL_POINTER, "bytes is NULL");
  if (B < 0 || Sq < 0 || Hq < 0 || Hkv < 1 || Hq % Hkv != 0 || D < 16 || D % 16 != 0)
    return fail(WD_ERR_SHAPE, "inconsistent sizes");
  *bytes = 0;
  if (B == 0 || Sq == 0 || Hq == 0 || !attn_on_tensor_cores(D)) return WD_OK;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  *bytes = prefix_layout(sms, B, Sq, Hq, Hkv, D).bytes;
  return WD_OK;
}

int wd_attn_decode_fp8_prefix(const void* q, long long q_batch_stride, long long q_token_stride,
                              long long q_head_stride, const uint8_t* k_cache, const uint8_t* k_scale,
                              const uint8_t* v_cache, const uint8_t* v_scale, const int32_t* table,
                              int table_stride, const int32_t* seq_lens, const int32_t* prefix_len, void* out,
                              float* lse, float softmax_scale, int window, int B, int Sq, int Hq, int Hkv, int D,
                              int page, int pages, void* workspace, size_t workspace_bytes, uint32_t* status,
                              void* stream) {
  if (int rc = check_cache(B, Hkv, D, page, pages, table_stride)) return rc;
  if (Sq < 0) return fail(WD_ERR_SHAPE, "Sq must be >= 0");
  if (Hq < 1 || Hq % Hkv != 0) return fail(WD_ERR_SHAPE, "Hq must be a positive multiple of Hkv");
  if (window < 0) return fail(WD_ERR_SHAPE, "window must be >= 0");
  if (B == 0 || Sq == 0) return WD_OK;
  if (int rc = check_cache_pointers(k_cache, k_scale, v_cache, v_scale, table, table_stride, seq_lens)) return rc;
  if (!q || !out || !prefix_len) return fail(WD_ERR_NULL_POINTER, "null tensor pointer");
  if (!aligned(q, 2) || !aligned(out, 16) || !aligned(lse, 4) || !aligned(prefix_len, 4))
    return fail(WD_ERR_ALIGNMENT, "misaligned tensor pointer (q 2, out 16, lse 4, prefix_len 4 bytes)");
  wdb::AttnArgs a{};
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.q_bs = q_batch_stride, a.q_ts = q_token_stride, a.q_hs = q_head_stride;
  a.kc = k_cache, a.ks = k_scale, a.vc = v_cache, a.vs = v_scale;
  a.table = table, a.seq_lens = seq_lens, a.prefix = prefix_len, a.out = static_cast<__nv_bfloat16*>(out), a.lse = lse;
  a.status = status;
  a.table_stride = table_stride, a.B = B, a.Sq = Sq, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.page = page;
  a.pages = pages, a.window = window;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!attn_fits_tensor_cores(a)) return attn_simt<true>(a, s);
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  if (!workspace) return fail(WD_ERR_NULL_POINTER, "workspace is NULL");
  if (!aligned(workspace, 16)) return fail(WD_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  const PrefixLayout l = prefix_layout(sms, B, Sq, Hq, Hkv, D);
  if (workspace_bytes < l.bytes)
    return fail(WD_ERR_SHAPE, "workspace is smaller than wd_attn_decode_fp8_prefix_workspace says");
  // rows, and tiles and units' costs, are counted in 32 bits
  const int reach = attn_reach(a);
  const long long most = reach / wdb::AP_TILE + 1 + wdb::AP_UNIT_COST;
  if ((long long)B * Sq * Hq > 0x7fffffffll / 2 ||
      (long long)Hkv * l.row_blocks * 2 * most + (long long)B * Hkv * l.own_blocks * most > 0x7fffffffll)
    return fail(WD_ERR_UNSUPPORTED, "B * Sq * Hq * table_stride * page is too large");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  wdb::AttnPrefixArgs t{};
  t.a = a;
  t.prefix = prefix_len;
  t.plan = ws + l.plan;
  t.own_start = reinterpret_cast<int32_t*>(ws + l.own_start);
  t.slots = reinterpret_cast<float*>(ws + l.slots);
  t.own_slots = reinterpret_cast<float*>(ws + l.own_slots);
  t.row_blocks = l.row_blocks;
  t.two = l.two;
  t.own_blocks = l.own_blocks;
  t.own_rows = l.own_rows;
  t.own_slot = l.own_slot;
  t.reach = reach;
  t.page_shift = page_shift(page);
  t.q_wide = attn_q_wide(a);
  CUtensorMap map[2];
  if (int rc = cache_map(a, k_cache, &map[0])) return rc;
  if (int rc = cache_map(a, v_cache, &map[1], false)) return rc;
  const int ctas = attn_ctas(sms);
  return D == 128 ? launch_prefix<128>(t, map, ctas, s) : launch_prefix<64>(t, map, ctas, s);
}

}  // extern "C"

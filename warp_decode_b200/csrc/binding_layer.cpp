// PyTorch surface of the operators around the FFN (include/warp_decode_layer.h).
// The conventions of binding.cpp: RuntimeError before any launch on bad
// arguments, outputs from the caching allocator, the current stream, no
// synchronisation.
#include "binding.h"

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>

#include "warp_decode_layer.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_rc(int rc) {
  TORCH_CHECK(rc == WD_OK, "warp_decode: ", wd_error_string(rc), ": ", wd_layer_last_error_message());
}

// A contiguous tensor beside `like`, without the dispatcher's detour.
Tensor empty_like_device(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// The current stream of the tensors' device; torch's guard only where another
// device is current.
struct OnDevice {
  c10::cuda::OptionalCUDAGuard guard;
  explicit OnDevice(const Tensor& t) {
    if (t.get_device() != c10::cuda::current_device()) guard.set_index(t.get_device());
  }
};

std::tuple<Tensor, Tensor> moe_router_scored_topk(const Tensor& logits, int64_t topk,
                                                  const std::string& scoring, const OptTensor& bias,
                                                  int64_t n_group, int64_t topk_group,
                                                  int64_t group_top, bool renormalize, double scale) {
  CHECK_CUDA(logits); CHECK_CONTIG(logits);
  TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat,
              "logits must be bf16 or fp32");
  TORCH_CHECK(logits.dim() == 2, "logits must be [T, E]");
  TORCH_CHECK(scoring == "softmax" || scoring == "sigmoid", "scoring must be 'softmax' or 'sigmoid'");
  const int T = to_int(logits.size(0), "T"), E = to_int(logits.size(1), "E"), K = to_int(topk, "topk");
  const float* b = nullptr;
  if (bias.has_value()) {
    CHECK_CUDA(*bias); CHECK_CONTIG(*bias); CHECK_F32(*bias);
    check_same_device(logits, *bias, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == E, "bias must be [E]");
    b = bias->data_ptr<float>();
  }
  const OnDevice on(logits);
  auto ids = empty_like_device(logits, {T, K}, at::kInt);
  auto w = empty_like_device(logits, {T, K}, at::kFloat);
  check_rc(wd_moe_router_scored_topk(logits.data_ptr(), logits.scalar_type() == at::kFloat, b,
                                     ids.data_ptr<int32_t>(), w.data_ptr<float>(), T, E, K,
                                     scoring == "sigmoid", to_int(n_group, "n_group"),
                                     to_int(topk_group, "topk_group"), to_int(group_top, "group_top"),
                                     renormalize, (float)scale, stream_ptr()));
  return {ids, w};
}

void check_rows(const Tensor& x, int64_t dims, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be CUDA");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, name, " must be bf16");
  TORCH_CHECK(x.dim() == dims, name, " must have ", dims, " dimensions");
  TORCH_CHECK(x.stride(dims - 1) == 1 || x.size(dims - 1) <= 1, name, " must be contiguous in its last dimension");
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& q_weight,
                                        const Tensor& k_weight, const Tensor& positions,
                                        const Tensor& cos_sin, double eps, bool interleaved,
                                        bool inplace) {
  check_rows(q, 3, "q");
  check_rows(k, 3, "k");
  const int T = to_int(q.size(0), "T"), Hq = to_int(q.size(1), "Hq"), D = to_int(q.size(2), "D");
  const int Hkv = to_int(k.size(1), "Hkv");
  TORCH_CHECK(k.size(0) == T && k.size(2) == D, "k must be [T, Hkv, D] with q's T and D");
  for (const Tensor* w : {&q_weight, &k_weight}) {
    CHECK_CUDA(*w); CHECK_CONTIG(*w);
    TORCH_CHECK(w->dim() == 1 && w->size(0) == D, "q_weight and k_weight must be [D]");
    TORCH_CHECK((w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat) &&
                    w->scalar_type() == q_weight.scalar_type(),
                "q_weight and k_weight must both be bf16 or both fp32");
  }
  CHECK_CUDA(positions); CHECK_CONTIG(positions); CHECK_I32(positions);
  TORCH_CHECK(positions.dim() == 1 && positions.size(0) == T, "positions must be [T]");
  CHECK_CUDA(cos_sin); CHECK_CONTIG(cos_sin); CHECK_F32(cos_sin);
  TORCH_CHECK(cos_sin.dim() == 2, "cos_sin must be [max_pos, rot]");
  check_same_device(q, k, "k");
  check_same_device(q, q_weight, "q_weight");
  check_same_device(q, k_weight, "k_weight");
  check_same_device(q, positions, "positions");
  check_same_device(q, cos_sin, "cos_sin");
  if (inplace) {  // a head or token that lies on another's place would be written twice
    at::assert_no_internal_overlap(q);
    at::assert_no_internal_overlap(k);
    at::assert_no_overlap(q, k);
  }
  const OnDevice on(q);
  Tensor qo = inplace ? q : empty_like_device(q, {T, Hq, D}, at::kBFloat16);
  Tensor ko = inplace ? k : empty_like_device(k, {T, Hkv, D}, at::kBFloat16);
  check_rc(wd_qk_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                           q_weight.data_ptr(), k_weight.data_ptr(),
                           q_weight.scalar_type() == at::kFloat, positions.data_ptr<int32_t>(),
                           cos_sin.data_ptr<float>(), to_int(cos_sin.size(0), "max_pos"), qo.data_ptr(),
                           qo.stride(0), qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1), T, Hq,
                           Hkv, D, to_int(cos_sin.size(1), "rot"), interleaved, (float)eps, nullptr,
                           stream_ptr()));
  return {qo, ko};
}

// The cache's tensors, checked once for all three entry points.
struct Cache {
  const Tensor &kc, &ks, &vc, &vs, &table;
  int pages, H, page, D, B, cols;
  Cache(const Tensor& k_cache, const Tensor& k_scale, const Tensor& v_cache, const Tensor& v_scale,
        const Tensor& block_table)
      : kc(k_cache), ks(k_scale), vc(v_cache), vs(v_scale), table(block_table) {
    for (const Tensor* t : {&kc, &vc}) {
      TORCH_CHECK(t->is_cuda() && t->is_contiguous() && t->scalar_type() == at::kByte && t->dim() == 4,
                  "k_cache and v_cache must be contiguous CUDA uint8 tensors [pages, Hkv, page, D]");
      TORCH_CHECK(t->sizes() == kc.sizes(), "k_cache and v_cache must have the same shape");
    }
    for (const Tensor* t : {&ks, &vs})
      TORCH_CHECK(t->is_cuda() && t->is_contiguous() && t->scalar_type() == at::kByte && t->dim() == 2 &&
                      t->size(0) == kc.size(0) && t->size(1) == kc.size(1),
                  "k_scale and v_scale must be contiguous CUDA uint8 tensors [pages, Hkv]");
    TORCH_CHECK(table.is_cuda() && table.scalar_type() == at::kInt && table.is_contiguous() &&
                    table.dim() == 2,
                "block_table must be a contiguous CUDA int32 tensor [B, columns]");
    check_same_device(kc, ks, "k_scale");
    check_same_device(kc, vc, "v_cache");
    check_same_device(kc, vs, "v_scale");
    check_same_device(kc, table, "block_table");
    pages = to_int(kc.size(0), "pages");
    H = to_int(kc.size(1), "Hkv");
    page = to_int(kc.size(2), "page");
    D = to_int(kc.size(3), "D");
    B = to_int(table.size(0), "B");
    cols = to_int(table.size(1), "block_table columns");
  }
  const int32_t* per_sequence(const Tensor& t, const char* name) const {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous() && t.dim() == 1 &&
                    t.size(0) == B,
                name, " must be a contiguous CUDA int32 tensor [B]");
    check_same_device(kc, t, name);
    return t.data_ptr<int32_t>();
  }
  const int32_t* per_sequence(const OptTensor& t, const char* name) const {
    return t.has_value() ? per_sequence(*t, name) : nullptr;
  }
};

void kv_cache_write_fp8(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& k_scale,
                        const Tensor& v_cache, const Tensor& v_scale, const Tensor& block_table,
                        const Tensor& start, const OptTensor& lens) {
  const Cache c(k_cache, k_scale, v_cache, v_scale, block_table);
  check_rows(k, 4, "k");
  check_rows(v, 4, "v");
  check_same_device(c.kc, k, "k");
  check_same_device(c.kc, v, "v");
  TORCH_CHECK(k.size(0) == c.B && k.size(2) == c.H && k.size(3) == c.D && v.sizes() == k.sizes(),
              "k and v must be [B, S, Hkv, D]");
  const int32_t* st = c.per_sequence(start, "start");
  const int32_t* ln = c.per_sequence(lens, "lens");
  const OnDevice on(k_cache);
  check_rc(wd_kv_cache_write_fp8(
      k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1),
      v.stride(2), c.kc.data_ptr<uint8_t>(), c.ks.data_ptr<uint8_t>(), c.vc.data_ptr<uint8_t>(),
      c.vs.data_ptr<uint8_t>(), c.table.data_ptr<int32_t>(), c.cols, st, ln, c.B,
      to_int(k.size(1), "S"), c.H, c.D, c.page, c.pages, nullptr, stream_ptr()));
}

std::tuple<Tensor, Tensor> kv_cache_read_fp8(const Tensor& k_cache, const Tensor& k_scale,
                                             const Tensor& v_cache, const Tensor& v_scale,
                                             const Tensor& block_table, const Tensor& start,
                                             int64_t length, const OptTensor& lens) {
  const Cache c(k_cache, k_scale, v_cache, v_scale, block_table);
  const int32_t* st = c.per_sequence(start, "start");
  const int32_t* ln = c.per_sequence(lens, "lens");
  const int R = to_int(length, "length");
  const OnDevice on(k_cache);
  auto ko = empty_like_device(c.kc, {c.B, R, c.H, c.D}, at::kBFloat16);
  auto vo = empty_like_device(c.kc, {c.B, R, c.H, c.D}, at::kBFloat16);
  check_rc(wd_kv_cache_read_fp8(c.kc.data_ptr<uint8_t>(), c.ks.data_ptr<uint8_t>(),
                                c.vc.data_ptr<uint8_t>(), c.vs.data_ptr<uint8_t>(),
                                c.table.data_ptr<int32_t>(), c.cols, st, ln, ko.data_ptr(), vo.data_ptr(),
                                c.B, R, c.H, c.D, c.page, c.pages, nullptr, stream_ptr()));
  return {ko, vo};
}

Tensor attn_decode_fp8_workspace(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D,
                                 c10::optional<int64_t> on) {
  const auto device = on.has_value() ? static_cast<c10::DeviceIndex>(*on) : c10::cuda::current_device();
  const c10::cuda::CUDAGuard guard(device);
  size_t n = 0;
  check_rc(wd_attn_decode_fp8_workspace(to_int(B, "B"), to_int(Sq, "Sq"), to_int(Hq, "Hq"),
                                        to_int(Hkv, "Hkv"), to_int(D, "D"), &n));
  return at::zeros({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
}

py::object attn_decode_fp8(const Tensor& q, const Tensor& k_cache, const Tensor& k_scale,
                           const Tensor& v_cache, const Tensor& v_scale, const Tensor& block_table,
                           const Tensor& seq_lens, c10::optional<double> softmax_scale, int64_t window,
                           const OptTensor& workspace, bool return_lse) {
  const Cache c(k_cache, k_scale, v_cache, v_scale, block_table);
  check_rows(q, 4, "q");
  check_same_device(c.kc, q, "q");
  TORCH_CHECK(q.size(0) == c.B && q.size(3) == c.D, "q must be [B, Sq, Hq, D]");
  const int Sq = to_int(q.size(1), "Sq"), Hq = to_int(q.size(2), "Hq");
  const int32_t* ln = c.per_sequence(seq_lens, "seq_lens");
  const OnDevice on(k_cache);
  Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
    TORCH_CHECK(ws.is_cuda() && ws.is_contiguous(), "workspace must be a contiguous CUDA tensor");
    check_same_device(c.kc, ws, "workspace");
  } else {
    size_t n = 0;
    check_rc(wd_attn_decode_fp8_workspace(c.B, Sq, Hq, c.H, c.D, &n));
    if (n) ws = at::zeros({(int64_t)n}, c.kc.options());
  }
  auto out = empty_like_device(q, {c.B, Sq, Hq, c.D}, at::kBFloat16);
  Tensor lse;
  if (return_lse) lse = empty_like_device(q, {c.B, Sq, Hq}, at::kFloat);
  check_rc(wd_attn_decode_fp8(
      q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), c.kc.data_ptr<uint8_t>(),
      c.ks.data_ptr<uint8_t>(), c.vc.data_ptr<uint8_t>(), c.vs.data_ptr<uint8_t>(),
      c.table.data_ptr<int32_t>(), c.cols, ln, out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
      softmax_scale.has_value() ? (float)*softmax_scale : (float)(1.0 / std::sqrt((double)c.D)),
      to_int(window, "window"), c.B, Sq, Hq, c.H, c.D, c.page, c.pages,
      ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.nbytes() : 0, nullptr, stream_ptr()));
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

}  // namespace

void bind_layer(py::module_& m) {
  m.def("moe_router_scored_topk", &moe_router_scored_topk,
        "expert choice from router logits [T, E]: softmax / sigmoid scores, balance bias, expert "
        "groups, top-k, weights -> (ids int32 [T, topk], weights fp32 [T, topk])",
        py::arg("logits"), py::arg("topk"), py::arg("scoring") = "softmax", py::arg("bias") = py::none(),
        py::arg("n_group") = 1, py::arg("topk_group") = 1, py::arg("group_top") = 1,
        py::arg("renormalize") = true, py::arg("scale") = 1.0);
  m.def("qk_norm_rope", &qk_norm_rope,
        "RMS norm of every query and key head and the position rotation in one pass -> (q, k)",
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("positions"),
        py::arg("cos_sin"), py::arg("eps") = 1e-6, py::arg("interleaved") = false,
        py::arg("inplace") = false);
  m.def("kv_cache_write_fp8", &kv_cache_write_fp8,
        "quantise new keys and values [B, S, Hkv, D] into the paged E4M3 cache (in place)",
        py::arg("k"), py::arg("v"), py::arg("k_cache"), py::arg("k_scale"), py::arg("v_cache"),
        py::arg("v_scale"), py::arg("block_table"), py::arg("start"), py::arg("lens") = py::none());
  m.def("kv_cache_read_fp8", &kv_cache_read_fp8,
        "read `length` tokens of each sequence back from the paged E4M3 cache -> (k, v) bf16",
        py::arg("k_cache"), py::arg("k_scale"), py::arg("v_cache"), py::arg("v_scale"),
        py::arg("block_table"), py::arg("start"), py::arg("length"), py::arg("lens") = py::none());
  m.def("attn_decode_fp8_workspace", &attn_decode_fp8_workspace,
        "zeroed workspace for attn_decode_fp8 calls of these sizes (one per concurrently used stream), on "
        "the current device or the one given",
        py::arg("B"), py::arg("Sq"), py::arg("Hq"), py::arg("Hkv"), py::arg("D"), py::arg("device") = py::none());
  m.def("attn_decode_fp8", &attn_decode_fp8,
        "attention of the last Sq tokens of each sequence over its paged E4M3 cache -> out bf16 "
        "[B, Sq, Hq, D], with return_lse (out, lse)",
        py::arg("q"), py::arg("k_cache"), py::arg("k_scale"), py::arg("v_cache"), py::arg("v_scale"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("softmax_scale") = py::none(),
        py::arg("window") = 0, py::arg("workspace") = py::none(), py::arg("return_lse") = false);
}

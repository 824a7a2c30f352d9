// PyTorch surface of the operators that complete a decoder layer's step
// (include/warp_decode_block.h), in the conventions of binding_layer.cpp.
#include "binding_cache.h"

#include <ATen/MemoryOverlap.h>

#include "warp_decode_block.h"

namespace {

void check_rc(int rc) {
  TORCH_CHECK(rc == WD_OK, "warp_decode: ", wd_error_string(rc), ": ", wd_block_last_error_message());
}

bool bf16_or_fp32(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

// Rows of bytes in device memory: `rows` of `bytes`, `stride` apart.
struct Rows {
  int64_t at, rows, stride, bytes;
  explicit Rows(const Tensor& t) {  // one or two dimensions, the last contiguous or one value repeated
    const int64_t d = t.dim(), size = t.element_size(), n = t.size(d - 1);
    at = reinterpret_cast<int64_t>(t.data_ptr());
    rows = t.numel() == 0 ? 0 : d == 2 ? t.size(0) : 1;
    stride = d == 2 ? t.stride(0) * size : 0;
    bytes = (n > 1 && t.stride(d - 1) != 0 ? n : 1) * size;
    if (rows > 1 && stride == 0) rows = 1;
  }
  int64_t end() const { return at + (rows - 1) * stride + bytes; }
};

// Whether some row of one lies on some row of the other; a's rows do not meet each other.
bool meet(const Rows& a, const Rows& b) {
  if (a.rows == 0 || b.rows == 0 || a.end() <= b.at || b.end() <= a.at) return false;
  if (a.rows > 1 && (b.rows == 1 || a.stride == b.stride)) {  // b's place among a's columns
    const int64_t from = ((b.at - a.at) % a.stride + a.stride) % a.stride;
    return from < a.bytes || from + b.bytes > a.stride;
  }
  for (int64_t i = 0; i < b.rows; ++i) {  // the last of a's rows that begins before a row of b ends
    const int64_t begin = b.at + i * b.stride, before = begin + b.bytes - 1 - a.at;
    if (before < 0) continue;
    const int64_t j = a.rows == 1 ? 0 : std::min(before / a.stride, a.rows - 1);
    if (a.at + j * a.stride + a.bytes > begin) return true;
  }
  return false;
}

std::tuple<Tensor, Tensor> block_norm(const Tensor& y, const Tensor& residual, const Tensor& norm_weight,
                                      const OptTensor& post_weight, const OptTensor& gate, double residual_scale,
                                      double eps, bool inplace) {
  check_rows(y, 2, "y");
  const int T = to_int(y.size(0), "T"), H = to_int(y.size(1), "H");
  TORCH_CHECK(residual.is_cuda() && bf16_or_fp32(residual), "residual must be a CUDA bf16 or fp32 tensor");
  TORCH_CHECK(residual.dim() == 2 && residual.size(0) == T && residual.size(1) == H &&
                  (residual.stride(1) == 1 || H <= 1),
              "residual must be [T, H] with y's sizes, contiguous in its last dimension");
  check_same_device(y, residual, "residual");
  for (const Tensor* w : {&norm_weight, post_weight.has_value() ? &*post_weight : &norm_weight}) {
    CHECK_CUDA(*w); CHECK_CONTIG(*w);
    TORCH_CHECK(w->dim() == 1 && w->size(0) == H, "norm_weight and post_weight must be [H]");
    TORCH_CHECK(bf16_or_fp32(*w) && w->scalar_type() == norm_weight.scalar_type(),
                "norm_weight and post_weight must both be bf16 or both fp32");
    check_same_device(y, *w, "norm_weight, post_weight");
  }
  const void* g = nullptr;
  long long g_ts = 0;
  int g_cs = 0, g_fp32 = 0;
  if (gate.has_value()) {  // [H], [T, 1], [1, H] or [T, H]
    TORCH_CHECK(gate->is_cuda() && bf16_or_fp32(*gate), "gate must be a CUDA bf16 or fp32 tensor");
    check_same_device(y, *gate, "gate");
    const int64_t d = gate->dim();
    TORCH_CHECK((d == 1 && gate->size(0) == H) ||
                    (d == 2 && (gate->size(0) == T || gate->size(0) == 1) && (gate->size(1) == H || gate->size(1) == 1)),
                "gate must be [H], [T, 1], [1, H] or [T, H]");
    const bool many = gate->size(d - 1) > 1;
    TORCH_CHECK(!many || gate->stride(d - 1) == 1 || gate->stride(d - 1) == 0,
                "gate must be contiguous in its last dimension");
    g = gate->data_ptr();
    g_cs = many ? (int)gate->stride(d - 1) : 0;
    g_ts = d == 2 && gate->size(0) > 1 ? gate->stride(0) : 0;
    g_fp32 = gate->scalar_type() == at::kFloat;
  }
  if (inplace) {  // a value written before another row reads it
    at::assert_no_internal_overlap(residual);
    TORCH_CHECK(T <= 1 || std::abs(residual.stride(0)) >= H, "residual's rows must not share memory when updated in place");
    const Rows r(residual);
    for (const Tensor* t : {&y, &norm_weight, post_weight.has_value() ? &*post_weight : nullptr,
                            gate.has_value() ? &*gate : nullptr})
      TORCH_CHECK(!t || !meet(r, Rows(*t)),
                  "residual, which is updated in place, has a memory location in common with another input");
  }
  const OnDevice on(y);
  Tensor x = empty_like_device(y, {T, H}, at::kBFloat16);
  Tensor ro = inplace ? residual : empty_like_device(y, {T, H}, residual.scalar_type());
  check_rc(wd_block_norm(y.data_ptr(), y.stride(0), residual.data_ptr(), residual.stride(0),
                         residual.scalar_type() == at::kFloat, norm_weight.data_ptr(),
                         post_weight.has_value() ? post_weight->data_ptr() : nullptr,
                         norm_weight.scalar_type() == at::kFloat, g, g_ts, g_cs, g_fp32, (float)residual_scale,
                         (float)eps, x.data_ptr(), x.stride(0), ro.data_ptr(), ro.stride(0), T, H, stream_ptr()));
  return {x, ro};
}

Tensor linear_w4(const Tensor& x, const Tensor& w, const Tensor& w_scale, const OptTensor& w_zero) {
  TORCH_CHECK(x.dim() == 2, "x must be [T, K]");
  check_rows(x, 2, "x");
  const int T = to_int(x.size(0), "T"), K = to_int(x.size(1), "K");
  CHECK_CUDA(w); CHECK_CONTIG(w); CHECK_U8(w);
  TORCH_CHECK(w.dim() == 2 && w.size(1) == (int64_t)(K + 127) / 128 * 64, "w must be [N, ceil(K / 128) * 64]");
  const int N = to_int(w.size(0), "N");
  CHECK_CUDA(w_scale); CHECK_CONTIG(w_scale);
  TORCH_CHECK(w_scale.dim() == 2 && w_scale.size(0) == N && w_scale.size(1) > 0 && K % w_scale.size(1) == 0,
              "w_scale must be [N, K / group]");
  const auto st = w_scale.scalar_type();
  TORCH_CHECK(st == at::kBFloat16 || st == at::kHalf || st == at::kFloat, "w_scale must be bf16, fp16 or fp32");
  check_same_device(x, w, "w");
  check_same_device(x, w_scale, "w_scale");
  const uint8_t* zero = nullptr;
  if (w_zero.has_value()) {
    CHECK_CUDA(*w_zero); CHECK_CONTIG(*w_zero); CHECK_U8(*w_zero);
    TORCH_CHECK(w_zero->sizes() == w_scale.sizes(), "w_zero must be [N, K / group] like w_scale");
    check_same_device(x, *w_zero, "w_zero");
    zero = w_zero->data_ptr<uint8_t>();
  }
  const OnDevice on(x);
  Tensor out = empty_like_device(x, {T, N}, at::kBFloat16);
  check_rc(wd_linear_w4(x.data_ptr(), x.stride(0), w.data_ptr<uint8_t>(), w_scale.data_ptr(),
                        st == at::kBFloat16 ? WD_W4_SCALE_BF16 : st == at::kHalf ? WD_W4_SCALE_FP16 : WD_W4_SCALE_FP32,
                        zero, out.data_ptr(), out.stride(0), T, N, K, K / to_int(w_scale.size(1), "groups"),
                        stream_ptr()));
  return out;
}

Tensor attn_decode_fp8_prefix_workspace(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D,
                                        c10::optional<int64_t> on) {
  const auto device = on.has_value() ? static_cast<c10::DeviceIndex>(*on) : c10::cuda::current_device();
  const c10::cuda::CUDAGuard guard(device);
  size_t n = 0;
  check_rc(wd_attn_decode_fp8_prefix_workspace(to_int(B, "B"), to_int(Sq, "Sq"), to_int(Hq, "Hq"),
                                               to_int(Hkv, "Hkv"), to_int(D, "D"), &n));
  return at::zeros({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, device));
}

py::object attn_decode_fp8_prefix(const Tensor& q, const Tensor& k_cache, const Tensor& k_scale,
                                  const Tensor& v_cache, const Tensor& v_scale, const Tensor& block_table,
                                  const Tensor& seq_lens, const Tensor& prefix_len,
                                  c10::optional<double> softmax_scale, int64_t window, const OptTensor& workspace,
                                  bool return_lse) {
  const Cache c(k_cache, k_scale, v_cache, v_scale, block_table);
  check_rows(q, 4, "q");
  check_same_device(c.kc, q, "q");
  TORCH_CHECK(q.size(0) == c.B && q.size(3) == c.D, "q must be [B, Sq, Hq, D]");
  const int Sq = to_int(q.size(1), "Sq"), Hq = to_int(q.size(2), "Hq");
  const int32_t* ln = c.per_sequence(seq_lens, "seq_lens");
  TORCH_CHECK(prefix_len.is_cuda() && prefix_len.scalar_type() == at::kInt && prefix_len.numel() == 1,
              "prefix_len must be a CUDA int32 tensor of one value");
  check_same_device(c.kc, prefix_len, "prefix_len");
  const OnDevice on(k_cache);
  Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
    TORCH_CHECK(ws.is_cuda() && ws.is_contiguous(), "workspace must be a contiguous CUDA tensor");
    check_same_device(c.kc, ws, "workspace");
  } else {
    size_t n = 0;
    check_rc(wd_attn_decode_fp8_prefix_workspace(c.B, Sq, Hq, c.H, c.D, &n));
    if (n) ws = at::zeros({(int64_t)n}, c.kc.options());
  }
  auto out = empty_like_device(q, {c.B, Sq, Hq, c.D}, at::kBFloat16);
  Tensor lse;
  if (return_lse) lse = empty_like_device(q, {c.B, Sq, Hq}, at::kFloat);
  check_rc(wd_attn_decode_fp8_prefix(
      q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), c.kc.data_ptr<uint8_t>(), c.ks.data_ptr<uint8_t>(),
      c.vc.data_ptr<uint8_t>(), c.vs.data_ptr<uint8_t>(), c.table.data_ptr<int32_t>(), c.cols, ln,
      prefix_len.data_ptr<int32_t>(), out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
      softmax_scale.has_value() ? (float)*softmax_scale : (float)(1.0 / std::sqrt((double)c.D)),
      to_int(window, "window"), c.B, Sq, Hq, c.H, c.D, c.page, c.pages, ws.defined() ? ws.data_ptr() : nullptr,
      ws.defined() ? ws.nbytes() : 0, nullptr, stream_ptr()));
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

}  // namespace

void bind_block(py::module_& m) {
  m.def("block_norm", &block_norm,
        "between two blocks: a block's output (normed with post_weight), gated onto the scaled residual, and the "
        "norm before the next block -> (x bf16 [T, H], residual [T, H])",
        py::arg("y"), py::arg("residual"), py::arg("norm_weight"), py::arg("post_weight") = py::none(),
        py::arg("gate") = py::none(), py::arg("residual_scale") = 1.0, py::arg("eps") = 1e-6,
        py::arg("inplace") = false);
  m.def("linear_w4", &linear_w4,
        "x [T, K] bf16 times 4-bit weights with a scale (and zero point) per group of 32, 64 or 128 -> [T, N] bf16",
        py::arg("x"), py::arg("w"), py::arg("w_scale"), py::arg("w_zero") = py::none());
  m.def("attn_decode_fp8_prefix_workspace", &attn_decode_fp8_prefix_workspace,
        "zeroed workspace for attn_decode_fp8_prefix calls of these sizes, on the current device unless one is named",
        py::arg("B"), py::arg("Sq"), py::arg("Hq"), py::arg("Hkv"), py::arg("D"), py::arg("device") = py::none());
  m.def("attn_decode_fp8_prefix", &attn_decode_fp8_prefix,
        "attn_decode_fp8 of sequences that begin with the same prefix_len tokens in the same pages, which are read "
        "once for all of them",
        py::arg("q"), py::arg("k_cache"), py::arg("k_scale"), py::arg("v_cache"), py::arg("v_scale"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("prefix_len"), py::arg("softmax_scale") = py::none(),
        py::arg("window") = 0, py::arg("workspace") = py::none(), py::arg("return_lse") = false);
}

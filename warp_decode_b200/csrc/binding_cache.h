// What the PyTorch surfaces of the operators around the FFN share: devices, rows
// and the checks of the FP8 cache's tensors.
#pragma once

#include "binding.h"

#include <ATen/cuda/EmptyTensor.h>

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

// A contiguous tensor beside `like`, without the dispatcher's detour.
inline Tensor empty_like_device(const Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
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

inline void check_rows(const Tensor& x, int64_t dims, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be CUDA");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, name, " must be bf16");
  TORCH_CHECK(x.dim() == dims, name, " must have ", dims, " dimensions");
  TORCH_CHECK(x.stride(dims - 1) == 1 || x.size(dims - 1) <= 1, name, " must be contiguous in its last dimension");
}

// The cache's tensors, checked once for all entry points that take it.
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

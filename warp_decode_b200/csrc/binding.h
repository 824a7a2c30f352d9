// Argument checks shared by the files of the PyTorch extension.
#pragma once

#include <torch/extension.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#define CHECK_CUDA(x) TORCH_CHECK((x).is_cuda(), #x " must be CUDA")
#define CHECK_CONTIG(x) TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")
#define CHECK_BF16(x) TORCH_CHECK((x).scalar_type() == at::kBFloat16, #x " must be bf16")
#define CHECK_F32(x) TORCH_CHECK((x).scalar_type() == at::kFloat, #x " must be fp32")
#define CHECK_I32(x) TORCH_CHECK((x).scalar_type() == at::kInt, #x " must be int32")
#define CHECK_U8(x) TORCH_CHECK((x).scalar_type() == at::kByte, #x " must be uint8")

inline void check_same_device(const torch::Tensor& a, const torch::Tensor& b, const char* name) {
  TORCH_CHECK(a.device() == b.device(), name, " must be on the same device as the first input");
}

inline int to_int(int64_t v, const char* what) {
  TORCH_CHECK(v >= 0 && v <= INT32_MAX, what, " out of int32 range");
  return static_cast<int>(v);
}

inline void* stream_ptr() { return reinterpret_cast<void*>(at::cuda::getCurrentCUDAStream().stream()); }

// Registers the operators around the FFN (binding_layer.cpp).
void bind_layer(pybind11::module_& m);
// Registers the operators that complete a layer's step (binding_block.cpp).
void bind_block(pybind11::module_& m);

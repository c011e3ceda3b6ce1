// Checks and conversions shared by the files of the PyTorch front end (torch_ext.cpp, torch_layer.cpp).
#pragma once

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <optional>

#include "ssd_b200.h"

namespace ssd_torch {

using torch::Tensor;
using OptTensor = std::optional<Tensor>;

inline int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return SSD_F32;
    case at::kBFloat16: return SSD_BF16;
    case at::kHalf: return SSD_F16;
    default: TORCH_CHECK(false, name, ": dtype ", t.scalar_type(), " is not fp32 / bf16 / fp16");
  }
}
inline int dtype_code(at::ScalarType st) {
  switch (st) {
    case at::kFloat: return SSD_F32;
    case at::kBFloat16: return SSD_BF16;
    case at::kHalf: return SSD_F16;
    default: TORCH_CHECK(false, "dtype ", st, " is not fp32 / bf16 / fp16");
  }
}

inline void check_cuda(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (libssd_b200 has no CPU path)");
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", expected ", like.device());
}

inline ssd_stream_t current_stream(const Tensor& t) {
  return reinterpret_cast<ssd_stream_t>(c10::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

inline void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == SSD_OK, what, " failed (status ", rc, "): ", ssd_last_error());
}

template <int N>
void copy_strides(int64_t (&dst)[N], const Tensor& t, std::initializer_list<int> dims) {
  int i = 0;
  for (int d : dims) dst[i++] = t.stride(d);
}

inline Tensor as_int32(const Tensor& seq_idx) {
  return seq_idx.scalar_type() == at::kInt ? seq_idx : seq_idx.to(at::kInt);
}

// An output tensor; between guard bands when debug_set_guard_bytes asked for them (torch_ext.cpp).
Tensor alloc_out(at::IntArrayRef sizes, const at::TensorOptions& opts);
// The same straight from the CUDA allocator, for the operators around the scan: what torch::empty's dispatch adds
// is a third of a small call's time.  Dispatch modes, the profiler's list of operators and the deterministic mode's
// fill do not see such an output.
Tensor alloc_direct(at::IntArrayRef sizes, const at::TensorOptions& opts);

// Adds the operators around the scan (torch_layer.cpp).
void bind_layer(pybind11::module& m);

}  // namespace ssd_torch

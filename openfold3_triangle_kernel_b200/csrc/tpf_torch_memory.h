// Memory, streams and element types for the operators that launch through C++ structures (tpf_torch_rows.cpp,
// tpf_torch_sequence.cpp).
#pragma once

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>

#include "tpf_torch.h"

namespace tpf_torch {

using MaybeTensor = std::optional<Tensor>;

// Straight from the allocator of the current device: a tensor through the dispatcher costs 1.2 us, and a small training
// pass makes six.
inline Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
struct Scratch {  // device memory of a call
  c10::DataPtr p;
  explicit Scratch(int64_t bytes) {
    if (bytes > 0) p = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  }
  void* get() const { return p.get(); }
};

inline cudaStream_t cu_stream() { return static_cast<cudaStream_t>(stream()); }

inline int row_type(const Tensor& t) {  // -1: not a type of these operators
  switch (t.scalar_type()) {
    case at::kFloat: return TPF_F32;
    case at::kBFloat16: return TPF_BF16;
    case at::kHalf: return TPF_F16;
    default: return -1;
  }
}

inline void* ptr_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline int type_of(const Tensor& t) { return t.defined() ? row_type(t) : 0; }

}  // namespace tpf_torch

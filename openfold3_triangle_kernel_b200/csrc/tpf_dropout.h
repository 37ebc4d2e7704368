// Host entry point of the dropout (tpf_dropout.cu) that the C ABI and the torch layer call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tpf {

// Elements (p, q, s, e), e contiguous; the mask is shared along s where `shared` is set.
struct DropoutCall {
  const void* x;
  const void* residual;  // or nullptr
  void* out;
  int64_t x_strides[3], residual_strides[3], out_strides[3];  // of p, q, s, in elements
  int64_t sizes[4];
  int type;              // RowType
  int shared;
  int threshold;         // of 65536: the probability of an element to be dropped
  const int64_t* seed_ptr;  // (seed, offset) on the device, or nullptr: the values
  int64_t seed, offset;
};
int dropout(const DropoutCall& c, cudaStream_t stream);

}  // namespace tpf

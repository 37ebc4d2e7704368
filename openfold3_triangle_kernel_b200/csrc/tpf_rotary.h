// Host entry points of the position rotation (tpf_rotary.cu) that the C ABI and the torch layer call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tpf {

// One of the two tensors of a call, [B, N, H, D]; heads = 0: it is not there.
struct RotaryTensor {
  const void* x;       // the forward's input; in a backward pass nullptr without a norm
  int64_t strides[3];  // of B, N, H in elements; D is contiguous
  int64_t heads;
  const void* weight;  // [D], or nullptr: ones
  int weight_type;
  const void* dy;      // backward: the output's gradient, contiguous
  void* out;           // forward: the result; backward: x's gradient; contiguous
  void* dweight;       // backward: [D] of weight_type, or nullptr
};
struct RotaryCall {
  RotaryTensor t[2];
  int type;                   // RowType of x, dy and out
  int64_t batch, tokens, dim, rot;
  const int64_t* turns;       // [rot / 2], turns a position as a fraction of 2^64
  float magnitude;
  const int64_t* positions;   // [batch, tokens], or nullptr: first, first + 1, ...
  int64_t first;
  int half;                   // 1: element i with i + rot / 2; 0: 2 i with 2 i + 1
  int norm;
  float eps;
};
int rotary_fwd(const RotaryCall& c, cudaStream_t stream);
int64_t rotary_bwd_workspace_bytes(int64_t dim);
int rotary_bwd(const RotaryCall& c, void* workspace, int64_t workspace_bytes, cudaStream_t stream);

}  // namespace tpf

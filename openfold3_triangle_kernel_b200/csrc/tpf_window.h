// Host entry points of the window attention (tpf_window.cu) that the C ABI and the torch layer call.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tpf {

constexpr int64_t kWindowMost = 1ll << 28;       // tokens, keys, reach of a limited window, magnitude of an offset
constexpr int kWindowUnlimited = 1 << 30;        // a reach beyond every key
constexpr int kMostSinks = 64;

// One problem.  Strides in elements, order (batch, token, head); the last dimension is contiguous.
struct WindowCall {
  int64_t B, N, M, H, HK, D;      // queries, keys, their heads, elements of a head (a multiple of 8, at most 128)
  int type;                       // TPF_BF16 or TPF_F16
  float scale;
  int left, right;                // kWindowUnlimited: no limit
  int sinks;
  const int* offsets;             // [B] position of query 0, or nullptr: `offset`
  int64_t offset;
  const int* lengths;             // [B] keys of a sequence, or nullptr: M
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  void* out;                      // [B, N, H, D] contiguous
  float* lse;                     // [B, H, N], or nullptr
  // backward
  const void* d_out;              // contiguous, as out
  void *dq, *dk, *dv;             // contiguous; nullptr: not wanted
};
int window_attn_fwd(const WindowCall& c, cudaStream_t stream);
int64_t window_attn_bwd_workspace_bytes(const WindowCall& c);
int window_attn_bwd(const WindowCall& c, void* workspace, int64_t workspace_bytes, cudaStream_t stream);

}  // namespace tpf

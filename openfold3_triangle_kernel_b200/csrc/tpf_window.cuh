// Window attention: which keys a query sees, and what its kernels share.
//
//   position of query i of batch b: p = offset_b + i;   it sees key j iff  j < len_b,  j <= p + right,  and j >= p - left or j < sinks
//   S = scale q k;  P = softmax over the seen keys (0 where there are none);  out = P v;  lse = log sum exp S (-inf)
//
// H / HK query heads share a key head.  Positions are 32-bit numbers: offsets are clamped to +-2^29, lengths to 0 .. M; M and N are at
// most 2^28, a limited reach below 2^28, an unlimited one is 2^30, so no sum of them passes 2^31.
#pragma once

#include "tpf_rows.cuh"
#include "tpf_window.h"

namespace tpf {

struct WindowParams {
  int B, N, M, H, HK, D, G;   // G = H / HK
  int left, right, sinks;
  const int* offsets;
  int offset;
  const int* lengths;
  float scale;
  __device__ __forceinline__ int first_position(int b) const {
    return offsets != nullptr ? max(-(1 << 29), min(1 << 29, __ldg(offsets + b))) : offset;
  }
  __device__ __forceinline__ int length(int b) const { return lengths != nullptr ? max(0, min(M, __ldg(lengths + b))) : M; }
};

// The keys that the queries at positions p0 .. p1 reach: [lo, hi) of the window, and the sinks [0, sink) before it.
struct KeyRange {
  int lo, hi, sink;
};
__device__ __forceinline__ KeyRange key_range(const WindowParams& p, int len, int p0, int p1) {
  KeyRange r;
  r.hi = max(0, min(len, p1 + p.right + 1));
  r.lo = min(max(0, p0 - p.left), r.hi);
  r.sink = min(min(p.sinks, r.lo), r.hi);
  return r;
}

// The lowest n of 64 bits, n at or beyond the ends included.
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
// Which of the 64 keys from j0 on the query at position `pos` sees, and which of the 64 queries from position p0 on see key j.
__device__ __forceinline__ uint64_t seen_keys(const WindowParams& p, int len, int pos, int j0) {
  const int hi = min(len, pos + p.right + 1) - j0;
  return low_bits(hi) & (~low_bits(pos - p.left - j0) | low_bits(p.sinks - j0));
}
__device__ __forceinline__ uint64_t seeing_queries(const WindowParams& p, int len, int j, int p0) {
  if (j >= len) return 0;
  return (j < p.sinks ? ~0ull : low_bits(j + p.left + 1 - p0)) & ~low_bits(j - p.right - p0);
}

// UMMA instruction descriptor of kind::f16 with fp32 sums: both operands bf16 or both fp16.
template <typename T>
__host__ __device__ constexpr uint32_t window_idesc(int M, int N, bool b_mn) {
  return (make_idesc_bf16(M, N, false, b_mn) & ~((7u << 7) | (7u << 10))) |
         (std::is_same<T, bf16>::value ? (1u << 7) | (1u << 10) : 0u);
}

constexpr float kWindowLog2e = 1.4426950408889634f;

}  // namespace tpf

// The parts of the normalised projection (tpf_norm_linear.cu).
#pragma once

#include "tpf_layer_norm.cuh"

namespace tpf {

int64_t norm_linear_dw_workspace_bytes(int64_t rows, int64_t cols, int64_t outs);
// dw [outs, cols] = d_out^T y~; y~ from norm.codes where they are given, else from norm.x.
int norm_linear_dw(const NormArgs& norm, const void* d_out, int64_t outs, void* dw, int dw_type, void* workspace,
                   cudaStream_t stream);

// A few rows (tpf_norm_linear_fwd.cu).
bool norm_linear_few(int64_t rows);
int norm_linear_few_fwd(const NormArgs& norm, const void* w, int64_t outs, void* out, float eps, cudaStream_t stream);

// Narrow rows: up to 128 columns and a weight that stays in shared memory.  Forward (tpf_norm_linear_fwd.cu; no scratch);
// backward (tpf_norm_linear_bwd.cu): scratch, all gradients that g asks for.
bool norm_linear_narrow(int64_t cols, int64_t outs);
int norm_linear_narrow_fwd(const NormArgs& norm, const void* w, int64_t outs, void* out, float eps, cudaStream_t stream);
int64_t norm_linear_narrow_bwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs);
int norm_linear_narrow_bwd(const NormArgs& norm, const void* w, int64_t outs, const NormLinearGrads& g, void* workspace,
                           cudaStream_t stream);

// A warp's block of 32 x 32 sums, a lane with a row of it (as they come from TMEM), through shared memory to put(row, column,
// four sums): eight lanes a row, so that memory gets whole lines.
constexpr int kBlockPitch = 36, kBlockStaging = 32 * kBlockPitch * 4;  // floats (16-byte pieces without conflicts), bytes
template <class Put>
__device__ __forceinline__ void put_block(void* staging, const uint32_t (&v)[32], int lane, const Put& put) {
  float* rows = static_cast<float*>(staging);
#pragma unroll
  for (int e = 0; e < 32; e += 4)
    *reinterpret_cast<uint4*>(rows + lane * kBlockPitch + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int r = p * 4 + (lane >> 3), c = (lane & 7) * 4;
    put(r, c, *reinterpret_cast<const float4*>(rows + r * kBlockPitch + c));
  }
  __syncwarp();
}

}  // namespace tpf

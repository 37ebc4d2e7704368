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

}  // namespace tpf

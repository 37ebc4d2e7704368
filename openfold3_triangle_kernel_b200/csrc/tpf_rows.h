// Host entry points of the row-wise operators (tpf_layer_norm.cu, tpf_int8.cu, tpf_norm_linear.cu) that the C ABI forwards to.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tpf {

// Codes of a layer norm: rows start on 16-byte boundaries.
inline int64_t code_pitch(int64_t cols) { return (cols + 15) / 16 * 16; }

struct NormCall {
  int64_t rows, cols;
  int type;               // of x, y, dy and dx: RowType
  const void* x;          // [rows, cols], row pitch x_pitch elements; may be nullptr in a backward pass from codes
  int64_t x_pitch;
  void* codes;            // int8 [rows, code_pitch(cols)], or nullptr
  float* scales;          // [rows, ceil(cols / 128)]
  float *mean, *rstd;     // [rows]; may be nullptr in a forward that keeps nothing
  const void *weight, *bias;  // [cols] or nullptr
  int weight_type, bias_type;
};
int layer_norm_fwd(const NormCall& c, void* y, float eps, cudaStream_t stream);

struct NormGrads {
  const void* dy;  // contiguous
  void* dx;        // contiguous, or nullptr
  void *dweight, *dbias;  // [cols] or nullptr
  int dweight_type, dbias_type;
};
int64_t layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols);
int layer_norm_bwd(const NormCall& c, const NormGrads& g, void* workspace, int64_t workspace_bytes, cudaStream_t stream);

// dweight[c], dbias[c] = sums over terms [count][2][cols]; either may be nullptr
int norm_fold(const float* terms, int count, int cols, void* dweight, int dweight_type, void* dbias, int dbias_type,
              cudaStream_t stream);

// x [rows, cols] (pitch in elements) <-> codes int8 [rows, cols], scales fp32 [rows, ceil(cols / 128)]
int int8_pack(const void* x, int64_t x_pitch, int type, void* codes, float* scales, int64_t rows, int64_t cols,
              cudaStream_t stream);
int int8_unpack(const void* codes, const float* scales, int type, void* x, int64_t rows, int64_t cols, cudaStream_t stream);

// out = layer_norm(x) W^T, bf16, cols and outs multiples of 8.  `norm`: as in the layer norm, with the codes, mean and rstd
// kept where they are not nullptr.
int64_t norm_linear_fwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs);
int norm_linear_fwd(const NormCall& norm, const void* w, int64_t outs, void* out, float eps, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream);
struct NormLinearGrads {
  const void* d_out;          // bf16 [rows, outs], contiguous
  void* dx;                   // bf16 [rows, cols], or nullptr
  void *dweight, *dbias;      // of the norm, or nullptr
  int dweight_type, dbias_type;
  void* dw;                   // [outs, cols], or nullptr
  int dw_type;
};
int64_t norm_linear_bwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs);
int norm_linear_bwd(const NormCall& norm, const void* w, int64_t outs, const NormLinearGrads& g, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream);

}  // namespace tpf

// The normalised projection: out = y W^T with y = layer_norm(x), bf16, no bias.
//
//   forward    y = w xh + b (bf16), out = y W^T
//   backward   dy = d_out W (bf16), the layer norm's backward on it, dW = d_out^T y~ with y~ from what was kept of x
//
// dy of wide rows goes through memory in bf16, as it does behind any bf16 Linear (narrow rows never leave the SM and stay in
// fp32).  In fp32 d_x and the norm's gradients would be off by their own rounding only, 0.0017 of their norm in the place of
// 0.0024, for twice the traffic between the two kernels: the whole backward of 4099 rows, 1024 -> 4096, takes 100 us in the
// place of 94, 16384 of 1024 -> 1024 131 / 115, 100000 of 256 -> 1024 174 / 156, 60000 of 512 -> 512 152 / 121, 300000 of 136 ->
// 512 389 / 295 (cold L2).
#include "tpf_norm_linear.cuh"

namespace tpf {

int bmm_bf16(const void* A, int64_t lda, int64_t bsa, int a_mn, const void* B, int64_t ldb, int64_t bsb, int b_mn,
             void* D, int64_t ldd, int64_t bsd, int out_f32, int64_t M, int64_t N, int64_t K, int64_t batch,
             int64_t k_per_split, int swizzle_bytes, cudaStream_t stream);

namespace {

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// What both passes ask of their arguments.  x (or its codes) is read eight elements at a time.
int check_linear(const NormCall& c, const void* w, int64_t outs, const char* who) {
  TPF_REQUIRE(c.type == kRowBF16, TPF_ERR_UNSUPPORTED, "%s: bf16 only", who);
  TPF_REQUIRE(c.cols >= 8 && c.cols <= kMaxNormCols && c.cols % 8 == 0 && outs >= 8 && outs % 8 == 0, TPF_ERR_UNSUPPORTED,
              "%s: columns and outputs must be multiples of 8, columns at most %lld", who, (long long)kMaxNormCols);
  TPF_REQUIRE(c.rows >= 0 && c.rows < (1ll << 31) - 256 && outs <= (1ll << 30), TPF_ERR_UNSUPPORTED,
              "%s: extent too large", who);
  TPF_REQUIRE(w != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  TPF_REQUIRE_ALIGNED16(w, who, "weight");
  TPF_REQUIRE(rows_vec_ok(c.x, c.x_pitch, c.type), TPF_ERR_INVALID_ARGUMENT, "%s: x must have 16-byte aligned rows", who);
  TPF_REQUIRE(c.x == nullptr || c.x_pitch >= c.cols, TPF_ERR_INVALID_ARGUMENT, "%s: rows overlap", who);
  TPF_REQUIRE_ALIGNED16(c.codes, who, "codes");
  return TPF_OK;
}

}  // namespace

int64_t norm_linear_fwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  return norm_linear_few(rows) || norm_linear_narrow(cols, outs) ? 0 : up256(rows * cols * 2);
}

int norm_linear_fwd(const NormCall& norm, const void* w, int64_t outs, void* out, float eps, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream) {
  const char* who = "norm_linear_fwd";
  if (int rc = check_linear(norm, w, outs, who)) return rc;
  if (norm.rows == 0) return TPF_OK;
  TPF_REQUIRE(out != nullptr && norm.x != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  TPF_REQUIRE_ALIGNED16(out, who, "out");
  NormArgs a;
  if (int rc = make_norm_args(&a, norm, who)) return rc;
  TPF_REQUIRE(norm.codes == nullptr || norm.mean != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: codes without mean and rstd", who);
  if (norm_linear_few(norm.rows)) return norm_linear_few_fwd(a, w, outs, out, eps, stream);
  if (norm_linear_narrow(norm.cols, outs)) return norm_linear_narrow_fwd(a, w, outs, out, eps, stream);
  const int64_t need = norm_linear_fwd_workspace_bytes(norm.rows, norm.cols, outs);
  TPF_REQUIRE(workspace != nullptr && workspace_bytes >= need, TPF_ERR_WORKSPACE,
              "%s: workspace of %lld bytes required, %lld given", who, (long long)need, (long long)workspace_bytes);
  TPF_REQUIRE_ALIGNED16(workspace, who, "workspace");
  if (int rc = layer_norm_fwd(norm, workspace, eps, stream)) return rc;
  return bmm_bf16(workspace, norm.cols, 0, 0, w, norm.cols, 0, 0, out, outs, 0, 0, norm.rows, outs, norm.cols, 1, 0, 128,
                  stream);
}

int64_t norm_linear_bwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  if (norm_linear_narrow(cols, outs)) return norm_linear_narrow_bwd_workspace_bytes(rows, cols, outs);
  return up256(rows * cols * 2) + up256(layer_norm_bwd_workspace_bytes(rows, cols)) +
         up256(norm_linear_dw_workspace_bytes(rows, cols, outs));
}

int norm_linear_bwd(const NormCall& norm, const void* w, int64_t outs, const NormLinearGrads& g, void* workspace,
                    int64_t workspace_bytes, cudaStream_t stream) {
  const char* who = "norm_linear_bwd";
  if (int rc = check_linear(norm, w, outs, who)) return rc;
  TPF_REQUIRE((norm.x != nullptr || norm.codes != nullptr || norm.rows == 0) && (g.d_out != nullptr || norm.rows == 0) &&
                  (norm.mean != nullptr || norm.rows == 0),
              TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  TPF_REQUIRE_ALIGNED16(g.d_out, who, "d_out");
  TPF_REQUIRE_ALIGNED16(g.dx, who, "dx");
  TPF_REQUIRE_ALIGNED16(g.dw, who, "d_weight");
  TPF_REQUIRE(g.dw == nullptr || row_type_ok(g.dw_type), TPF_ERR_INVALID_ARGUMENT, "%s: unknown parameter type", who);
  const int64_t need = norm_linear_bwd_workspace_bytes(norm.rows, norm.cols, outs);
  TPF_REQUIRE(norm.rows == 0 || (workspace != nullptr && workspace_bytes >= need), TPF_ERR_WORKSPACE,
              "%s: workspace of %lld bytes required, %lld given", who, (long long)need, (long long)workspace_bytes);
  TPF_REQUIRE_ALIGNED16(workspace, who, "workspace");
  const int64_t R = norm.rows, C = norm.cols;
  char* base = static_cast<char*>(workspace);
  NormArgs a;
  if (int rc = make_norm_args(&a, norm, who)) return rc;
  TPF_REQUIRE((g.dweight == nullptr || row_type_ok(g.dweight_type)) && (g.dbias == nullptr || row_type_ok(g.dbias_type)),
              TPF_ERR_INVALID_ARGUMENT, "%s: unknown parameter type", who);
  if (R > 0 && norm_linear_narrow(C, outs)) return norm_linear_narrow_bwd(a, w, outs, g, workspace, stream);
  const int64_t ln_bytes = layer_norm_bwd_workspace_bytes(R, C);
  void* dy = base;
  void* ln_ws = base + up256(R * C * 2);
  void* dw_ws = base + up256(R * C * 2) + up256(ln_bytes);
  if (g.dx != nullptr || g.dweight != nullptr || g.dbias != nullptr) {
    if (R > 0)
      if (int rc = bmm_bf16(g.d_out, outs, 0, 0, w, C, 0, 1, dy, C, 0, 0, R, C, outs, 1, 0, 128, stream)) return rc;
    const NormGrads n{dy, g.dx, g.dweight, g.dbias, g.dweight_type, g.dbias_type};
    if (int rc = layer_norm_bwd(norm, n, ln_ws, ln_bytes, stream)) return rc;
  }
  if (g.dw == nullptr) return TPF_OK;
  if (R == 0) {
    TPF_CUDA_OK(cudaMemsetAsync(g.dw, 0, outs * C * row_type_size(g.dw_type), stream));
    return TPF_OK;
  }
  return norm_linear_dw(a, g.d_out, outs, g.dw, g.dw_type, dw_ws, stream);
}

}  // namespace tpf

// extern "C" surface of libtpf_b200.so (declarations: include/tpf_b200.h).
#include "../../include/tpf_b200.h"
#include "tpf_host.cuh"
#include "tpf_dropout.h"
#include "tpf_internal.h"
#include "tpf_rotary.h"
#include "tpf_rows.h"
#include "tpf_window.h"

namespace tpf {

char* last_error_buffer() {
  static thread_local char buf[512] = "";
  return buf;
}

int bmm_status_fetch_and_clear(int* out);
int bmm_bf16(const void* A, int64_t lda, int64_t bsa, int a_mn, const void* B, int64_t ldb, int64_t bsb, int b_mn,
             void* D, int64_t ldd, int64_t bsd, int out_f32, int64_t M, int64_t N, int64_t K, int64_t batch,
             int64_t k_per_split, int swizzle_bytes, cudaStream_t stream);

int attn_fwd_status_fetch_and_clear(int* out);
int attn_fwd(const void* q, const void* k, const void* v, const int64_t* q_strides, const int64_t* k_strides,
             const int64_t* v_strides, const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch,
             int64_t bias_batch, void* out, float* lse, int64_t B, int64_t O, int64_t H, int64_t N, int64_t D,
             float scale, cudaStream_t stream);

int attn_bwd_status_fetch_and_clear(int* out);
int64_t attn_bwd_workspace_bytes(int64_t B, int64_t O, int64_t H, int64_t N, int64_t D);
int64_t attn_dbias_workspace_bytes(int64_t B, int64_t O, int64_t H, int64_t N, int64_t G);
int attn_bwd_dqkv(const void* q, const void* k, const void* v, const void* d_out, const int64_t* q_strides,
                  const int64_t* k_strides, const int64_t* v_strides, const void* out, const float* lse,
                  const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch, int64_t bias_batch,
                  void* dq, void* dk, void* dv, float* delta, void* workspace, int64_t workspace_bytes, int64_t B,
                  int64_t O, int64_t H, int64_t N, int64_t D, float scale, int stages, cudaStream_t stream);
int attn_bwd_dbias(const void* q, const void* k, const void* v, const void* d_out, const int64_t* q_strides,
                   const int64_t* k_strides, const int64_t* v_strides, const float* lse, const float* delta,
                   const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch, int64_t bias_batch,
                   float* dbias, void* workspace, int64_t workspace_bytes, int64_t B, int64_t O, int64_t H, int64_t N,
                   int64_t D, float scale, cudaStream_t stream, double dbias_limit);

int64_t attn_bwd_static_scratch_capacity();
int attn_bwd_static_scratch(const void* q, const void* k, const void* v, const void* d_out, const int64_t* q_strides,
                            const int64_t* k_strides, const int64_t* v_strides, const void* out, const float* lse,
                            const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch,
                            int64_t bias_batch, void* dq, void* dk, void* dv, float* dbias, float* delta, int64_t B,
                            int64_t O, int64_t H, int64_t N, int64_t D, float scale, cudaStream_t stream);
int pair_attn_status_fetch_and_clear(int* out);
int selftest_status_fetch_and_clear(int* out);
int norm_linear_dw_status_fetch_and_clear(int* out);
int norm_linear_fwd_status_fetch_and_clear(int* out);
int norm_linear_bwd_status_fetch_and_clear(int* out);
int window_fwd_status_fetch_and_clear(int* out);
int window_bwd_status_fetch_and_clear(int* out);
int selftest_bounded_wait(unsigned int* report, cudaStream_t stream);

int trimul_status_fetch_and_clear(int* out);
int trimul_fwd_status_fetch_and_clear(int* out);
int64_t trimul_fwd_workspace_bytes(int64_t B, int64_t N, int64_t C);
int64_t trimul_bwd_workspace_bytes(int64_t B, int64_t N, int64_t C);
int trimul_fwd(const void* z, const float* mask, const float* p_in, const float* g_in, const float* p_out,
               const float* g_out, const float* gin, const float* bin, const float* gout, const float* bout,
               int incoming, int64_t B, int64_t N, int64_t C, void* out, void* zln, float* mean_in, float* rstd_in,
               void* a_cm, void* b_cm, void* gate, void* x_cm, void* xln, float* mean_out, float* rstd_out,
               void* workspace, int64_t workspace_bytes, int64_t NN, int stages, cudaStream_t stream);
int trimul_bwd(const void* d_out, const void* z, const float* mask, const float* p_in, const float* g_in,
               const float* p_out, const float* g_out, const float* gin, const float* gout, int incoming, int64_t B,
               int64_t N, int64_t C, const void* out, const void* zln, const float* mean_in, const float* rstd_in,
               const void* a_cm, const void* b_cm, const void* gate, const void* x_cm, const void* xln,
               const float* mean_out, const float* rstd_out, void* d_z, float* d_p_in, float* d_g_in, float* d_p_out,
               float* d_g_out, float* d_gin, float* d_bin, float* d_gout, float* d_bout, void* workspace,
               int64_t workspace_bytes, int64_t NN, int stages, void* dx_io, void* da_io, void* db_io,
               cudaStream_t stream);

}  // namespace tpf

extern "C" {

const char* tpf_version(void) { return "tpf_b200 0.1 sm_100a"; }

const char* tpf_last_error_string(void) { return tpf::last_error_buffer(); }

int64_t tpf_launch_count(void) { return tpf::launch_counter().load(); }

int tpf_device_status(int* status) {
  TPF_REQUIRE(status != nullptr, TPF_ERR_INVALID_ARGUMENT, "tpf_device_status: status is NULL");
  int total = 0, v = 0;
  int rc = tpf::bmm_status_fetch_and_clear(&v);
  if (rc) return rc;
  total |= v;
  if ((rc = tpf::attn_fwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::attn_bwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::trimul_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::trimul_fwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::pair_attn_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::norm_linear_dw_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::norm_linear_fwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::norm_linear_bwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::window_fwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::window_bwd_status_fetch_and_clear(&v))) return rc;
  total |= v;
  if ((rc = tpf::selftest_status_fetch_and_clear(&v))) return rc;
  total |= v;
  *status = total;
  return TPF_OK;
}

int tpf_selftest_bounded_wait(unsigned int* report, void* stream) {
  return tpf::selftest_bounded_wait(report, static_cast<cudaStream_t>(stream));
}

int tpf_bmm_bf16(const void* A, int64_t lda, int64_t batch_stride_a, int a_mn, const void* B, int64_t ldb,
                 int64_t batch_stride_b, int b_mn, void* D, int64_t ldd, int64_t batch_stride_d, int out_f32,
                 int64_t M, int64_t N, int64_t K, int64_t batch, int64_t k_per_split, int swizzle_bytes,
                 void* stream) {
  return tpf::bmm_bf16(A, lda, batch_stride_a, a_mn, B, ldb, batch_stride_b, b_mn, D, ldd, batch_stride_d, out_f32,
                       M, N, K, batch, k_per_split, swizzle_bytes, static_cast<cudaStream_t>(stream));
}

int tpf_attn_fwd(const void* q, const void* k, const void* v, const int64_t* q_strides, const int64_t* k_strides,
                 const int64_t* v_strides, const float* mask, int64_t mask_pitch, const void* bias,
                 int64_t bias_pitch, int64_t bias_batch, void* out, float* lse, int64_t B, int64_t O, int64_t H,
                 int64_t N, int64_t D, float scale, void* stream) {
  TPF_REQUIRE(q_strides && k_strides && v_strides, TPF_ERR_INVALID_ARGUMENT, "tpf_attn_fwd: stride arrays are NULL");
  return tpf::attn_fwd(q, k, v, q_strides, k_strides, v_strides, mask, mask_pitch, bias, bias_pitch, bias_batch, out,
                       lse, B, O, H, N, D, scale, static_cast<cudaStream_t>(stream));
}

static int64_t round_up_256(int64_t x) { return (x + 255) / 256 * 256; }

int64_t tpf_attn_bwd_workspace_bytes(int64_t B, int64_t O, int64_t H, int64_t N, int64_t D, int64_t bias_batch) {
  if (B <= 0 || O <= 0 || H <= 0 || N <= 0 || (bias_batch != 1 && bias_batch != B)) return 0;
  return round_up_256(tpf::attn_bwd_workspace_bytes(B, O, H, N, D)) +
         round_up_256(tpf::attn_dbias_workspace_bytes(B, O, H, N, bias_batch));
}

int tpf_attn_bwd(const void* q, const void* k, const void* v, const void* d_out, const int64_t* q_strides,
                 const int64_t* k_strides, const int64_t* v_strides, const void* out, const float* lse,
                 const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch, int64_t bias_batch,
                 void* dq, void* dk, void* dv, float* dbias, float* delta, void* workspace, int64_t workspace_bytes,
                 int64_t B, int64_t O, int64_t H, int64_t N, int64_t D, float scale, void* stream) {
  return tpf_attn_bwd_stages(q, k, v, d_out, q_strides, k_strides, v_strides, out, lse, mask, mask_pitch, bias,
                             bias_pitch, bias_batch, dq, dk, dv, dbias, delta, workspace, workspace_bytes, B, O, H, N,
                             D, scale, TPF_ATTN_BWD_STAGE_ALL, stream);
}

int tpf_attn_bwd_stages(const void* q, const void* k, const void* v, const void* d_out, const int64_t* q_strides,
                        const int64_t* k_strides, const int64_t* v_strides, const void* out, const float* lse,
                        const float* mask, int64_t mask_pitch, const void* bias, int64_t bias_pitch,
                        int64_t bias_batch, void* dq, void* dk, void* dv, float* dbias, float* delta, void* workspace,
                        int64_t workspace_bytes, int64_t B, int64_t O, int64_t H, int64_t N, int64_t D, float scale,
                        int stages, void* stream) {
  TPF_REQUIRE(stages > 0 && stages <= TPF_ATTN_BWD_STAGE_ALL, TPF_ERR_INVALID_ARGUMENT,
              "tpf_attn_bwd_stages: stages must be a non-empty mask of TPF_ATTN_BWD_STAGE_*");
  TPF_REQUIRE(q_strides && k_strides && v_strides, TPF_ERR_INVALID_ARGUMENT, "tpf_attn_bwd: stride arrays are NULL");
  TPF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, TPF_ERR_INVALID_ARGUMENT,
              "tpf_attn_bwd: workspace must be 256-byte aligned");
  TPF_REQUIRE(B > 0 && O > 0 && H > 0 && N > 0 && (bias_batch == 1 || bias_batch == B), TPF_ERR_INVALID_ARGUMENT,
              "tpf_attn_bwd: bad extents");
  const int64_t ws_a = round_up_256(tpf::attn_bwd_workspace_bytes(B, O, H, N, D));
  const int64_t ws_b = round_up_256(tpf::attn_dbias_workspace_bytes(B, O, H, N, bias_batch));
  TPF_REQUIRE(workspace_bytes >= ws_a + ws_b && (ws_a + ws_b == 0 || workspace), TPF_ERR_WORKSPACE,
              "tpf_attn_bwd: workspace of %lld bytes required, %lld given", (long long)(ws_a + ws_b),
              (long long)workspace_bytes);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = TPF_OK;
  if (stages & (TPF_ATTN_BWD_STAGE_DELTA | TPF_ATTN_BWD_STAGE_DQKV))
    rc = tpf::attn_bwd_dqkv(q, k, v, d_out, q_strides, k_strides, v_strides, out, lse, mask, mask_pitch, bias,
                            bias_pitch, bias_batch, dq, dk, dv, delta, workspace, ws_a, B, O, H, N, D, scale,
                            stages & 3, st);
  if (rc) return rc;
  if (!(stages & TPF_ATTN_BWD_STAGE_DBIAS)) return TPF_OK;
  return tpf::attn_bwd_dbias(q, k, v, d_out, q_strides, k_strides, v_strides, lse, delta, mask, mask_pitch, bias,
                             bias_pitch, bias_batch, dbias, static_cast<char*>(workspace) + ws_a, ws_b, B, O, H, N, D,
                             scale, st, tpf::kNoByteLimit);
}

int64_t tpf_attn_bwd_static_scratch_capacity(void) { return tpf::attn_bwd_static_scratch_capacity(); }

int tpf_attn_bwd_static_scratch(const void* q, const void* k, const void* v, const void* d_out,
                                const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                const void* out, const float* lse, const float* mask, int64_t mask_pitch,
                                const void* bias, int64_t bias_pitch, int64_t bias_batch, void* dq, void* dk, void* dv,
                                float* dbias, float* delta, int64_t B, int64_t O, int64_t H, int64_t N, int64_t D,
                                float scale, void* stream) {
  TPF_REQUIRE(q_strides && k_strides && v_strides, TPF_ERR_INVALID_ARGUMENT,
              "tpf_attn_bwd_static_scratch: stride arrays are NULL");
  return tpf::attn_bwd_static_scratch(q, k, v, d_out, q_strides, k_strides, v_strides, out, lse, mask, mask_pitch,
                                      bias, bias_pitch, bias_batch, dq, dk, dv, dbias, delta, B, O, H, N, D, scale,
                                      static_cast<cudaStream_t>(stream));
}

static bool trimul_shape_ok(int64_t B, int64_t N, int64_t C) {
  return B > 0 && N > 0 && (C == 32 || C == 64 || C == 96 || C == 128);
}

int64_t tpf_trimul_fwd_workspace_bytes(int64_t B, int64_t N, int64_t C) {
  return trimul_shape_ok(B, N, C) ? tpf::trimul_fwd_workspace_bytes(B, N, C) : 0;
}

int64_t tpf_trimul_bwd_workspace_bytes(int64_t B, int64_t N, int64_t C) {
  return trimul_shape_ok(B, N, C) ? tpf::trimul_bwd_workspace_bytes(B, N * N, C) : 0;
}

int64_t tpf_trimul_bwd_stages_workspace_bytes(int64_t B, int64_t rows_per_batch, int64_t C) {
  return (trimul_shape_ok(B, 8, C) && rows_per_batch > 0) ? tpf::trimul_bwd_workspace_bytes(B, rows_per_batch, C) : 0;
}

int tpf_trimul_fwd_stages(const void* z, const float* mask, const float* p_in, const float* g_in, const float* p_out,
                          const float* g_out, const float* norm_in_w, const float* norm_in_b, const float* norm_out_w,
                          const float* norm_out_b, int direction, int64_t B, int64_t N, int64_t C, void* out, void* zln,
                          float* mean_in, float* rstd_in, void* a_cm, void* b_cm, void* gate, void* x_cm, void* xln,
                          float* mean_out, float* rstd_out, void* workspace, int64_t workspace_bytes,
                          int64_t rows_per_batch, int stages, void* stream) {
  TPF_REQUIRE(direction == 0 || direction == 1, TPF_ERR_INVALID_ARGUMENT,
              "tpf_trimul_fwd: direction must be 0 (outgoing) or 1 (incoming)");
  return tpf::trimul_fwd(z, mask, p_in, g_in, p_out, g_out, norm_in_w, norm_in_b, norm_out_w, norm_out_b, direction, B,
                         N, C, out, zln, mean_in, rstd_in, a_cm, b_cm, gate, x_cm, xln, mean_out, rstd_out, workspace,
                         workspace_bytes, rows_per_batch, stages, static_cast<cudaStream_t>(stream));
}

int tpf_trimul_fwd(const void* z, const float* mask, const float* p_in, const float* g_in, const float* p_out,
                   const float* g_out, const float* norm_in_w, const float* norm_in_b, const float* norm_out_w,
                   const float* norm_out_b, int direction, int64_t B, int64_t N, int64_t C, void* out, void* zln,
                   float* mean_in, float* rstd_in, void* a_cm, void* b_cm, void* gate, void* x_cm, void* xln,
                   float* mean_out, float* rstd_out, void* workspace, int64_t workspace_bytes, void* stream) {
  return tpf_trimul_fwd_stages(z, mask, p_in, g_in, p_out, g_out, norm_in_w, norm_in_b, norm_out_w, norm_out_b,
                               direction, B, N, C, out, zln, mean_in, rstd_in, a_cm, b_cm, gate, x_cm, xln, mean_out,
                               rstd_out, workspace, workspace_bytes, 0, 7, stream);
}

int tpf_trimul_bwd_stages(const void* d_out, const void* z, const float* mask, const float* p_in, const float* g_in,
                          const float* p_out, const float* g_out, const float* norm_in_w, const float* norm_out_w,
                          int direction, int64_t B, int64_t N, int64_t C, const void* out, const void* zln,
                          const float* mean_in, const float* rstd_in, const void* a_cm, const void* b_cm,
                          const void* gate, const void* x_cm, const void* xln, const float* mean_out,
                          const float* rstd_out, void* d_z, float* d_p_in, float* d_g_in, float* d_p_out,
                          float* d_g_out, float* d_norm_in_w, float* d_norm_in_b, float* d_norm_out_w,
                          float* d_norm_out_b, void* workspace, int64_t workspace_bytes, int64_t rows_per_batch,
                          int stages, void* dx_cm, void* da_cm, void* db_cm, void* stream) {
  TPF_REQUIRE(direction == 0 || direction == 1, TPF_ERR_INVALID_ARGUMENT,
              "tpf_trimul_bwd: direction must be 0 (outgoing) or 1 (incoming)");
  return tpf::trimul_bwd(d_out, z, mask, p_in, g_in, p_out, g_out, norm_in_w, norm_out_w, direction, B, N, C, out, zln,
                         mean_in, rstd_in, a_cm, b_cm, gate, x_cm, xln, mean_out, rstd_out, d_z, d_p_in, d_g_in,
                         d_p_out, d_g_out, d_norm_in_w, d_norm_in_b, d_norm_out_w, d_norm_out_b, workspace,
                         workspace_bytes, rows_per_batch, stages, dx_cm, da_cm, db_cm,
                         static_cast<cudaStream_t>(stream));
}

int tpf_trimul_bwd(const void* d_out, const void* z, const float* mask, const float* p_in, const float* g_in,
                   const float* p_out, const float* g_out, const float* norm_in_w, const float* norm_out_w,
                   int direction, int64_t B, int64_t N, int64_t C, const void* out, const void* zln,
                   const float* mean_in, const float* rstd_in, const void* a_cm, const void* b_cm, const void* gate,
                   const void* x_cm, const void* xln, const float* mean_out, const float* rstd_out, void* d_z,
                   float* d_p_in, float* d_g_in, float* d_p_out, float* d_g_out, float* d_norm_in_w,
                   float* d_norm_in_b, float* d_norm_out_w, float* d_norm_out_b, void* workspace,
                   int64_t workspace_bytes, void* stream) {
  return tpf_trimul_bwd_stages(d_out, z, mask, p_in, g_in, p_out, g_out, norm_in_w, norm_out_w, direction, B, N, C, out,
                               zln, mean_in, rstd_in, a_cm, b_cm, gate, x_cm, xln, mean_out, rstd_out, d_z, d_p_in,
                               d_g_in, d_p_out, d_g_out, d_norm_in_w, d_norm_in_b, d_norm_out_w, d_norm_out_b,
                               workspace, workspace_bytes, 0, 7, nullptr, nullptr, nullptr, stream);
}

int tpf_layer_norm_fwd(const void* x, int64_t x_pitch, int type, const void* weight, int weight_type, const void* bias,
                       int bias_type, void* y, void* codes, float* scales, float* mean, float* rstd, int64_t rows,
                       int64_t cols, float eps, void* stream) {
  const tpf::NormCall c{rows, cols, type, x, x_pitch, codes, scales, mean, rstd, weight, bias, weight_type, bias_type};
  return tpf::layer_norm_fwd(c, y, eps, static_cast<cudaStream_t>(stream));
}

int64_t tpf_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  return rows > 0 && cols > 0 ? tpf::layer_norm_bwd_workspace_bytes(rows, cols) : 0;
}

int tpf_layer_norm_bwd(const void* dy, const void* x, int64_t x_pitch, const void* codes, const float* scales, int type,
                       const float* mean, const float* rstd, const void* weight, int weight_type, void* dx, void* dweight,
                       int dweight_type, void* dbias, int dbias_type, void* workspace, int64_t workspace_bytes,
                       int64_t rows, int64_t cols, void* stream) {
  const tpf::NormCall c{rows, cols, type, x, x_pitch, const_cast<void*>(codes), const_cast<float*>(scales),
                        const_cast<float*>(mean), const_cast<float*>(rstd), weight, nullptr, weight_type, 0};
  const tpf::NormGrads g{dy, dx, dweight, dbias, dweight_type, dbias_type};
  return tpf::layer_norm_bwd(c, g, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int tpf_int8_pack(const void* x, int64_t x_pitch, int type, void* codes, float* scales, int64_t rows, int64_t cols,
                  void* stream) {
  return tpf::int8_pack(x, x_pitch, type, codes, scales, rows, cols, static_cast<cudaStream_t>(stream));
}

int tpf_int8_unpack(const void* codes, const float* scales, int type, void* x, int64_t rows, int64_t cols, void* stream) {
  return tpf::int8_unpack(codes, scales, type, x, rows, cols, static_cast<cudaStream_t>(stream));
}

static bool norm_linear_shape_ok(int64_t rows, int64_t cols, int64_t outs) { return rows > 0 && cols > 0 && outs > 0; }

int64_t tpf_norm_linear_fwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  return norm_linear_shape_ok(rows, cols, outs) ? tpf::norm_linear_fwd_workspace_bytes(rows, cols, outs) : 0;
}

int64_t tpf_norm_linear_bwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  return norm_linear_shape_ok(rows, cols, outs) ? tpf::norm_linear_bwd_workspace_bytes(rows, cols, outs) : 0;
}

int tpf_norm_linear_fwd(const void* x, int64_t x_pitch, const void* norm_weight, int norm_weight_type,
                        const void* norm_bias, int norm_bias_type, const void* weight, void* out, void* codes,
                        float* scales, float* mean, float* rstd, void* workspace, int64_t workspace_bytes, int64_t rows,
                        int64_t cols, int64_t outs, float eps, void* stream) {
  const tpf::NormCall c{rows, cols, TPF_BF16, x, x_pitch, codes, scales, mean, rstd, norm_weight, norm_bias,
                        norm_weight_type, norm_bias_type};
  return tpf::norm_linear_fwd(c, weight, outs, out, eps, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int tpf_norm_linear_bwd(const void* d_out, const void* x, int64_t x_pitch, const void* codes, const float* scales,
                        const float* mean, const float* rstd, const void* norm_weight, int norm_weight_type,
                        const void* norm_bias, int norm_bias_type, const void* weight, void* dx, void* d_norm_weight,
                        int d_norm_weight_type, void* d_norm_bias, int d_norm_bias_type, void* d_weight,
                        int d_weight_type, void* workspace, int64_t workspace_bytes, int64_t rows, int64_t cols,
                        int64_t outs, void* stream) {
  const tpf::NormCall c{rows, cols, TPF_BF16, x, x_pitch, const_cast<void*>(codes), const_cast<float*>(scales),
                        const_cast<float*>(mean), const_cast<float*>(rstd), norm_weight, norm_bias, norm_weight_type,
                        norm_bias_type};
  const tpf::NormLinearGrads g{d_out, dx, d_norm_weight, d_norm_bias, d_norm_weight_type, d_norm_bias_type, d_weight,
                               d_weight_type};
  return tpf::norm_linear_bwd(c, weight, outs, g, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int tpf_dropout(const void* x, const int64_t* x_strides, const void* residual, const int64_t* residual_strides, void* out,
                const int64_t* out_strides, const int64_t* sizes, int type, int shared, int threshold, const int64_t* seed_offset,
                int64_t seed, int64_t offset, void* stream) {
  TPF_REQUIRE(x_strides && out_strides && sizes && (residual == nullptr || residual_strides), TPF_ERR_INVALID_ARGUMENT,
              "dropout: null pointer");
  tpf::DropoutCall c = {};
  c.x = x, c.residual = residual, c.out = out;
  for (int i = 0; i < 3; ++i) {
    c.x_strides[i] = x_strides[i];
    c.residual_strides[i] = residual != nullptr ? residual_strides[i] : 0;
    c.out_strides[i] = out_strides[i];
  }
  for (int i = 0; i < 4; ++i) c.sizes[i] = sizes[i];
  c.type = type, c.shared = shared, c.threshold = threshold;
  c.seed_ptr = seed_offset, c.seed = seed, c.offset = offset;
  return tpf::dropout(c, static_cast<cudaStream_t>(stream));
}

static int rotary_tensor(tpf::RotaryTensor* t, const void* x, const int64_t* strides, int64_t heads, const void* weight,
                         int weight_type, const void* dy, void* out, void* dweight) {
  TPF_REQUIRE(heads <= 0 || x == nullptr || strides != nullptr, TPF_ERR_INVALID_ARGUMENT, "rotary: null pointer");
  *t = {x, {0, 0, 0}, heads, weight, weight_type, dy, out, dweight};
  for (int i = 0; i < 3 && strides != nullptr; ++i) t->strides[i] = strides[i];
  return TPF_OK;
}

int tpf_rotary_fwd(const void* q, const int64_t* q_strides, int64_t q_heads, const void* q_weight, int q_weight_type, void* q_out,
                   const void* k, const int64_t* k_strides, int64_t k_heads, const void* k_weight, int k_weight_type, void* k_out,
                   int type, int64_t batch, int64_t tokens, int64_t dim, int64_t rot, const int64_t* turns, float magnitude,
                   const int64_t* positions, int64_t first, int half, int norm, float eps, void* stream) {
  tpf::RotaryCall c = {};
  if (int rc = rotary_tensor(&c.t[0], q, q_strides, q_heads, q_weight, q_weight_type, nullptr, q_out, nullptr)) return rc;
  if (int rc = rotary_tensor(&c.t[1], k, k_strides, k_heads, k_weight, k_weight_type, nullptr, k_out, nullptr)) return rc;
  c.type = type, c.batch = batch, c.tokens = tokens, c.dim = dim, c.rot = rot, c.turns = turns, c.magnitude = magnitude;
  c.positions = positions, c.first = first, c.half = half, c.norm = norm, c.eps = eps;
  return tpf::rotary_fwd(c, static_cast<cudaStream_t>(stream));
}

int64_t tpf_rotary_bwd_workspace_bytes(int64_t dim) { return tpf::rotary_bwd_workspace_bytes(dim); }

int tpf_rotary_bwd(const void* dq_out, const void* q, const int64_t* q_strides, int64_t q_heads, const void* q_weight,
                   int q_weight_type, void* dq, void* d_q_weight, const void* dk_out, const void* k, const int64_t* k_strides,
                   int64_t k_heads, const void* k_weight, int k_weight_type, void* dk, void* d_k_weight, int type, int64_t batch,
                   int64_t tokens, int64_t dim, int64_t rot, const int64_t* turns, float magnitude, const int64_t* positions,
                   int64_t first, int half, int norm, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  tpf::RotaryCall c = {};
  if (int rc = rotary_tensor(&c.t[0], q, q_strides, q_heads, q_weight, q_weight_type, dq_out, dq, d_q_weight)) return rc;
  if (int rc = rotary_tensor(&c.t[1], k, k_strides, k_heads, k_weight, k_weight_type, dk_out, dk, d_k_weight)) return rc;
  c.type = type, c.batch = batch, c.tokens = tokens, c.dim = dim, c.rot = rot, c.turns = turns, c.magnitude = magnitude;
  c.positions = positions, c.first = first, c.half = half, c.norm = norm, c.eps = eps;
  return tpf::rotary_bwd(c, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

static tpf::WindowCall window_call(int type, int64_t B, int64_t N, int64_t M, int64_t H, int64_t HK, int64_t D, float scale,
                                   int64_t left, int64_t right, int64_t sinks, const int* offsets, int64_t offset,
                                   const int* lengths) {
  auto reach = [](int64_t n) { return n < 0 ? tpf::kWindowUnlimited : n < tpf::kWindowMost ? (int)n : -1; };  // -1 is refused
  tpf::WindowCall c = {};
  c.B = B, c.N = N, c.M = M, c.H = H, c.HK = HK, c.D = D, c.type = type, c.scale = scale;
  c.left = reach(left), c.right = reach(right);
  c.sinks = sinks < 0 || sinks > tpf::kMostSinks ? -1 : (int)sinks;
  c.offsets = offsets, c.offset = offset, c.lengths = lengths;
  return c;
}

static int window_operands(tpf::WindowCall* c, const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v,
                           const int64_t* vs) {
  TPF_REQUIRE(qs && ks && vs, TPF_ERR_INVALID_ARGUMENT, "window_attn: null pointer");
  c->q = q, c->k = k, c->v = v;
  for (int i = 0; i < 3; ++i) c->qs[i] = qs[i], c->ks[i] = ks[i], c->vs[i] = vs[i];
  return TPF_OK;
}

int tpf_window_attn_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                        const int64_t* v_strides, void* out, float* lse, int type, int64_t B, int64_t N, int64_t M, int64_t H,
                        int64_t HK, int64_t D, float scale, int64_t left, int64_t right, int64_t sinks, const int* offsets,
                        int64_t offset, const int* lengths, void* stream) {
  tpf::WindowCall c = window_call(type, B, N, M, H, HK, D, scale, left, right, sinks, offsets, offset, lengths);
  if (int rc = window_operands(&c, q, q_strides, k, k_strides, v, v_strides)) return rc;
  c.out = out, c.lse = lse;
  return tpf::window_attn_fwd(c, static_cast<cudaStream_t>(stream));
}

int64_t tpf_window_attn_bwd_workspace_bytes(int64_t B, int64_t N, int64_t M, int64_t H, int64_t HK, int64_t D, int64_t left,
                                            int64_t right, int64_t sinks) {
  const tpf::WindowCall c = window_call(TPF_BF16, B, N, M, H, HK, D, 1.f, left, right, sinks, nullptr, 0, nullptr);
  return c.left >= 0 && c.right >= 0 && c.sinks >= 0 ? tpf::window_attn_bwd_workspace_bytes(c) : 0;
}

int tpf_window_attn_bwd(const void* d_out, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                        const void* v, const int64_t* v_strides, const void* out, const float* lse, void* dq, void* dk, void* dv,
                        int type, int64_t B, int64_t N, int64_t M, int64_t H, int64_t HK, int64_t D, float scale, int64_t left,
                        int64_t right, int64_t sinks, const int* offsets, int64_t offset, const int* lengths, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  tpf::WindowCall c = window_call(type, B, N, M, H, HK, D, scale, left, right, sinks, offsets, offset, lengths);
  if (int rc = window_operands(&c, q, q_strides, k, k_strides, v, v_strides)) return rc;
  c.out = const_cast<void*>(out), c.lse = const_cast<float*>(lse);
  c.d_out = d_out, c.dq = dq, c.dk = dk, c.dv = dv;
  return tpf::window_attn_bwd(c, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

// Window attention: checks and the choice of the kernel.
#include "tpf_window.h"

#include "tpf_window_kernels.h"

namespace tpf {

namespace {

int make_params(WindowParams* p, const WindowCall& c, const char* who) {
  TPF_REQUIRE(c.type == kRowBF16 || c.type == kRowF16, TPF_ERR_INVALID_ARGUMENT, "%s: the type must be BF16 or FP16", who);
  TPF_REQUIRE(c.B >= 0 && c.N >= 0 && c.M >= 0 && c.H >= 1 && c.HK >= 1, TPF_ERR_INVALID_ARGUMENT,
              "%s: extents must not be negative", who);
  TPF_REQUIRE(c.H % c.HK == 0, TPF_ERR_INVALID_ARGUMENT, "%s: the heads must be a multiple of the key heads", who);
  TPF_REQUIRE(c.D >= 8 && c.D <= 128 && c.D % 8 == 0, TPF_ERR_UNSUPPORTED, "%s: head dim %lld is no multiple of 8 up to 128", who,
              (long long)c.D);
  TPF_REQUIRE(c.N <= kWindowMost && c.M <= kWindowMost && c.B <= 65535 && c.HK <= 65535 && c.H < (1 << 20), TPF_ERR_UNSUPPORTED,
              "%s: extent too large", who);
  TPF_REQUIRE(c.left >= 0 && c.right >= 0 && (c.left < kWindowMost || c.left == kWindowUnlimited) &&
                  (c.right < kWindowMost || c.right == kWindowUnlimited),
              TPF_ERR_INVALID_ARGUMENT, "%s: the reach of the window must be in 0 .. 2^28 - 1 or unlimited", who);
  TPF_REQUIRE(c.sinks >= 0 && c.sinks <= kMostSinks, TPF_ERR_UNSUPPORTED, "%s: 0 to %d sinks", who, kMostSinks);
  TPF_REQUIRE(c.offset >= -kWindowMost && c.offset <= kWindowMost, TPF_ERR_INVALID_ARGUMENT,
              "%s: the position of the first query must be within 2^28", who);
  TPF_REQUIRE(c.scale > 0.f && c.scale <= 3.402823466e38f, TPF_ERR_INVALID_ARGUMENT, "%s: the scale must be positive and finite",
              who);
  *p = {};
  p->B = (int)c.B, p->N = (int)c.N, p->M = (int)c.M, p->H = (int)c.H, p->HK = (int)c.HK, p->D = (int)c.D;
  p->G = (int)(c.H / c.HK);
  p->left = c.left, p->right = c.right, p->sinks = c.sinks;
  p->offsets = c.offsets, p->offset = (int)c.offset, p->lengths = c.lengths;
  p->scale = c.scale;
  return TPF_OK;
}

int check_operand(const void* x, const int64_t* strides, const int64_t (&sizes)[3], const char* who, const char* name) {
  TPF_REQUIRE(x != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: %s is a null pointer", who, name);
  TPF_REQUIRE((reinterpret_cast<uintptr_t>(x) & 15) == 0, TPF_ERR_INVALID_ARGUMENT, "%s: %s must be 16-byte aligned", who, name);
  for (int i = 0; i < 3; ++i)
    TPF_REQUIRE(sizes[i] <= 1 || (strides[i] > 0 && strides[i] % 8 == 0 && strides[i] < (1ll << 38)), TPF_ERR_INVALID_ARGUMENT,
                "%s: strides of %s must be positive multiples of 8 elements", who, name);
  return TPF_OK;
}

int check_inputs(const WindowCall& c, const char* who) {
  const int64_t q[3] = {c.B, c.N, c.H}, k[3] = {c.B, c.M, c.HK};
  if (int rc = check_operand(c.q, c.qs, q, who, "q")) return rc;
  if (int rc = check_operand(c.out, c.qs, {0, 0, 0}, who, "out")) return rc;
  if (c.M == 0) return TPF_OK;
  if (int rc = check_operand(c.k, c.ks, k, who, "k")) return rc;
  return check_operand(c.v, c.vs, k, who, "v");
}

}  // namespace

int window_attn_fwd(const WindowCall& c, cudaStream_t stream) {
  WindowParams p;
  if (int rc = make_params(&p, c, "window_attn_fwd")) return rc;
  if (c.B == 0 || c.N == 0) return TPF_OK;
  if (int rc = check_inputs(c, "window_attn_fwd")) return rc;
  // A CTA of the one kernel has 16 rows, queries times heads of a group, of the other 128 queries of a head.  The first is quicker while
  // its CTAs find an SM each, and beyond that where there are fewer of them by a quarter.  (Heads 32 on 8 of 128 elements, window 1024,
  // us, few / many: 8 sequences of 8 queries 17 / 20, of 16 26 / 20, of 64 95 / 20; one sequence of 32 12 / 16, of 128 26 / 18; 64
  // single queries 55 / 116.  As many key heads as heads, where both have as many CTAs: 32 of 128, single queries of 4 sequences 18.5 /
  // 19.5, of 16 56 / 49, of 64 191 / 175; 16 of 64: of 16 20.6 / 20.8, of 64 61 / 64, 2 to 8 queries of 64 61 / 69, the rule's worst; 8 of
  // 64: of 64 39 / 34.  Heads 64 on 8: 16 sequences of 8 queries 53 / 71, of 16 102 / 71; 32 on 1: of 8 28 / 39, of 16 52 / 38.)
  const int64_t few = c.B * c.HK * ((c.N * p.G + 15) / 16), many = c.B * c.H * ((c.N + 127) / 128);
  if (c.M > 0 && few > sm_count() && 4 * few > 3 * many) return window_many(c, p, stream);
  return window_few(c, p, stream);
}

int64_t window_attn_bwd_workspace_bytes(const WindowCall& c) {
  return c.B > 0 && c.N > 0 && c.M > 0 && c.H > 0 && c.HK > 0 && c.D > 0 ? window_bwd_workspace_bytes(c) : 0;
}

int window_attn_bwd(const WindowCall& c, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  const char* who = "window_attn_bwd";
  WindowParams p;
  if (int rc = make_params(&p, c, who)) return rc;
  TPF_REQUIRE((c.dk == nullptr) == (c.dv == nullptr), TPF_ERR_INVALID_ARGUMENT, "%s: dk and dv come together", who);
  if (c.B == 0 || c.N == 0 || c.M == 0) {
    const size_t q = (size_t)(c.B * c.N * c.H * c.D) * 2, k = (size_t)(c.B * c.M * c.HK * c.D) * 2;
    if (c.dq != nullptr && q > 0) TPF_CUDA_OK(cudaMemsetAsync(c.dq, 0, q, stream));
    if (c.dk != nullptr && k > 0) {
      TPF_CUDA_OK(cudaMemsetAsync(c.dk, 0, k, stream));
      TPF_CUDA_OK(cudaMemsetAsync(c.dv, 0, k, stream));
    }
    return TPF_OK;
  }
  if (int rc = check_inputs(c, who)) return rc;
  TPF_REQUIRE(c.lse != nullptr && c.d_out != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  TPF_REQUIRE_ALIGNED16(c.d_out, who, "d_out");
  TPF_REQUIRE_ALIGNED16(c.dq, who, "dq");
  TPF_REQUIRE_ALIGNED16(c.dk, who, "dk");
  TPF_REQUIRE_ALIGNED16(c.dv, who, "dv");
  if (c.dq == nullptr && c.dk == nullptr) return TPF_OK;
  return window_bwd(c, p, workspace, workspace_bytes, stream);
}

}  // namespace tpf

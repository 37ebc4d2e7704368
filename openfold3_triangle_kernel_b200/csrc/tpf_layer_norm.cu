// Layer norm of rows: forward (the backward is tpf_layer_norm_bwd.cu).
//
//   mean = sum x / C,  rstd = (sum (x - mean)^2 / C + eps)^-1/2,  xh = (x - mean) rstd,  y = w xh + b
//   dx = rstd (w dy - m1 - xh m2) with m1 = mean(w dy), m2 = mean(w dy xh);  dw = sum_r dy xh,  db = sum_r dy
//
// Both passes are bound by memory: a row is loaded once, stays in registers (32 elements a thread at most), and leaves
// once.  The mean is subtracted before the squares are summed: a row whose mean is large against its spread loses nothing.
// All sums are fp32 in a fixed order.  The parameter gradients are summed in registers by each CTA over the rows it walks
// and folded by a second small kernel in CTA order: no atomics, the same bits every time.
//
// With an 8-bit checkpoint (tpf_rows.cuh) the forward writes the codes of x next to y, and the backward takes x from them
// and the statistics from the true x.
#include "tpf_layer_norm.cuh"

namespace tpf {

namespace {

// ROWS rows a team at a time, all their loads issued before the first use.
template <typename T, class Tm, int ROWS, bool KEEP>
__global__ void __launch_bounds__(Tm::BLOCK) norm_fwd_kernel(const NormArgs a, T* __restrict__ y, float eps) {
  griddep_wait();
  constexpr int E = Tm::E, VEC = Tm::VEC;
  __shared__ float red[Tm::TS > 32 ? 2 * Tm::WARPS * ROWS : 1];
  const Tm tm;
  int turn = 0;
  const int64_t row0 = ((int64_t)blockIdx.x * Tm::TEAMS + tm.index) * ROWS;
  float x[ROWS][E];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int i = 0; i < Tm::ITEMS; ++i) {
      const int c = tm.column(i);
      if (row0 + r < a.rows && c < a.cols)
        load_vec<T, VEC>(static_cast<const T*>(a.x) + (row0 + r) * a.x_pitch + c, &x[r][i * VEC]);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[r][i * VEC + e] = 0.f;
    }
  if constexpr (KEEP) {
    constexpr int NG = VEC == 8 ? Tm::ITEMS : (Tm::ITEMS + 3) / 4;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float amax[NG];
      group_amax<Tm>(x[r], amax);
#pragma unroll
      for (int i = 0; i < Tm::ITEMS; ++i) {
        const int c = tm.column(i);
        const GroupScale s = group_scale(amax[VEC == 8 ? i : i / 4]);
        if (row0 + r < a.rows && c < a.cols) {
          store_codes<VEC>(a.codes + (row0 + r) * a.cols + c, &x[r][i * VEC], s);
          if (c % kGroup == 0) a.scales[(row0 + r) * a.groups + c / kGroup] = s.down;
        }
      }
    }
  }
  float sum[ROWS], mean[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    sum[r] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[r] += x[r][e];
  }
  team_sum<Tm, ROWS>(sum, red, turn);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    mean[r] = sum[r] * a.inv_cols;
    sum[r] = 0.f;
#pragma unroll
    for (int i = 0; i < Tm::ITEMS; ++i) {
      const bool on = tm.column(i) < a.cols;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float& v = x[r][i * VEC + e];
        v = on ? v - mean[r] : 0.f;
        sum[r] += v * v;
      }
    }
  }
  team_sum<Tm, ROWS>(sum, red, turn);
  float rstd[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    rstd[r] = rsqrtf(sum[r] * a.inv_cols + eps);
    if (a.mean != nullptr && tm.t == 0 && row0 + r < a.rows) {
      a.mean[row0 + r] = mean[r];
      a.rstd[row0 + r] = rstd[r];
    }
  }
#pragma unroll
  for (int i = 0; i < Tm::ITEMS; ++i) {
    const int c = tm.column(i);
    if (c >= a.cols) continue;
    float w[VEC], b[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[e] = param_at(a.w, c + e, 1.f);
      b[e] = param_at(a.b, c + e, 0.f);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (row0 + r >= a.rows) continue;
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] = x[r][i * VEC + e] * rstd[r] * w[e] + b[e];
      store_vec<T, VEC>(y + (row0 + r) * a.cols + c, o);
    }
  }
}

struct FwdLaunch {
  const NormArgs& a;
  void* y;
  float eps;
  cudaStream_t stream;
  template <typename T, class Tm>
  int run() const {
    constexpr int ROWS = rows_in_flight<Tm>();
    const int64_t blocks = (a.rows + Tm::TEAMS * ROWS - 1) / (Tm::TEAMS * ROWS);
    TPF_REQUIRE(blocks < (1ll << 31), TPF_ERR_INVALID_ARGUMENT, "layer norm: too many rows");
    if (a.codes != nullptr)
      launch_kernel(norm_fwd_kernel<T, Tm, ROWS, true>, dim3((unsigned)blocks), dim3(Tm::BLOCK), 0, stream, a,
                    static_cast<T*>(y), eps);
    else
      launch_kernel(norm_fwd_kernel<T, Tm, ROWS, false>, dim3((unsigned)blocks), dim3(Tm::BLOCK), 0, stream, a,
                    static_cast<T*>(y), eps);
    TPF_LAUNCH_OK();
    return TPF_OK;
  }
};

}  // namespace

int layer_norm_fwd(const NormCall& c, void* y, float eps, cudaStream_t stream) {
  NormArgs a;
  if (int rc = make_norm_args(&a, c, "layer_norm_fwd")) return rc;
  if (c.rows == 0) return TPF_OK;
  TPF_REQUIRE(c.x != nullptr && y != nullptr, TPF_ERR_INVALID_ARGUMENT, "layer_norm_fwd: null pointer");
  const bool vec = c.cols % 8 == 0 && rows_vec_ok(c.x, c.x_pitch, c.type) && vec_ok(y, c.type) &&
                   (reinterpret_cast<uintptr_t>(c.codes) & 7) == 0;
  return by_type(FwdLaunch{a, y, eps, stream}, c.type, a.cols, vec);
}

}  // namespace tpf

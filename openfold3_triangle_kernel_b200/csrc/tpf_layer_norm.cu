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

// A CTA walks the row groups blockIdx.x, + gridDim.x, ..., ROWS rows a team at a time; the next rows are loaded while these
// are worked on, and the parameters stay in registers.
template <typename T, class Tm, int ROWS, bool KEEP>
__global__ void __launch_bounds__(Tm::MAXB, min_ctas<Tm, false>()) norm_fwd_kernel(const NormArgs a, T* __restrict__ y, float eps) {
  griddep_wait();
  constexpr int E = Tm::E, P = E / 2, ITEMS = Tm::ITEMS;
  __shared__ __align__(8) float red[Tm::BLOCK ? 2 * 64 : 1];
  const Tm tm;
  int turn = 0;
  int at[ITEMS];
  bool on[ITEMS], ragged = false;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    on[i] = tm.column(i) < a.cols;
    at[i] = on[i] ? tm.column(i) : 0;
    ragged |= !on[i];
  }
  // (BLOCK) columns of this warp; only the last warp of the team has fewer than 32 E
  const float warp_inv = 1.f / (float)min(32 * E, a.cols - (int)(threadIdx.x >> 5) * 32 * E);
  const int64_t step = (int64_t)gridDim.x * Tm::TEAMS * ROWS;
  int64_t base = (int64_t)blockIdx.x * Tm::TEAMS * ROWS;
  Frag<T, Tm> raw[ROWS];
  auto load = [&](const RowSet<ROWS>& rows) {
    const T* src = static_cast<const T*>(a.x) + rows.first * a.x_pitch;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) raw[r].load(src + rows.at(r) * a.x_pitch, at);
  };
  RowSet<ROWS> next(base + tm.index * ROWS, a.rows);
  load(next);
  uint64_t w[P], b[P];
  {
    float f[E], g[E];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      param_load<Tm::VEC, 1>(a.w, tm.column(i), a.cols, 1.f, f + i * Tm::VEC);
      param_load<Tm::VEC, 1>(a.b, tm.column(i), a.cols, 0.f, g + i * Tm::VEC);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      w[k] = f2_pack(f[2 * k], f[2 * k + 1]);
      b[k] = f2_pack(g[2 * k], g[2 * k + 1]);
    }
  }
  // every team of a block makes the same number of rounds: the sums over a team are converged
  for (; base < a.rows; base += step) {
    const RowSet<ROWS> rows = next;
    uint64_t x[ROWS][P];
    constexpr int NG = Groups<Tm>::N, N = ROWS * NG;
    float amax[KEEP ? N : 1];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (ragged) raw[r].mask(on);
      raw[r].get(x[r]);
      if constexpr (KEEP) raw[r].amax(amax + r * NG);
    }
    if (base + step < a.rows) {
      next = RowSet<ROWS>(base + step + tm.index * ROWS, a.rows);
      load(next);
    }
    if constexpr (KEEP) {
      float up[N];
      const float down = group_scales<N, Groups<Tm>::LANES>(amax, up);
      int8_t* codes = a.codes + rows.first * a.code_pitch;
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (r < rows.count) store_codes<Tm>(codes + r * (int64_t)a.code_pitch, x[r], up + r * NG, at, on);
      // of the lanes that hold a group, number n (mod N) has the scale of group n
      const int mine = threadIdx.x & (N - 1), first = threadIdx.x & (Groups<Tm>::LANES - 1);
      const int r = mine / NG, g = mine % NG;
      // first column of the group
      const int c0 = tm.column(0) + (Tm::VEC == 8 ? (g * (Tm::BLOCK ? 32 : Tm::TS) - first) * 8 : g * 128 - first);
      if (first == mine && r < rows.count && c0 < a.cols) a.scales[(rows.first + r) * a.groups + c0 / kGroup] = down;
    }
    float sum[ROWS], mean[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint64_t s = x[r][0];
#pragma unroll
      for (int k = 1; k < P; ++k) s = f2_add(s, x[r][k]);
      sum[r] = f2_sum(s);
    }
    if constexpr (!Tm::BLOCK) {
      team_sum<Tm, ROWS>(sum, red, turn);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) mean[r] = sum[r] * a.inv_cols;
    } else {
      // each warp about its own mean; the warps' means and sums of squares are put together below
      warp_sum(sum);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) mean[r] = sum[r] * warp_inv;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const uint64_t m = f2_dup(-mean[r]);
      uint64_t s = 0;
#pragma unroll
      for (int k = 0; k < P; ++k) x[r][k] = f2_add(x[r][k], m);
      if (ragged) mask_pairs<Tm>(x[r], on);
#pragma unroll
      for (int k = 0; k < P; ++k) s = f2_fma(x[r][k], x[r][k], s);
      sum[r] = f2_sum(s);
    }
    if constexpr (!Tm::BLOCK) {
      team_sum<Tm, ROWS>(sum, red, turn);
    } else {
      // n values with mean m and sum of squares q about it, and others: q + q' + n (m - M)^2 + n' (m' - M)^2 about the
      // common mean M (Chan, Golub and LeVeque, "Updating formulae", 1979): one barrier for both statistics
      using X = CrossWarp<Tm, ROWS>;
      warp_sum(sum);
      float2* m = reinterpret_cast<float2*>(red) + turn * 32;
      turn ^= 1;
      const int lane = threadIdx.x & 31, warps = blockDim.x >> 5, k = lane & (X::W - 1);
      if (lane == 0)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) m[r * X::W + (threadIdx.x >> 5)] = make_float2(mean[r], sum[r]);
      __syncthreads();
      const bool exists = X::exists() && lane < ROWS * X::W;
      const float2 part = exists ? m[lane] : make_float2(0.f, 0.f);
      const float n = exists ? (float)(k + 1 < warps ? 32 * E : a.cols - k * 32 * E) : 0.f;
      const float all = X::sum(part.x * (n * a.inv_cols)), d = part.x - all;
      const float sq = X::sum(fmaf(d * n, d, part.y));
      float own[ROWS];
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        own[r] = mean[r];
        mean[r] = __shfl_sync(0xffffffffu, all, r * X::W);
        sum[r] = __shfl_sync(0xffffffffu, sq, r * X::W);
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const uint64_t shift = f2_dup(own[r] - mean[r]);
#pragma unroll
        for (int k = 0; k < P; ++k) x[r][k] = f2_add(x[r][k], shift);
      }
    }
    T* dst = y + rows.first * a.cols;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float rstd = rsqrtf(fmaf(sum[r], a.inv_cols, eps));
      if (r >= rows.count) continue;
      if (a.mean != nullptr && tm.t == 0) {
        a.mean[rows.first + r] = mean[r];
        a.rstd[rows.first + r] = rstd;
      }
      const uint64_t rs = f2_dup(rstd);
#pragma unroll
      for (int k = 0; k < P; ++k) x[r][k] = f2_fma(f2_mul(x[r][k], rs), w[k], b[k]);
      store_row<T, Tm>(dst + r * (int64_t)a.cols, x[r], at, on);
    }
  }
}

struct FwdLaunch {
  const NormArgs& a;
  void* y;
  float eps;
  cudaStream_t stream;
  // The team for rows of `cols` elements.  vec: eight elements at a time are possible.
  template <typename T>
  int by_width(int cols, bool vec) const {
    if (vec) {
      if (cols <= 32) return run<T, Team<8, 4, 1>>();
      // 16-bit types: half the lanes with two pieces each, which saves a step of every sum over the team and shares the
      // bookkeeping of a row (768 * 768 rows of 128 bf16 channels: 49.7 us against 50.6, with codes 62.8 against 63.5;
      // 147456 rows 11.4 against 12.5).  32-bit ones have no registers for it (300000 rows with codes: 59 against 57).
      if constexpr (sizeof(T) == 2) {
        if (cols <= 64) return run<T, Team<8, 4, 2>>();
        if (cols <= 128) return run<T, Team<8, 8, 2>>();
        if (cols <= 256) return run<T, Team<8, 16, 2>>();
      }
      if (cols <= 64) return run<T, Team<8, 8, 1>>();
      if (cols <= 128) return run<T, Team<8, 16, 1>>();
      if (cols <= 256) return run<T, Team<8, 32, 1>>();
      if (cols <= 512) return run<T, Team<8, 32, 2>>();
      if (cols <= 1024) return run<T, Team<8, 0, 1, 128>>();
      if (cols <= 4096) return run<T, Team<8, 0, 2, 256>>();
      return run<T, Team<8, 0, 4, 256>>();
    }
    // (Few lanes a row: what is done once a row weighs most.  300000 rows of 60 bf16 channels take 29.3 us, 55.7 with a warp
    // and four elements a lane; 97: 55, 58; 60000 of 501 from codes 63, 74 with two warps.)
    if (cols <= 32) return run<T, Team<1, 8, 4>>();
    if (cols <= 64) return run<T, Team<1, 8, 8>>();
    if (cols <= 128) return run<T, Team<1, 16, 8>>();
    if (cols <= 256) return run<T, Team<1, 16, 16>>();
    if (cols <= 512) return run<T, Team<1, 32, 16>>();
    if (cols <= 2048) return run<T, Team<1, 0, 8, 256>>();
    if (cols <= 4096) return run<T, Team<1, 0, 8, 512>>();
    return run<T, Team<1, 0, 16, 512>>();
  }
  template <typename T, class Tm>
  int run() const {
    return a.codes != nullptr ? go<T, Tm, true>() : go<T, Tm, false>();
  }
  template <typename T, class Tm, bool KEEP>
  int go() const {
    constexpr int ROWS = rows_in_flight<T, Tm, false>();
    static PerDeviceInt regs;
    const auto kern = norm_fwd_kernel<T, Tm, ROWS, KEEP>;
    const int threads = Tm::threads(a.cols);
    int fit = 1;
    if (int rc = resident_ctas(kern, threads, regs, &fit)) return rc;
    const int64_t want = (a.rows + Tm::TEAMS * ROWS - 1) / (Tm::TEAMS * ROWS), most = (int64_t)fit * sm_count();
    launch_kernel(kern, dim3((unsigned)(want < most ? want : most)), dim3(threads), 0, stream, a, static_cast<T*>(y), eps);
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
                   (reinterpret_cast<uintptr_t>(c.codes) & 15) == 0;
  return by_type(FwdLaunch{a, y, eps, stream}, c.type, a.cols, vec);
}

}  // namespace tpf

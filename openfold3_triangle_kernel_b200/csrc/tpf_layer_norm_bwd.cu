// Layer norm of rows: backward (formulas in tpf_layer_norm.cu).
#include "tpf_layer_norm.cuh"

namespace tpf {

namespace {

// A CTA walks the row groups blockIdx.x, + gridDim.x, ...; partials: [gridDim.x][2][cols], the CTA's sums of dy xh and dy.
template <typename T, class Tm, int ROWS, bool CODES>
__global__ void __launch_bounds__(Tm::BLOCK) norm_bwd_kernel(const NormArgs a, const T* __restrict__ dy, T* __restrict__ dx,
                                                             float* __restrict__ partials) {
  griddep_wait();
  constexpr int E = Tm::E, VEC = Tm::VEC;
  __shared__ float red[Tm::TS > 32 ? 2 * Tm::WARPS * 2 * ROWS : 2 * Tm::COLS];
  const Tm tm;
  int turn = 0;
  float w[E], aw[E], ab[E];
#pragma unroll
  for (int i = 0; i < Tm::ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = tm.column(i);
      w[i * VEC + e] = c < a.cols ? param_at(a.w, c + e, 1.f) : 0.f;
      aw[i * VEC + e] = ab[i * VEC + e] = 0.f;
    }
  const int64_t step = (int64_t)gridDim.x * Tm::TEAMS * ROWS;
  // every team of a block makes the same number of rounds: the sums over a team are converged
  for (int64_t base = (int64_t)blockIdx.x * Tm::TEAMS * ROWS; base < a.rows; base += step) {
    const int64_t row0 = base + tm.index * ROWS;
    float d[ROWS][E], xh[ROWS][E], rstd[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t row = row0 + r;
      const bool live = row < a.rows;
      const float mean = live ? a.mean[row] : 0.f;
      rstd[r] = live ? a.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < Tm::ITEMS; ++i) {
        const int c = tm.column(i);
        if (live && c < a.cols) {
          load_vec<T, VEC>(dy + row * a.cols + c, &d[r][i * VEC]);
          if constexpr (CODES)
            load_codes<VEC>(a.codes + row * a.cols + c, a.scales[row * a.groups + c / kGroup], &xh[r][i * VEC]);
          else
            load_vec<T, VEC>(static_cast<const T*>(a.x) + row * a.x_pitch + c, &xh[r][i * VEC]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) xh[r][i * VEC + e] = (xh[r][i * VEC + e] - mean) * rstd[r];
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[r][i * VEC + e] = xh[r][i * VEC + e] = 0.f;
        }
      }
    }
    float s[2 * ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float wd = w[e] * d[r][e];
        s[2 * r] += wd;
        s[2 * r + 1] += wd * xh[r][e];
        aw[e] += d[r][e] * xh[r][e];
        ab[e] += d[r][e];
      }
    }
    team_sum<Tm, 2 * ROWS>(s, red, turn);
    if (dx != nullptr) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float m1 = s[2 * r] * a.inv_cols, m2 = s[2 * r + 1] * a.inv_cols;
#pragma unroll
        for (int i = 0; i < Tm::ITEMS; ++i) {
          const int c = tm.column(i);
          float o[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int k = i * VEC + e;
            o[e] = rstd[r] * (w[k] * d[r][k] - m1 - xh[r][k] * m2);
          }
          if (row0 + r < a.rows && c < a.cols) store_vec<T, VEC>(dx + (row0 + r) * a.cols + c, o);
        }
      }
    }
  }
  if (partials == nullptr) return;
  float* pw = partials + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (Tm::TS > 32) {
#pragma unroll
    for (int i = 0; i < Tm::ITEMS; ++i) {
      const int c = tm.column(i);
      if (c < a.cols)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          pw[c + e] = aw[i * VEC + e];
          pw[a.cols + c + e] = ab[i * VEC + e];
        }
    }
  } else {
    // the teams of a warp, then the warps one after the other
#pragma unroll
    for (int k = 0; k < E; ++k)
#pragma unroll
      for (int off = Tm::TS; off < 32; off <<= 1) {
        aw[k] += __shfl_xor_sync(0xffffffffu, aw[k], off);
        ab[k] += __shfl_xor_sync(0xffffffffu, ab[k], off);
      }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int turn_of = 0; turn_of < Tm::WARPS; ++turn_of) {
      if (warp == turn_of && lane < Tm::TS) {
#pragma unroll
        for (int i = 0; i < Tm::ITEMS; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int c = tm.column(i) + e, k = i * VEC + e;
            red[c] = turn_of == 0 ? aw[k] : red[c] + aw[k];
            red[Tm::COLS + c] = turn_of == 0 ? ab[k] : red[Tm::COLS + c] + ab[k];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.cols; c += Tm::BLOCK) {
      pw[c] = red[c];
      pw[a.cols + c] = red[Tm::COLS + c];
    }
  }
}

// out[j] = sum over terms of partials[term][j], j < 2 cols.  A CTA owns 32 columns; eight threads of each add a contiguous
// range of the terms (eight loads in flight), then their sums are added in range order.
__global__ void __launch_bounds__(256) norm_fold_kernel(const float* __restrict__ partials, int terms, int cols, ParamOut dw,
                                                        ParamOut db) {
  griddep_wait();
  __shared__ float red[256];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int j = blockIdx.x * 32 + lane;
  const int per = (terms + 7) / 8, k0 = g * per, k1 = min(terms, k0 + per);
  const bool first = j < cols;
  const ParamOut& out = first ? dw : db;
  float s = 0.f;
  if (j < 2 * cols && out.p != nullptr)
    for (int k = k0; k < k1; k += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = k + u < k1 ? partials[(int64_t)(k + u) * 2 * cols + j] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (g == 0 && j < 2 * cols && out.p != nullptr) {
    for (int w = 1; w < 8; ++w) s += red[w * 32 + lane];
    param_put(out, first ? j : j - cols, s);
  }
}

constexpr int kMaxCtasPerSm = 8;

struct BwdLaunch {
  const NormArgs& a;
  const NormGrads& g;
  float* partials;
  cudaStream_t stream;
  template <typename T, class Tm>
  int run() const {
    constexpr int ROWS = rows_in_flight<Tm>();
    const int64_t want = (a.rows + Tm::TEAMS * ROWS - 1) / (Tm::TEAMS * ROWS);
    const int64_t most = (int64_t)sm_count() * (Tm::BLOCK >= 512 ? 2 : Tm::BLOCK >= 256 ? 3 : kMaxCtasPerSm);
    const int blocks = (int)(want < most ? want : most);
    const T* dy = static_cast<const T*>(g.dy);
    T* dx = static_cast<T*>(g.dx);
    if (a.codes != nullptr)
      launch_kernel(norm_bwd_kernel<T, Tm, ROWS, true>, dim3(blocks), dim3(Tm::BLOCK), 0, stream, a, dy, dx, partials);
    else
      launch_kernel(norm_bwd_kernel<T, Tm, ROWS, false>, dim3(blocks), dim3(Tm::BLOCK), 0, stream, a, dy, dx, partials);
    TPF_LAUNCH_OK();
    if (partials == nullptr) return TPF_OK;
    launch_kernel(norm_fold_kernel, dim3((2 * a.cols + 31) / 32), dim3(256), 0, stream, partials, blocks, a.cols,
                  ParamOut{g.dweight, g.dweight_type}, ParamOut{g.dbias, g.dbias_type});
    TPF_LAUNCH_OK();
    return TPF_OK;
  }
};

}  // namespace

int64_t layer_norm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  const int64_t most = (int64_t)sm_count() * kMaxCtasPerSm;
  return (rows < most ? rows : most) * 2 * cols * 4;
}

int layer_norm_bwd(const NormCall& c, const NormGrads& g, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  NormArgs a;
  if (int rc = make_norm_args(&a, c, "layer_norm_bwd")) return rc;
  const bool params = g.dweight != nullptr || g.dbias != nullptr;
  TPF_REQUIRE((g.dweight == nullptr || row_type_ok(g.dweight_type)) && (g.dbias == nullptr || row_type_ok(g.dbias_type)),
              TPF_ERR_INVALID_ARGUMENT, "layer_norm_bwd: unknown parameter type");
  if (c.rows == 0) {
    for (int k = 0; k < 2; ++k) {
      void* p = k == 0 ? g.dweight : g.dbias;
      const int type = k == 0 ? g.dweight_type : g.dbias_type;
      if (p != nullptr) TPF_CUDA_OK(cudaMemsetAsync(p, 0, c.cols * row_type_size(type), stream));
    }
    return TPF_OK;
  }
  if (!params && g.dx == nullptr) return TPF_OK;
  TPF_REQUIRE((c.x != nullptr || c.codes != nullptr) && c.mean != nullptr && g.dy != nullptr, TPF_ERR_INVALID_ARGUMENT,
              "layer_norm_bwd: null pointer");
  const int64_t need = layer_norm_bwd_workspace_bytes(c.rows, c.cols);
  TPF_REQUIRE(!params || (workspace != nullptr && workspace_bytes >= need), TPF_ERR_WORKSPACE,
              "layer_norm_bwd: workspace of %lld bytes required, %lld given", (long long)need, (long long)workspace_bytes);
  TPF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 3) == 0, TPF_ERR_INVALID_ARGUMENT,
              "layer_norm_bwd: misaligned workspace");
  const bool from_codes = c.codes != nullptr;
  const bool vec = c.cols % 8 == 0 && (from_codes ? (reinterpret_cast<uintptr_t>(c.codes) & 7) == 0
                                                  : rows_vec_ok(c.x, c.x_pitch, c.type)) &&
                   vec_ok(g.dy, c.type) && (g.dx == nullptr || vec_ok(g.dx, c.type));
  return by_type(BwdLaunch{a, g, params ? static_cast<float*>(workspace) : nullptr, stream}, c.type, a.cols, vec);
}

}  // namespace tpf

// Layer norm of rows: backward (formulas in tpf_layer_norm.cu).
#include "tpf_layer_norm.cuh"

namespace tpf {

namespace {

// Where a CTA's sums of dy xh and dy go: its terms, or, from the only CTA, the gradients themselves.
struct SumsOut {
  float* terms;  // [gridDim.x][2][cols], or nullptr
  ParamOut dw, db;
  __device__ __forceinline__ bool wanted() const { return terms != nullptr || dw.p != nullptr || db.p != nullptr; }
  __device__ __forceinline__ void put(int cols, int c, float w, float b) const {
    if (terms != nullptr) {
      float* t = terms + (int64_t)blockIdx.x * 2 * cols;
      t[c] = w;
      t[cols + c] = b;
    } else {
      if (dw.p != nullptr) param_put(dw, c, w);
      if (db.p != nullptr) param_put(db, c, b);
    }
  }
};

// A CTA walks the row groups blockIdx.x, + gridDim.x, ... as in the forward.  From codes xh = code (s rstd) - mean rstd, one
// FMA, off by three roundings of what it subtracts; from x itself the mean is taken off first, where it may be large.
template <typename T, class Tm, int ROWS, bool CODES>
__global__ void __launch_bounds__(Tm::MAXB, min_ctas<Tm, true>())
    norm_bwd_kernel(const NormArgs a, const T* __restrict__ dy, T* __restrict__ dx, const SumsOut out) {
  griddep_wait();
  constexpr int E = Tm::E, P = E / 2, ITEMS = Tm::ITEMS, NG = Groups<Tm>::N;
  constexpr int WARPS = Tm::MAXB / 32;
  __shared__ __align__(16) float red[Tm::BLOCK ? 2 * 32 : WARPS * 2 * Tm::COLS];
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
  const int64_t step = (int64_t)gridDim.x * Tm::TEAMS * ROWS;
  int64_t base = (int64_t)blockIdx.x * Tm::TEAMS * ROWS;
  Frag<T, Tm> dy_raw[ROWS], x_raw[CODES ? 1 : ROWS];
  CodeFrag<Tm> c_raw[CODES ? ROWS : 1];
  float down[CODES ? ROWS : 1][NG], mean[ROWS], rstd[ROWS];
  auto request = [&](int64_t row0) {
    const RowSet<ROWS> rows(row0, a.rows);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t row = rows.first + rows.at(r);
      dy_raw[r].load(dy + row * a.cols, at);
      if constexpr (CODES) {
        c_raw[r].load(a.codes + row * a.code_pitch, at);
        const float* s = a.scales + row * a.groups;
#pragma unroll
        for (int g = 0; g < NG; ++g) down[r][g] = s[at[g * (ITEMS / NG)] / kGroup];
      } else {
        x_raw[r].load(static_cast<const T*>(a.x) + row * a.x_pitch, at);
      }
      mean[r] = a.mean[row];
      rstd[r] = a.rstd[row];
    }
  };
  // Three rounds ahead into L2: what a request waits for is then L2's latency (8192 rows of 4096 channels 51.3 -> 48.0 us,
  // 5000 of 8192 61.4 -> 57.6; two rounds and five the same or less).  Single elements: 8000 rows of 4099 257 -> 197, narrower ones
  // gain nothing.
  constexpr int AHEAD = 3;
  auto prefetch = [&](int64_t first) {
    if constexpr (Tm::VEC == 8 || Tm::E >= 16) {
      constexpr int NR = Tm::TEAMS * ROWS;
      if (threadIdx.x != 0 || first + NR > a.rows) return;
      row_prefetch(dy + first * a.cols, NR * a.cols * (int)sizeof(T));
      if constexpr (CODES) row_prefetch(a.codes + first * a.code_pitch, NR * a.code_pitch);
      else if (a.x_pitch == a.cols) row_prefetch(static_cast<const T*>(a.x) + first * a.x_pitch, NR * a.cols * (int)sizeof(T));
    }
  };
  request(base + tm.index * ROWS);
  for (int k = 1; k < AHEAD; ++k) prefetch(base + k * step);
  uint64_t w[P], aw[P], ab[P];
  {
    float f[E];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) param_load<Tm::VEC, 1>(a.w, tm.column(i), a.cols, 1.f, f + i * Tm::VEC);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      w[k] = f2_pack(f[2 * k], f[2 * k + 1]);
      aw[k] = ab[k] = 0;
    }
  }
  // every team of a block makes the same number of rounds: the sums over a team are converged
  for (; base < a.rows; base += step) {
    const RowSet<ROWS> rows(base + tm.index * ROWS, a.rows);
    prefetch(base + AHEAD * step);
    uint64_t d[ROWS][P], xh[ROWS][P];
    float rs[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      rs[r] = rstd[r];
      if (ragged) dy_raw[r].mask(on);
      dy_raw[r].get(d[r]);
      if (r >= rows.count)
#pragma unroll
        for (int k = 0; k < P; ++k) d[r][k] = 0;
      if constexpr (CODES) {
        c_raw[r].get(xh[r]);
        const uint64_t g = f2_dup(-mean[r] * rstd[r]);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const uint64_t f = f2_dup(down[r][n] * rstd[r]);
#pragma unroll
          for (int k = n * (P / NG); k < (n + 1) * (P / NG); ++k) xh[r][k] = f2_fma(xh[r][k], f, g);
        }
      } else {
        if (ragged) x_raw[r].mask(on);
        x_raw[r].get(xh[r]);
        const uint64_t m = f2_dup(-mean[r]), f = f2_dup(rstd[r]);
#pragma unroll
        for (int k = 0; k < P; ++k) xh[r][k] = f2_mul(f2_add(xh[r][k], m), f);
      }
    }
    if (base + step < a.rows) request(base + step + tm.index * ROWS);
    float s[2 * ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint64_t s1 = 0, s2 = 0;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        aw[k] = f2_fma(d[r][k], xh[r][k], aw[k]);
        ab[k] = f2_add(ab[k], d[r][k]);
        d[r][k] = f2_mul(d[r][k], w[k]);
        s1 = f2_add(s1, d[r][k]);
        s2 = f2_fma(d[r][k], xh[r][k], s2);
      }
      s[2 * r] = f2_sum(s1);
      s[2 * r + 1] = f2_sum(s2);
    }
    team_sum<Tm, 2 * ROWS>(s, red, turn);
    if (dx != nullptr) {
      T* dst = dx + rows.first * a.cols;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        if (r >= rows.count) continue;
        const uint64_t m1 = f2_dup(-s[2 * r] * a.inv_cols), m2 = f2_dup(-s[2 * r + 1] * a.inv_cols), f = f2_dup(rs[r]);
#pragma unroll
        for (int k = 0; k < P; ++k) d[r][k] = f2_mul(f2_fma(xh[r][k], m2, f2_add(d[r][k], m1)), f);
        store_row<T, Tm>(dst + r * (int64_t)a.cols, d[r], at, on);
      }
    }
  }
  if (!out.wanted()) return;
  float fw[E], fb[E];
#pragma unroll
  for (int k = 0; k < P; ++k) {
    f2_unpack(aw[k], fw[2 * k], fw[2 * k + 1]);
    f2_unpack(ab[k], fb[2 * k], fb[2 * k + 1]);
  }
  if constexpr (Tm::BLOCK) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = tm.column(i);
      if (c >= a.cols) continue;
      if (Tm::VEC == 8 && out.terms != nullptr) {  // (element by element: 10 us at 296 CTAs of 4096 columns)
        float* t = out.terms + (int64_t)blockIdx.x * 2 * a.cols + c;
#pragma unroll
        for (int e = 0; e < Tm::VEC; e += 4) {
          const int k = i * Tm::VEC + e;
          *reinterpret_cast<float4*>(t + e) = make_float4(fw[k], fw[k + 1], fw[k + 2], fw[k + 3]);
          *reinterpret_cast<float4*>(t + a.cols + e) = make_float4(fb[k], fb[k + 1], fb[k + 2], fb[k + 3]);
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < Tm::VEC; ++e) out.put(a.cols, c + e, fw[i * Tm::VEC + e], fb[i * Tm::VEC + e]);
    }
  } else {
    // the teams of a warp, then the warps in order (one warp after the other into the same place: 30000 rows of 512, 24.5 us
    // in the place of 19.7)
#pragma unroll
    for (int k = 0; k < E; ++k)
#pragma unroll
      for (int off = Tm::TS; off < 32; off <<= 1) {
        fw[k] += __shfl_xor_sync(0xffffffffu, fw[k], off);
        fb[k] += __shfl_xor_sync(0xffffffffu, fb[k], off);
      }
    const int warp = threadIdx.x >> 5;
    float* own = red + warp * 2 * Tm::COLS;
    if ((threadIdx.x & 31) < Tm::TS) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = tm.column(i), k = i * Tm::VEC;
        if constexpr (Tm::VEC == 8) {
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<float4*>(own + c + e) = make_float4(fw[k + e], fw[k + e + 1], fw[k + e + 2], fw[k + e + 3]);
            *reinterpret_cast<float4*>(own + Tm::COLS + c + e) = make_float4(fb[k + e], fb[k + e + 1], fb[k + e + 2], fb[k + e + 3]);
          }
        } else {
          own[c] = fw[k];
          own[Tm::COLS + c] = fb[k];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.cols; c += Tm::MAXB) {
      float w0 = red[c], b0 = red[Tm::COLS + c];
#pragma unroll
      for (int n = 1; n < WARPS; ++n) {
        w0 += red[n * 2 * Tm::COLS + c];
        b0 += red[(n * 2 + 1) * Tm::COLS + c];
      }
      out.put(a.cols, c, w0, b0);
    }
  }
}

// out[j] = sum over terms of partials[term][j], j < 2 cols.  A CTA owns eight columns (a sector of each term), 32 threads
// of each add a contiguous range of the terms (eight loads in flight), and their sums are added in a fixed tree.  With 32
// columns a CTA and eight threads for each the chain of loads took 9 us at 444 terms of 256 columns.
__global__ void __launch_bounds__(256) norm_fold_kernel(const float* __restrict__ partials, int terms, int cols, ParamOut dw,
                                                        ParamOut db) {
  griddep_wait();
  __shared__ float red[8][8];
  const int lane = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int j = blockIdx.x * 8 + lane;
  const int per = (terms + 31) / 32, k0 = g * per, k1 = min(terms, k0 + per);
  const bool on = j < 2 * cols;
  float s = 0.f;
  for (int k = k0; k < k1; k += 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = on && k + u < k1 ? partials[(int64_t)(k + u) * 2 * cols + j] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
  s += __shfl_xor_sync(0xffffffffu, s, 8);
  s += __shfl_xor_sync(0xffffffffu, s, 16);
  if ((threadIdx.x & 31) < 8) red[threadIdx.x >> 5][lane] = s;
  __syncthreads();
  if (threadIdx.x < 8 && on) {
    s = red[0][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += red[w][lane];
    const ParamOut& out = j < cols ? dw : db;
    if (out.p != nullptr) param_put(out, j < cols ? j : j - cols, s);
  }
}

constexpr int kMaxCtasPerSm = 8;  // each leaves a term of the parameter gradients

struct BwdLaunch {
  const NormArgs& a;
  const NormGrads& g;
  float* partials;
  cudaStream_t stream;
  // The team for rows of `cols` elements.  vec: eight elements at a time are possible.  Sixteen elements a thread in narrow
  // rows, where the sums over a team and what is done once a row weigh most (66049 rows of 96 fp32 channels: 15.9 us, 18.3
  // with eight); eight from 512 to 1024 columns (4099 rows of 1024 from codes: 12.5 us, 21.7 with sixteen, 16.4 with a warp
  // a row).
  template <typename T>
  int by_width(int cols, bool vec) const {
    if (vec) {
      if (cols <= 32) return run<T, Team<8, 4, 1>>();
      if (cols <= 64) return run<T, Team<8, 4, 2>>();
      if (cols <= 128) return run<T, Team<8, 8, 2>>();
      if (cols <= 256) return run<T, Team<8, 16, 2>>();
      if (cols <= 512) return run<T, Team<8, 32, 2>>();
      if (cols <= 1024) return run<T, Team<8, 0, 1, 128>>();
      if (cols <= 4096) return run<T, Team<8, 0, 2, 256>>();
      return run<T, Team<8, 0, 4, 256>>();
    }
    // (as in the forward; 16 elements a lane have no registers here: 300000 rows of 60: 40 us, 83 with a warp and four elements a
    // lane, 64 with four lanes)
    if (cols <= 32) return run<T, Team<1, 4, 8>>();
    if (cols <= 64) return run<T, Team<1, 8, 8>>();
    if (cols <= 128) return run<T, Team<1, 16, 8>>();
    if (cols <= 256) return run<T, Team<1, 32, 8>>();
    if (cols <= 2048) return run<T, Team<1, 0, 8, 256>>();
    if (cols <= 4096) return run<T, Team<1, 0, 8, 512>>();
    return run<T, Team<1, 0, 16, 512>>();
  }
  template <typename T, class Tm>
  int run() const {
    return a.codes != nullptr ? go<T, Tm, true>() : go<T, Tm, false>();
  }
  template <typename T, class Tm, bool CODES>
  int go() const {
    constexpr int ROWS = rows_in_flight<T, Tm, true>();
    static PerDeviceInt regs;
    const auto kern = norm_bwd_kernel<T, Tm, ROWS, CODES>;
    const int threads = Tm::threads(a.cols);
    int fit = 1;
    if (int rc = resident_ctas(kern, threads, regs, &fit)) return rc;
    const int64_t want = (a.rows + Tm::TEAMS * ROWS - 1) / (Tm::TEAMS * ROWS);
    const int64_t most = (int64_t)(fit < kMaxCtasPerSm ? fit : kMaxCtasPerSm) * sm_count();
    const ParamOut dw{g.dweight, g.dweight_type}, db{g.dbias, g.dbias_type};
    // One CTA is done with two rounds before a second launch would be: 64 rows of 128 channels, in a graph, 4.3 us in the
    // place of 5.0 (128 rows 5.2 and 5.0), and a launch less for the host.
    const bool one = want <= 2;
    const int blocks = one ? 1 : (int)(want < most ? want : most);
    launch_kernel(kern, dim3(blocks), dim3(threads), 0, stream, a, static_cast<const T*>(g.dy), static_cast<T*>(g.dx),
                  SumsOut{one ? nullptr : partials, one ? dw : ParamOut{nullptr, 0}, one ? db : ParamOut{nullptr, 0}});
    TPF_LAUNCH_OK();
    if (partials == nullptr || one) return TPF_OK;
    return norm_fold(partials, blocks, a.cols, g.dweight, g.dweight_type, g.dbias, g.dbias_type, stream);
  }
};

}  // namespace

int norm_fold(const float* terms, int count, int cols, void* dweight, int dweight_type, void* dbias, int dbias_type,
              cudaStream_t stream) {
  launch_kernel(norm_fold_kernel, dim3((2 * cols + 7) / 8), dim3(256), 0, stream, terms, count, cols,
                ParamOut{dweight, dweight_type}, ParamOut{dbias, dbias_type});
  TPF_LAUNCH_OK();
  return TPF_OK;
}

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
  TPF_REQUIRE_ALIGNED16(workspace, "layer_norm_bwd", "workspace");
  const bool from_codes = c.codes != nullptr;
  const bool vec = c.cols % 8 == 0 && (from_codes ? (reinterpret_cast<uintptr_t>(c.codes) & 15) == 0
                                                  : rows_vec_ok(c.x, c.x_pitch, c.type)) &&
                   vec_ok(g.dy, c.type) && (g.dx == nullptr || vec_ok(g.dx, c.type));
  return by_type(BwdLaunch{a, g, params ? static_cast<float*>(workspace) : nullptr, stream}, c.type, a.cols, vec);
}

}  // namespace tpf

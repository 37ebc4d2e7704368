// Weight gradient of the normalised projection: dW[o][c] = sum_r d_out[r][o] y~[r][c], straight from what was kept of x.
//
// y~ = w xh~ + b is made on the way: a stage of the ring holds 64 rows of d_out (an MN-major operand as TMA brings it) and
// of the codes (or of x), eight warps turn the latter into bf16 rows in a second buffer (the other operand), and the
// products of up to 256 outputs and 128 or 256 columns are summed in TMEM over the rows of a CTA.  Rounding y~ to bf16 is
// what the tensor cores ask for; the forward rounded y the same way.  The rows are split over CTAs where there are fewer
// tiles than SMs; the splits' fp32 sums are added in order by a second kernel.
//
// With a kernel of its own for y~ and a plain product behind it, 768 * 768 rows of 128 channels to 512 outputs took 67 and
// 112 us: y~ was written and read once more.  The floor is the read of d_out and the codes, 682 MB, 104 us.
#include "tpf_gemm_host.cuh"
#include "tpf_layer_norm.cuh"
#include "tpf_norm_linear.cuh"

namespace tpf {

namespace {

__device__ int g_dw_status;

constexpr int kRows = 64;  // of a stage

template <int MT_, int BN_, bool CODES_>
struct DwConfig {
  static constexpr int MT = MT_, BN = BN_;  // tiles of 128 outputs, columns
  static constexpr bool CODES = CODES_;
  static constexpr int A_BYTES = MT * 128 * kRows * 2, RAW_BYTES = BN * kRows * (CODES ? 1 : 2), B_BYTES = BN * kRows * 2;
  static constexpr int STAGE = A_BYTES + RAW_BYTES;
  static constexpr int STAGES = (224 * 1024 - 2 * B_BYTES) / STAGE > 5 ? 5 : (224 * 1024 - 2 * B_BYTES) / STAGE;
  static constexpr int SMEM = STAGES * STAGE + 2 * B_BYTES + 2048;
  static constexpr int TMEM_COLS = MT * BN;
  static constexpr int WARPS = 10;  // TMA, UMMA, eight that make y~ and write the sums
  static_assert(8 * kBlockStaging <= STAGES * STAGE, "");
  static_assert(STAGES >= 2 && TMEM_COLS >= 128 && TMEM_COLS <= 512, "");
};

struct DwArgs {
  NormArgs norm;
  int64_t rows_per_split;
  int outs, splits;
  float* part;    // [splits][outs][cols], or nullptr where there is one split:
  ParamOut out;   // [outs][cols]
};

template <class Cfg>
__global__ void __launch_bounds__(32 * Cfg::WARPS, 1)
    dw_kernel(const __grid_constant__ CUtensorMap tm_d, const __grid_constant__ CUtensorMap tm_x, const DwArgs a,
              int* __restrict__ status) {
  constexpr int MT = Cfg::MT, BN = Cfg::BN, STAGES = Cfg::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_dyn[];
  uint8_t* smem = smem_dyn + ((1024u - (smem_u32(smem_dyn) & 1023u)) & 1023u);
  uint8_t* b_buf = smem + STAGES * Cfg::STAGE;
  __shared__ uint64_t full[STAGES], empty[STAGES], b_full[2], b_empty[2], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const WaitCtx wctx{&abort_flag, status};
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 9);  // the UMMAs that read d_out, the eight warps that read the kept rows
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&b_full[b], 8);
      mbar_init(&b_empty[b], 1);
    }
    mbar_init(&done, 1);
    abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_d);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();

  const int m0 = blockIdx.x * (MT * 128), n0 = blockIdx.y * BN;
  const int64_t row_begin = (int64_t)blockIdx.z * a.rows_per_split;
  const int64_t row_end = min(a.norm.rows, row_begin + a.rows_per_split);
  const int steps = (int)((row_end - row_begin + kRows - 1) / kRows);

  if (warp == 0) {
    const uint32_t el = elect_one();
    int s = 0;
    uint32_t ph = 1;
    for (int k = 0; k < steps; ++k) {
      warp_wait(&empty[s], ph, wctx);
      mbar_expect_tx(el, &full[s], Cfg::STAGE);
      uint8_t* dst = smem + s * Cfg::STAGE;
      const int row = (int)(row_begin + (int64_t)k * kRows);
#pragma unroll
      for (int c = 0; c < MT * 2; ++c) tma_load_3d(el, dst + c * (kRows * 128), &tm_d, &full[s], m0 + c * 64, row, 0);
      if constexpr (Cfg::CODES) {
        tma_load_3d(el, dst + Cfg::A_BYTES, &tm_x, &full[s], n0, row, 0);
      } else {
#pragma unroll
        for (int c = 0; c < BN / 64; ++c)
          tma_load_3d(el, dst + Cfg::A_BYTES + c * (kRows * 128), &tm_x, &full[s], n0 + c * 64, row, 0);
      }
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_one();
    const int n = min(BN, (a.norm.cols - n0 + 15) / 16 * 16);
    const uint32_t idesc = make_idesc_bf16(128, n, true, true);
    const uint64_t a_desc = make_smem_desc(smem_u32(smem), kRows * 128, 8 * 128, swizzle_mode_for_bytes(128));
    const uint64_t b_desc = make_smem_desc(smem_u32(b_buf), kRows * 128, 8 * 128, swizzle_mode_for_bytes(128));
    int s = 0;
    uint32_t ph = 0;
    for (int k = 0; k < steps; ++k) {
      const int b = k & 1;
      warp_wait2(&full[s], ph, &b_full[b], (k >> 1) & 1, wctx);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint64_t ad = a_desc + ((s * Cfg::STAGE + i * (128 * kRows * 2)) >> 4);
        const uint64_t bd = b_desc + ((b * Cfg::B_BYTES) >> 4);
#pragma unroll
        for (int j = 0; j < kRows / 16; ++j)
          umma_ss(el, tmem + i * BN, ad + j * (16 * 128 >> 4), bd + j * (16 * 128 >> 4), idesc, (k | j) != 0 ? 1u : 0u);
      }
      umma_commit(el, &empty[s]);
      umma_commit(el, &b_empty[b]);
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
    umma_commit(el, &done);
  } else {
    // A lane makes 16 consecutive columns of a row at a time: 8 lanes (BN = 128) or 16 (256) a row.
    constexpr int LPR = BN / 16, RPW = 32 / LPR, PASSES = kRows / 8 / RPW;
    const int w8 = warp - 2, piece = lane % LPR, sub = lane / LPR;
    const int col = n0 + piece * 16;
    uint64_t g[8], bias[8];
    {
      float f[16], h[16];
      param_load<16, 1>(a.norm.w, col, a.norm.cols, 1.f, f);
      param_load<16, 1>(a.norm.b, col, a.norm.cols, 0.f, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] = f2_pack(f[2 * e], f[2 * e + 1]);
        bias[e] = f2_pack(h[2 * e], h[2 * e + 1]);
      }
    }
    const int group = min(col, a.norm.cols - 1) / kGroup;
    // statistics of the rows, one stage ahead
    float mean[PASSES], rstd[PASSES], down[PASSES];
    auto stats = [&](int k) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int64_t row = min(row_begin + (int64_t)k * kRows + w8 * 8 + p * RPW + sub, a.norm.rows - 1);
        mean[p] = a.norm.mean[row];
        rstd[p] = a.norm.rstd[row];
        down[p] = Cfg::CODES ? a.norm.scales[row * a.norm.groups + group] : 1.f;
      }
    };
    stats(0);
    int s = 0;
    uint32_t ph = 0;
    for (int k = 0; k < steps; ++k) {
      const int b = k & 1;
      uint64_t f2[PASSES], m2[PASSES];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        f2[p] = f2_dup(Cfg::CODES ? down[p] * rstd[p] : rstd[p]);
        m2[p] = f2_dup(Cfg::CODES ? -mean[p] * rstd[p] : -mean[p]);
      }
      if (k + 1 < steps) stats(k + 1);
      warp_wait2(&full[s], ph, &b_empty[b], ((k >> 1) & 1) ^ 1, wctx);
      const uint8_t* raw = smem + s * Cfg::STAGE + Cfg::A_BYTES;
      uint8_t* dst = b_buf + b * Cfg::B_BYTES + (piece >> 2) * (kRows * 128);
      uint4 u[PASSES][Cfg::CODES ? 1 : 2];
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int r = w8 * 8 + p * RPW + sub;
        if constexpr (Cfg::CODES) {
          u[p][0] = *reinterpret_cast<const uint4*>(raw + r * BN + piece * 16);
        } else {
          const uint4* src = reinterpret_cast<const uint4*>(raw + (piece >> 2) * (kRows * 128) + r * 128 + (piece & 3) * 32);
          u[p][0] = src[0];
          u[p][1] = src[1];
        }
      }
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int r = w8 * 8 + p * RPW + sub;
        uint64_t x[8];
        if constexpr (Cfg::CODES) {
          unpack_codes(u[p][0].x, x);
          unpack_codes(u[p][0].y, x + 2);
          unpack_codes(u[p][0].z, x + 4);
          unpack_codes(u[p][0].w, x + 6);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = f2_fma(x[e], f2[p], m2[p]);
        } else {
          const uint32_t v[8] = {u[p][0].x, u[p][0].y, u[p][0].z, u[p][0].w, u[p][1].x, u[p][1].y, u[p][1].z, u[p][1].w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[e] = f2_mul(f2_add(f2_pack_bits(v[e] << 16, v[e] & 0xffff0000u), m2[p]), f2[p]);
        }
        uint32_t o[8];
        const bool live = row_begin + (int64_t)k * kRows + r < row_end;  // (rows of the next split meet d_out, not zeros)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float lo, hi;
          f2_unpack(f2_fma(x[e], g[e], bias[e]), lo, hi);
          o[e] = live ? pack_bf16x2(lo, hi) : 0u;
        }
        uint8_t* row = dst + r * 128;
        const int q = (piece & 3) * 2, sw = r & 7;
        *reinterpret_cast<uint4*>(row + ((q ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(row + (((q + 1) ^ sw) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&b_full[b]);
        mbar_arrive(&empty[s]);
      }
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
    // the sums: two warps a lane quarter, which share the tiles or the columns
    warp_wait(&done, 0, wctx);
    tc_fence_after();
    const int quarter = warp & 3, half = w8 >> 2;
    constexpr int COLS = MT == 2 ? BN : BN / 2;  // of a warp
    const int o = m0 + (MT == 2 ? half * 128 : 0) + quarter * 32;  // first output of the warp
    const int first = MT == 2 ? 0 : half * COLS;
    const uint32_t t = tmem_addr(tmem, quarter * 32, (MT == 2 ? half * BN : 0) + first);
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32) {
      if (n0 + first + c >= a.norm.cols) break;
      uint32_t v[32];
      tmem_ld32(t + c, v);
      tmem_ld_wait();
      const int64_t at = (int64_t)o * a.norm.cols + n0 + first + c;
      const int left = a.norm.cols - (n0 + first + c);
      float* p = a.part + (int64_t)blockIdx.z * a.outs * a.norm.cols + at;
      // (the stages are all used up)
      put_block(smem + w8 * kBlockStaging, v, lane, [&](int r, int e, const float4& x) {
        if (o + r >= a.outs || e >= left) return;
        if (a.part != nullptr) *reinterpret_cast<float4*>(p + (int64_t)r * a.norm.cols + e) = x;
        else param_put4(a.out, at + (int64_t)r * a.norm.cols + e, x);
      });
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// out[i] = sum over the splits, in order; four elements a thread, eight loads in flight.  (Rows are split only where there
// are fewer tiles than SMs, and narrow rows are another kernel's, so there are few splits of many elements.)
__global__ void __launch_bounds__(256) dw_fold_kernel(const float* __restrict__ part, int splits, int64_t n, ParamOut out) {
  griddep_wait();
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; k += 8) {
    float4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      v[u] = k + u < splits ? *reinterpret_cast<const float4*>(part + (k + u) * n + i) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      s.x += v[u].x;
      s.y += v[u].y;
      s.z += v[u].z;
      s.w += v[u].w;
    }
  }
  param_put4(out, i, s);
}

struct DwPlan {
  int mt, bn, tiles_m, tiles_n, splits;
  int64_t rows_per_split;
};
DwPlan dw_plan(int64_t rows, int64_t cols, int64_t outs) {
  DwPlan p;
  p.mt = outs > 128 ? 2 : 1;
  p.bn = cols > 128 ? 256 : 128;
  p.tiles_m = (int)((outs + p.mt * 128 - 1) / (p.mt * 128));
  p.tiles_n = (int)((cols + p.bn - 1) / p.bn);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  int64_t splits = sm_count() / tiles;
  if (splits < 1) splits = 1;
  // a split has 512 rows at least: its sums are written and read once more
  const int64_t most = rows > 0 ? (rows + 511) / 512 : 1;
  if (splits > most) splits = most;
  p.rows_per_split = ((rows + splits - 1) / splits + kRows - 1) / kRows * kRows;
  p.splits = rows > 0 ? (int)((rows + p.rows_per_split - 1) / p.rows_per_split) : 1;
  return p;
}

template <int MT, int BN, bool CODES>
int dw_launch(const DwArgs& a, const DwPlan& p, const void* d_out, cudaStream_t stream) {
  using Cfg = DwConfig<MT, BN, CODES>;
  CUtensorMap tm_d, tm_x;
  if (int rc = make_operand_tmap(&tm_d, d_out, true, a.outs, a.norm.rows, a.outs, 1, 0, 128, 64, kRows)) return rc;
  if constexpr (CODES) {
    const uint64_t dims[3] = {(uint64_t)a.norm.code_pitch, (uint64_t)a.norm.rows, 1};
    const uint64_t strides[2] = {(uint64_t)a.norm.code_pitch, 16};
    const uint32_t box[3] = {(uint32_t)BN, (uint32_t)kRows, 1};
    if (int rc = make_tmap(&tm_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.norm.codes, 3, dims, strides, box, 0)) return rc;
  } else {
    const uint64_t dims[3] = {(uint64_t)a.norm.cols, (uint64_t)a.norm.rows, 1};
    const uint64_t strides[2] = {(uint64_t)a.norm.x_pitch * 2, 16};
    const uint32_t box[3] = {64, (uint32_t)kRows, 1};
    if (int rc = make_tmap_bf16(&tm_x, a.norm.x, 3, dims, strides, box, 0)) return rc;
  }
  int* status = nullptr;
  static PerDeviceAddress status_at;
  if (int rc = device_symbol_address(g_dw_status, status_at, reinterpret_cast<void**>(&status))) return rc;
  const auto kern = dw_kernel<Cfg>;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(kern, Cfg::SMEM, once)) return rc;
  launch_kernel(kern, dim3(p.tiles_m, p.tiles_n, p.splits), dim3(32 * Cfg::WARPS), Cfg::SMEM, stream, tm_d, tm_x, a, status);
  TPF_LAUNCH_OK();
  if (a.part == nullptr) return TPF_OK;
  const int64_t n = (int64_t)a.outs * a.norm.cols;
  TPF_REQUIRE(n / 1024 < (1ll << 31) - 1, TPF_ERR_UNSUPPORTED, "norm_linear: extent too large");
  launch_kernel(dw_fold_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream, a.part, p.splits, n, a.out);
  TPF_LAUNCH_OK();
  return TPF_OK;
}

}  // namespace

int norm_linear_dw_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  TPF_CUDA_OK(cudaMemcpyFromSymbol(&v, g_dw_status, sizeof(int)));
  if (v) TPF_CUDA_OK(cudaMemcpyToSymbol(g_dw_status, &zero, sizeof(int)));
  *out = v;
  return TPF_OK;
}

int64_t norm_linear_dw_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  const DwPlan p = dw_plan(rows, cols, outs);
  return p.splits > 1 ? p.splits * outs * cols * 4 : 0;
}

int norm_linear_dw(const NormArgs& norm, const void* d_out, int64_t outs, void* dw, int dw_type, void* workspace,
                   cudaStream_t stream) {
  const DwPlan p = dw_plan(norm.rows, norm.cols, outs);
  TPF_REQUIRE(p.splits <= 65535 && p.tiles_n <= 65535, TPF_ERR_UNSUPPORTED, "norm_linear: extent too large");
  const DwArgs a{norm, p.rows_per_split, (int)outs, p.splits, p.splits > 1 ? static_cast<float*>(workspace) : nullptr,
                 {dw, dw_type}};
  const bool codes = norm.codes != nullptr;
  if (p.mt == 2 && p.bn == 256) return codes ? dw_launch<2, 256, true>(a, p, d_out, stream) : dw_launch<2, 256, false>(a, p, d_out, stream);
  if (p.mt == 2) return codes ? dw_launch<2, 128, true>(a, p, d_out, stream) : dw_launch<2, 128, false>(a, p, d_out, stream);
  // (128 outputs or fewer and 128 columns or fewer are a narrow projection)
  TPF_REQUIRE(p.bn == 256, TPF_ERR_UNSUPPORTED, "norm_linear: a narrow projection");
  return codes ? dw_launch<1, 256, true>(a, p, d_out, stream) : dw_launch<1, 256, false>(a, p, d_out, stream);
}

}  // namespace tpf

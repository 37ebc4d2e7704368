// Forward of the normalised projection for narrow rows (up to 128 columns, a weight that stays in shared memory) and for a
// few rows.
//
// Narrow rows: a tile of 128 rows of x comes by TMA in the layout of a K-major operand, some warps normalise it where it
// lies (and write its codes, scales and statistics), the products with the resident weight go to TMEM, 128 outputs at a
// time, and eight other warps store them.  x is read and out written once; y never leaves the SM.  As two kernels
// 768 * 768 rows of 128 channels to 512 outputs, with codes, took 195 us, with y written and read in between; this takes
// 143, the floor is 833 MB, 127.
#include "tpf_gemm_host.cuh"
#include "tpf_norm_linear.cuh"

namespace tpf {

namespace {

__device__ int g_nl_fwd_status;

// Warps that normalise and warps that store.  With few outputs a tile waits for the former, with many for the latter, which
// sixteen normalising warps keep from issuing (16 and 4 / 8 and 8, us: 500000 rows of 128 to 128 outputs 72 / 90, 262144 to
// 256 50 / 57, 589824 to 512 166 / 143).
template <int NORM_, int STORE_>
struct Split {
  static constexpr int NORM = NORM_, STORE = STORE_, WARPS = 2 + NORM + STORE;
  static constexpr int STAGING = STORE * kTmaTiles;
};
constexpr int kBlock = 128 * 128;           // 128 rows of 64 bf16 columns
constexpr int kWBytes = 128 * 1024;         // most of the weight
constexpr int kSharedBytes = 2048;           // barriers; from 1024 on the norm's weight and bias
constexpr int kSmem = 227 * 1024;
static_assert(kSharedBytes + kWBytes + Split<8, 8>::STAGING + 2 * 2 * kBlock <= kSmem, "");

struct FwdArgs {
  NormArgs norm;  // codes, scales, mean and rstd are written where they are not nullptr
  float eps;
  int outs, tiles, w_rows;  // w_rows: outs rounded up to 64
  int stages;               // tiles of x that shared memory holds
};

struct Shared {
  uint64_t full[4], ready[4], empty[4], acc_full[4], acc_empty[4], w_full;
  uint32_t tmem;
  volatile int abort_flag;
};
static_assert(sizeof(Shared) <= 1024, "");

template <bool KEEP, int CB, class Warps>
__global__ void __launch_bounds__(32 * Warps::WARPS, 1)
    nl_fwd_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                  const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ FwdArgs a, int* __restrict__ status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int cb = CB, x_bytes = CB * kBlock, kNormWarps = Warps::NORM, kStoreWarps = Warps::STORE;
  uint8_t* w_buf = smem;
  uint8_t* ring = smem + a.w_rows * cb * 128;
  uint8_t* staging = ring + a.stages * x_bytes;
  Shared* sh = reinterpret_cast<Shared*>(smem + kSmem - kSharedBytes);
  const WaitCtx wctx{&sh->abort_flag, status};
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < 4; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->ready[s], kNormWarps);
      mbar_init(&sh->empty[s], 1);
      mbar_init(&sh->acc_full[s], 1);
      mbar_init(&sh->acc_empty[s], kStoreWarps);
    }
    mbar_init(&sh->w_full, 1);
    sh->abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_out);
  }
  if (warp == 1) {
    tmem_alloc(&sh->tmem, 512);
    tmem_relinquish();
  }
  griddep_wait();
  float* params = reinterpret_cast<float*>(smem + kSmem - kSharedBytes + 1024);  // weight, bias
  if (threadIdx.x < 256) {
    const int i = threadIdx.x & 127;
    param_load<1, 1>(threadIdx.x < 128 ? a.norm.w : a.norm.b, i, a.norm.cols, threadIdx.x < 128 ? 1.f : 0.f, params + threadIdx.x);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem;
  const int count = (a.tiles - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // tiles of this CTA
  const int chunks = (a.outs + 127) / 128;

  if (warp == 0) {
    const uint32_t el = elect_one();
    int s = 0;
    uint32_t ph = 1;
    for (int t = 0; t < count; ++t) {
      warp_wait(&sh->empty[s], ph, wctx);
      mbar_expect_tx(el, &sh->full[s], x_bytes);
      const int row = ((int)blockIdx.x + t * (int)gridDim.x) * 128;
      for (int c = 0; c < cb; ++c) tma_load_3d(el, ring + s * x_bytes + c * kBlock, &tm_x, &sh->full[s], c * 64, row, 0);
      if (t == 0) {  // the first tile is normalised meanwhile
        mbar_expect_tx(el, &sh->w_full, a.w_rows * cb * 128);
        for (int c = 0; c < cb; ++c)
          for (int o = 0; o < a.w_rows; o += 64)
            tma_load_3d(el, w_buf + (c * a.w_rows + o) * 128, &tm_w, &sh->w_full, c * 64, o, 0);
      }
      if (++s == a.stages) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_one();
    const uint64_t a_desc = make_smem_desc(smem_u32(ring), 16, 1024, swizzle_mode_for_bytes(128));
    const uint64_t b_desc = make_smem_desc(smem_u32(w_buf), 16, 1024, swizzle_mode_for_bytes(128));
    const int steps = (a.norm.cols + 15) / 16;  // of 16 columns
    warp_wait(&sh->w_full, 0, wctx);
    int s = 0, acc = 0;
    uint32_t ph = 0, acc_ph = 1;
    for (int t = 0; t < count; ++t) {
      warp_wait(&sh->ready[s], ph, wctx);
      for (int j = 0; j < chunks; ++j) {
        warp_wait(&sh->acc_empty[acc], acc_ph, wctx);
        tc_fence_after();
        const uint32_t idesc = make_idesc_bf16(128, min(128, a.w_rows - j * 128), false, false);
        for (int k = 0; k < steps; ++k) {
          const uint64_t ad = a_desc + ((s * x_bytes + (k >> 2) * kBlock + (k & 3) * 32) >> 4);
          const uint64_t bd = b_desc + ((((k >> 2) * a.w_rows + j * 128) * 128 + (k & 3) * 32) >> 4);
          umma_ss(el, tmem + acc * 128, ad, bd, idesc, k != 0 ? 1u : 0u);
        }
        umma_commit(el, &sh->acc_full[acc]);
        if (++acc == 4) {
          acc = 0;
          acc_ph ^= 1;
        }
      }
      umma_commit(el, &sh->empty[s]);
      if (++s == a.stages) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp < 2 + kNormWarps) {
    // Eight lanes a row, eight columns of each block of 64, four rows side by side.  (With 16 lanes a row the sums took a
    // step more, and what is done once a row weighed twice as much: 64 columns 54.7 us at 262144 rows and 256 outputs.)
    constexpr int P = 4 * CB, ROWS = 128 / kNormWarps, U = 2;
    const int wn = warp - 2, piece = lane & 7, sub = lane >> 3;
    bool on[CB];
#pragma unroll
    for (int i = 0; i < CB; ++i) on[i] = i * 64 + piece * 8 < a.norm.cols;
    int s = 0;
    uint32_t ph = 0;
    for (int t = 0; t < count; ++t) {
      const int64_t row0 = (int64_t)((int)blockIdx.x + t * (int)gridDim.x) * 128 + wn * ROWS;
      uint8_t* tile = ring + s * x_bytes + wn * ROWS * 128;
      const int left = (int)(a.norm.rows - row0 < ROWS ? a.norm.rows - row0 : ROWS);  // rows that exist
      warp_wait(&sh->full[s], ph, wctx);
#pragma unroll 1
      for (int r0 = 0; r0 < ROWS; r0 += 4 * U) {
        uint64_t x[U][P];
        float sum[U], mean[U], amax[U];
        uint8_t* at[U];  // of the lane's piece in the first block
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * 4 + sub;
          at[u] = tile + r * 128 + ((piece ^ (r & 7)) << 4);
          Piece<bf16, 8> raw[CB];
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            raw[i].load(reinterpret_cast<const bf16*>(at[u] + i * kBlock));
            if (!on[i]) raw[i].zero();
          }
          uint64_t q = 0;
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            float f[8];
            raw[i].get(f);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[u][i * 4 + e] = f2_pack(f[2 * e], f[2 * e + 1]);
              q = f2_add(q, x[u][i * 4 + e]);
            }
          }
          sum[u] = f2_sum(q);
          if constexpr (KEEP) amax[u] = CB == 2 ? max_nan(raw[0].amax(), raw[CB - 1].amax()) : raw[0].amax();
        }
        if (KEEP && a.norm.codes != nullptr) {
#pragma unroll
          for (int off = 4; off > 0; off >>= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) amax[u] = max_nan(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], off));
          float up[U];
          const float down = group_scales<U, 8>(amax, up);
          int8_t* codes = a.norm.codes + (row0 + r0) * a.norm.code_pitch + piece * 8;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int r = u * 4 + sub;
            const uint64_t f = f2_dup(up[u]);
            const bool good = up[u] == up[u];
#pragma unroll
            for (int i = 0; i < CB; ++i)
              if (r0 + r < left && on[i])
                *reinterpret_cast<uint2*>(codes + r * a.norm.code_pitch + i * 64) =
                    make_uint2(pack_codes(x[u][4 * i], x[u][4 * i + 1], f, good),
                               pack_codes(x[u][4 * i + 2], x[u][4 * i + 3], f, good));
          }
          const int r = r0 + piece * 4 + sub;  // lane n of a row's has the scale of its n-th row
          if (piece < U && r < left) a.norm.scales[row0 + r] = down;
        }
        warp_sum(sum, 8);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          mean[u] = sum[u] * a.norm.inv_cols;
          const uint64_t m = f2_dup(-mean[u]);
          uint64_t q = 0;
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            if (!on[i]) continue;  // (its values stay zeros)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[u][i * 4 + e] = f2_add(x[u][i * 4 + e], m);
              q = f2_fma(x[u][i * 4 + e], x[u][i * 4 + e], q);
            }
          }
          sum[u] = f2_sum(q);
        }
        warp_sum(sum, 8);
        float rstd[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * 4 + sub;
          rstd[u] = rsqrtf(fmaf(sum[u], a.norm.inv_cols, a.eps));
          if (KEEP && piece == 0 && r < left) {
            a.norm.mean[row0 + r] = mean[u];
            a.norm.rstd[row0 + r] = rstd[u];
          }
        }
#pragma unroll
        for (int i = 0; i < CB; ++i) {
          if (!on[i]) continue;  // (columns behind the last: zeros, which is what TMA put there and the weight's rows have)
          uint64_t w[4], b[4];
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float* q = params + i * 64 + piece * 8 + 2 * e;
            const float4 f = *reinterpret_cast<const float4*>(q), h = *reinterpret_cast<const float4*>(q + 128);
            w[e] = f2_pack(f.x, f.y);
            w[e + 1] = f2_pack(f.z, f.w);
            b[e] = f2_pack(h.x, h.y);
            b[e + 1] = f2_pack(h.z, h.w);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint64_t rs = f2_dup(rstd[u]);
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float lo, hi;
              f2_unpack(f2_fma(f2_mul(x[u][i * 4 + e], rs), w[e], b[e]), lo, hi);
              o[e] = pack_bf16x2(lo, hi);
            }
            *reinterpret_cast<uint4*>(at[u] + i * kBlock) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->ready[s]);
      if (++s == a.stages) {
        s = 0;
        ph ^= 1;
      }
    }
  } else {
    // two warps a lane quarter, which take turns with the blocks of 32 outputs
    const int ws = warp - 2 - kNormWarps, quarter = warp & 3;
    uint8_t* tiles = staging + ws * kTmaTiles;
    int buf = 0, acc = 0;
    uint32_t ph = 0;
    for (int t = 0; t < count; ++t) {
      const int row = ((int)blockIdx.x + t * (int)gridDim.x) * 128 + quarter * 32;
      for (int j = 0; j < chunks; ++j) {
        warp_wait(&sh->acc_full[acc], ph, wctx);
        tc_fence_after();
        const int n = min(128, a.outs - j * 128);
        // two blocks of 32 outputs at a time
        constexpr int GROUPS = kStoreWarps / 4, ROUNDS = 2 / GROUPS;
#pragma unroll
        for (int q = 0; q < ROUNDS; ++q) {
          uint32_t v[2][32];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = ((ws >> 2) + GROUPS * (2 * q + i)) * 32;
            if (col < n) tmem_ld32(tmem_addr(tmem, quarter * 32, acc * 128 + col), v[i]);
          }
          tmem_ld_wait();
          if (q == ROUNDS - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->acc_empty[acc]);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int col = ((ws >> 2) + GROUPS * (2 * q + i)) * 32;
            if (col >= n) continue;
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = pack_bf16x2(__uint_as_float(v[i][2 * e]), __uint_as_float(v[i][2 * e + 1]));
            warp_tile_store_tma<2>(tiles, buf, lane, pk, &tm_out, j * 128 + col, row, 0);
          }
        }
        if (++acc == 4) {
          acc = 0;
          ph ^= 1;
        }
      }
    }
    bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

// A few rows (a token at a time): every CTA normalises the rows for itself, in shared memory, and its warps take one output
// after the other: a lane multiplies eight columns of W at a time with those of all rows.  The first CTA writes what is kept
// for a backward.  Bound by latency: one launch in the place of two, and the weight's rows spread over as many SMs as there
// are.  y stays in fp32: nothing here asks for less.  A call with one row of 128 channels and 512 outputs takes 6.6 us in the
// place of 10.5.
constexpr int kFewRows = 4, kFewWarps = 8;
__global__ void __launch_bounds__(32 * kFewWarps) nl_few_kernel(const NormArgs a, float eps, const bf16* __restrict__ w, int outs,
                                                               int outs_per_warp, bf16* __restrict__ out) {
  griddep_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  float* y = reinterpret_cast<float*>(smem);  // [rows][cols]
  const int warp = warp_index(), lane = threadIdx.x & 31, pieces = a.cols / 8;
  if (warp < a.rows) {  // a warp normalises a row, in three passes over it (L1 has it after the first)
    const bf16* x = static_cast<const bf16*>(a.x) + warp * a.x_pitch;
    float s[1] = {0.f};
    for (int p = lane; p < pieces; p += 32) {
      Piece<bf16, 8> v;
      v.load(x + p * 8);
      float f[8];
      v.get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += f[e];
    }
    warp_sum(s);
    const float mean = s[0] * a.inv_cols;
    s[0] = 0.f;
    for (int p = lane; p < pieces; p += 32) {
      Piece<bf16, 8> v;
      v.load(x + p * 8);
      float f[8];
      v.get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] = fmaf(f[e] - mean, f[e] - mean, s[0]);
    }
    warp_sum(s);
    const float rstd = rsqrtf(fmaf(s[0], a.inv_cols, eps));
    if (blockIdx.x == 0 && a.mean != nullptr && lane == 0) {
      a.mean[warp] = mean;
      a.rstd[warp] = rstd;
    }
    if (blockIdx.x == 0 && a.codes != nullptr) {
      for (int p0 = 0; p0 < pieces; p0 += 32) {  // 16 lanes a group of 128
        const int p = p0 + lane;
        Piece<bf16, 8> v;
        v.zero();
        if (p < pieces) v.load(x + p * 8);
        float amax = v.amax();
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, off));
        const GroupScale q = group_scale(amax);
        const uint64_t up = f2_dup(q.up);
        float f[8];
        v.get(f);
        const uint2 codes = make_uint2(pack_codes(f2_pack(f[0], f[1]), f2_pack(f[2], f[3]), up, q.up == q.up),
                                       pack_codes(f2_pack(f[4], f[5]), f2_pack(f[6], f[7]), up, q.up == q.up));
        if (p < pieces) {
          *reinterpret_cast<uint2*>(a.codes + warp * a.code_pitch + p * 8) = codes;
          if ((lane & 15) == 0) a.scales[warp * a.groups + p / 16] = q.down;
        }
      }
    }
    for (int p = lane; p < pieces; p += 32) {
      Piece<bf16, 8> v;
      v.load(x + p * 8);
      float f[8], g[8], b[8];
      v.get(f);
      param_load<8, 1>(a.w, p * 8, a.cols, 1.f, g);
      param_load<8, 1>(a.b, p * 8, a.cols, 0.f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fmaf((f[e] - mean) * rstd, g[e], b[e]);
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<float4*>(y + warp * a.cols + p * 8 + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    }
  }
  __syncthreads();
  const int rows = (int)a.rows;
  const int o0 = (blockIdx.x * kFewWarps + warp) * outs_per_warp;
  for (int o = o0; o < min(outs, o0 + outs_per_warp); ++o) {
    float s[kFewRows] = {};
    for (int p = lane; p < pieces; p += 32) {
      Piece<bf16, 8> v;
      v.load(w + (int64_t)o * a.cols + p * 8);
      float f[8];
      v.get(f);
#pragma unroll
      for (int r = 0; r < kFewRows; ++r) {
        if (r < rows) {
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float4 h = *reinterpret_cast<const float4*>(y + r * a.cols + p * 8 + e);
            s[r] = fmaf(f[e], h.x, s[r]);
            s[r] = fmaf(f[e + 1], h.y, s[r]);
            s[r] = fmaf(f[e + 2], h.z, s[r]);
            s[r] = fmaf(f[e + 3], h.w, s[r]);
          }
        }
      }
    }
    warp_sum(s);
#pragma unroll
    for (int r = 0; r < kFewRows; ++r)
      if (r < rows && lane == r) out[(int64_t)r * outs + o] = __float2bfloat16_rn(s[r]);
  }
}

}  // namespace

bool norm_linear_few(int64_t rows) { return rows <= kFewRows; }

int norm_linear_few_fwd(const NormArgs& norm, const void* w, int64_t outs, void* out, float eps, cudaStream_t stream) {
  const int64_t warps = (int64_t)sm_count() * 2 * kFewWarps;  // two CTAs an SM
  const int per = (int)((outs + warps - 1) / warps);
  const int smem = (int)norm.rows * norm.cols * 4;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(nl_few_kernel, kFewRows * (int)kMaxNormCols * 4, once)) return rc;
  launch_kernel(nl_few_kernel, dim3((unsigned)((outs + per * kFewWarps - 1) / (per * kFewWarps))), dim3(32 * kFewWarps), smem,
                stream, norm, eps, static_cast<const bf16*>(w), (int)outs, per, static_cast<bf16*>(out));
  TPF_LAUNCH_OK();
  return TPF_OK;
}

int norm_linear_fwd_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  TPF_CUDA_OK(cudaMemcpyFromSymbol(&v, g_nl_fwd_status, sizeof(int)));
  if (v) TPF_CUDA_OK(cudaMemcpyToSymbol(g_nl_fwd_status, &zero, sizeof(int)));
  *out = v;
  return TPF_OK;
}

int norm_linear_narrow_fwd(const NormArgs& norm, const void* w, int64_t outs, void* out, float eps, cudaStream_t stream) {
  const int64_t R = norm.rows, C = norm.cols;
  const int cb = (int)((C + 63) / 64), w_rows = (int)((outs + 63) / 64 * 64);
  const bool few_outs = outs <= 256;
  const int staging = few_outs ? Split<16, 4>::STAGING : Split<8, 8>::STAGING;
  int stages = (kSmem - kSharedBytes - staging - w_rows * cb * 128) / (cb * kBlock);
  if (stages > 4) stages = 4;
  const FwdArgs a{norm, eps, (int)outs, (int)((R + 127) / 128), w_rows, stages};
  CUtensorMap tm_x, tm_w, tm_out;
  if (int rc = make_operand_tmap(&tm_x, norm.x, false, R, C, norm.x_pitch, 1, 0, 128, 128, 64)) return rc;
  if (int rc = make_operand_tmap(&tm_w, w, false, outs, C, C, 1, 0, 128, 64, 64)) return rc;
  if (int rc = make_store_tmap(&tm_out, out, outs, R, outs, 1, 0)) return rc;
  int* status = nullptr;
  static PerDeviceAddress status_at;
  if (int rc = device_symbol_address(g_nl_fwd_status, status_at, reinterpret_cast<void**>(&status))) return rc;
  const int grid = a.tiles < sm_count() ? a.tiles : sm_count();
  const auto go = [&](auto kern, int warps, PerDeviceOnce& once) {
    if (int rc = ensure_dynamic_smem(kern, kSmem, once, 1024)) return rc;
    launch_kernel(kern, dim3(grid), dim3(32 * warps), kSmem, stream, tm_x, tm_w, tm_out, a, status);
    TPF_LAUNCH_OK();
    return (int)TPF_OK;
  };
  const auto by_split = [&](auto split, PerDeviceOnce* once) {
    using S = decltype(split);
    if (norm.mean != nullptr)
      return cb == 2 ? go(nl_fwd_kernel<true, 2, S>, S::WARPS, once[0]) : go(nl_fwd_kernel<true, 1, S>, S::WARPS, once[1]);
    return cb == 2 ? go(nl_fwd_kernel<false, 2, S>, S::WARPS, once[2]) : go(nl_fwd_kernel<false, 1, S>, S::WARPS, once[3]);
  };
  static PerDeviceOnce once[2][4];
  return few_outs ? by_split(Split<16, 4>{}, once[0]) : by_split(Split<8, 8>{}, once[1]);
}

}  // namespace tpf

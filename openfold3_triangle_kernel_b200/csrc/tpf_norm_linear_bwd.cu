// Backward of the normalised projection for narrow rows (up to 128 columns, a weight that stays in shared memory), in one
// kernel that reads d_out from memory once.
//
//   dx: dy = d_out W, then the layer norm's backward on the rows of dy while they are in TMEM
//   G = d_out^T xh~ and s = d_out^T 1, from what was kept of x
//
// The parameters' gradients all follow from G and s:
//   dW = G diag(w) + s b^T,   dw_c = sum_r dy_rc xh~_rc = sum_o W_oc G_oc,   db_c = sum_r dy_rc = sum_o W_oc s_o,
// so that nothing is summed over the rows of dy.  xh~ is rounded to bf16 for the tensor cores, sums are fp32.  That rounding is
// the one that the forward makes of y, and what a bf16 Linear's weight gradient has: dW and dw are off by 0.0016 of their norm
// (0.0023 with that of a bf16 parameter's gradient).  Without it, with xh~ as a sum of two bf16 operands, they are off by the
// last rounding only (0.0017) and the backward takes 235 us in the place of 230 from codes at 589824 rows, 128 -> 512, but 254 /
// 208 from whole rows and 129 / 96 at 500000 of 128 -> 128, where making the operand is what G waits for.  dw alone from
// dy and xh~ in fp32 (31 shuffles a warp and tile): 250 / 230, 219 / 209, 115 / 96; as tensor products of the two parts of dy xh~ with
// ones 263 / 230, 242 / 209, 115 / 96.
//
// Both products need the same d_out, one as rows and one as columns, and neither fits beside the other: G takes the whole
// of TMEM, W most of shared memory.  So CTAs of the two kinds work side by side through the same ranges of rows, and what
// one of them brought from memory the others find in L2.  A range has `tiles` CTAs for G (256 outputs each, or 128) and as
// many for dx (every tiles-th 128 rows).
#include "tpf_gemm_host.cuh"
#include "tpf_norm_linear.cuh"

namespace tpf {

namespace {

__device__ int g_nl_bwd_status;

constexpr int kRows = 64;         // of a stage of G
constexpr int kWorkers = 16;       // warps that work on elements
constexpr int kWarps = 3 + kWorkers;  // TMA, UMMA; last: TMA of the kept rows (dx)
constexpr int kChunk = kRows * 128;  // 64 rows of 64 bf16 columns
constexpr int kSmemMax = 227 * 1024;

struct BwdArgs {
  NormArgs norm;
  int64_t rows_per_range;
  int outs, g_ctas, dx_ctas;  // CTAs of a range (0: not wanted)
  int w_blocks;    // blocks of 64 outputs
  int col_blocks;  // blocks of 64 columns: 1 or 2
  int dx_stages, dx_kept;  // dx: blocks of d_out and tiles of kept rows that shared memory holds,
  int dx_width;            // columns of dx that a warp stages at a time: 32 or 16
  float* g;        // [ranges][outs][cols]
  float* s;        // [ranges][outs]
};

// Everything in dynamic shared memory, which then starts on a 1024-byte boundary.
struct Shared {
  uint64_t full[8], empty[8], second_full[2], second_empty[2], kept_full[2], kept_empty[2], w_full, done;
  uint32_t tmem;
  volatile int abort_flag;
};
constexpr int kSharedBytes = 1024;
static_assert(sizeof(Shared) <= 512, "");  // the other 512 bytes: the norm's weight

// ---- G and s -------------------------------------------------------------------------------------
template <int MT, bool CODES>
struct GradConfig {
  static constexpr int A_BYTES = MT * 2 * kChunk, RAW_BYTES = CODES ? kChunk : 2 * kChunk, STAGE = A_BYTES + RAW_BYTES;
  static constexpr int B_BYTES = 3 * kChunk;  // up to 128 columns of xh~, a block whose first column is ones
  static constexpr int FIT = (kSmemMax - kSharedBytes - 2 * B_BYTES) / STAGE, STAGES = FIT > 6 ? 6 : FIT;
  static constexpr int SMEM = kSharedBytes + 2 * B_BYTES + STAGES * STAGE;
  static_assert(kWorkers * kBlockStaging <= SMEM - kSharedBytes, "");
  static constexpr int TMEM = MT == 2 ? 512 : 256;  // 256 columns a tile: up to 144 are used
};

template <int MT, bool CODES>
__device__ __forceinline__ void grad_role(uint8_t* smem, Shared* sh, const WaitCtx& wctx, const CUtensorMap& tm_cols,
                                          const CUtensorMap& tm_x, const BwdArgs& a, int tile, int range) {
  using Cfg = GradConfig<MT, CODES>;
  constexpr int STAGES = Cfg::STAGES;
  uint8_t* b_buf = smem;
  uint8_t* ring = smem + 2 * Cfg::B_BYTES;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int m0 = tile * (MT * 128);
  const int64_t row_begin = range * a.rows_per_range;
  const int64_t row_end = min(a.norm.rows, row_begin + a.rows_per_range);
  const int steps = (int)((row_end - row_begin + kRows - 1) / kRows);
  const int ones = a.col_blocks;  // block of the ones

  if (warp == 0) {
    const uint32_t el = elect_one();
    int s = 0;
    uint32_t ph = 1;
    for (int k = 0; k < steps; ++k) {
      warp_wait(&sh->empty[s], ph, wctx);
      mbar_expect_tx(el, &sh->full[s], Cfg::STAGE);
      uint8_t* dst = ring + s * Cfg::STAGE;
      const int row = (int)(row_begin + (int64_t)k * kRows);
#pragma unroll
      for (int c = 0; c < MT * 2; ++c) tma_load_3d(el, dst + c * kChunk, &tm_cols, &sh->full[s], m0 + c * 64, row, 0);
#pragma unroll
      for (int c = 0; c < (CODES ? 1 : 2); ++c)
        tma_load_3d(el, dst + Cfg::A_BYTES + c * kChunk, &tm_x, &sh->full[s], c * 64, row, 0);
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_one();
    const uint32_t idesc = make_idesc_bf16(128, ones * 64 + 16, true, true);
    const uint64_t a_desc = make_smem_desc(smem_u32(ring), kChunk, 1024, swizzle_mode_for_bytes(128));
    const uint64_t b_desc = make_smem_desc(smem_u32(b_buf), kChunk, 1024, swizzle_mode_for_bytes(128));
    const uint32_t tmem = sh->tmem;
    int s = 0;
    uint32_t ph = 0;
    for (int k = 0; k < steps; ++k) {
      const int b = k & 1;
      warp_wait2(&sh->full[s], ph, &sh->second_full[b], (k >> 1) & 1, wctx);
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint64_t ad = a_desc + ((s * Cfg::STAGE + i * 2 * kChunk) >> 4), bd = b_desc + ((b * Cfg::B_BYTES) >> 4);
#pragma unroll
        for (int j = 0; j < kRows / 16; ++j)
          umma_ss(el, tmem + i * 256, ad + j * (16 * 128 >> 4), bd + j * (16 * 128 >> 4), idesc, (k | j) != 0 ? 1u : 0u);
      }
      umma_commit(el, &sh->empty[s]);
      umma_commit(el, &sh->second_empty[b]);
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
    umma_commit(el, &sh->done);
  } else if (warp < 2 + kWorkers) {
    // Two groups of eight warps make every other stage's xh~, each in a buffer of its own: making one takes longer than its
    // products.  A lane makes 16 consecutive columns of a row: 8 lanes a row, twice 4 rows a warp.
    const int wk = warp - 2, group = wk >> 3, piece = lane & 7, sub = lane >> 3;
    // The block of ones: its first column is 1, the rest 0, in both buffers and for good.  In a range of one step the second
    // group must not write it: nothing that `done` stands for would come after its stores, and the sums are staged over them.
    for (int i = (wk & 7) * 32 + lane; group < steps && i < kRows * 8; i += 256) {
      const int r = i >> 3, q = i & 7;
      *reinterpret_cast<uint4*>(b_buf + group * Cfg::B_BYTES + ones * kChunk + r * 128 + ((q ^ (r & 7)) << 4)) =
          make_uint4(q == 0 ? 0x3f80u : 0u, 0u, 0u, 0u);
    }
    const bool mine = piece < 4 * ones;  // (64 columns or fewer: the lanes of the second block have nothing to write)
    const int r0 = (wk & 7) * 8 + sub;
    float mean[2], rstd[2], down[2];
    auto stats = [&](int k) {  // of the rows, before their stage is waited for
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int64_t row = min(row_begin + (int64_t)k * kRows + r0 + p * 4, a.norm.rows - 1);
        mean[p] = a.norm.mean[row];
        rstd[p] = a.norm.rstd[row];
        down[p] = CODES ? a.norm.scales[row] : 1.f;
      }
    };
    if (group < steps) stats(group);
    int s = group;
    uint32_t ph = 0;
    for (int k = group; k < steps; k += 2) {
      uint64_t f2[2], m2[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        f2[p] = f2_dup(CODES ? down[p] * rstd[p] : rstd[p]);
        m2[p] = f2_dup(CODES ? -mean[p] * rstd[p] : -mean[p]);
      }
      if (k + 2 < steps) stats(k + 2);
      // In this order: with an odd number of stages a stage goes from group to group, and its barrier may be a phase further
      // back than `ph` tells from the one before.  The products of step k - 2 are done, so that step k - STAGES has landed.
      warp_wait(&sh->second_empty[group], ((k >> 1) & 1) ^ 1, wctx);
      warp_wait(&sh->full[s], ph, wctx);
      const uint8_t* raw = ring + s * Cfg::STAGE + Cfg::A_BYTES;
      uint4 u[2][CODES ? 1 : 2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int r = r0 + p * 4;
        if constexpr (CODES) {
          u[p][0] = *reinterpret_cast<const uint4*>(raw + r * 128 + piece * 16);
        } else {
          const uint4* src = reinterpret_cast<const uint4*>(raw + (piece >> 2) * kChunk + r * 128 + (piece & 3) * 32);
          u[p][0] = src[0];
          u[p][1] = src[1];
        }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int r = r0 + p * 4;
        uint64_t x[8];
        if constexpr (CODES) {
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
        const bool live = row_begin + (int64_t)k * kRows + r < row_end;  // (where d_out is zero: a NaN must not meet it)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float lo, hi;
          f2_unpack(x[e], lo, hi);
          o[e] = live ? pack_bf16x2(lo, hi) : 0u;
        }
        uint8_t* row = b_buf + group * Cfg::B_BYTES + (piece >> 2) * kChunk + r * 128;
        const int q = (piece & 3) * 2, sw = r & 7;
        if (mine) {
          *reinterpret_cast<uint4*>(row + ((q ^ sw) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(row + (((q + 1) ^ sw) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh->second_full[group]);
        mbar_arrive(&sh->empty[s]);
      }
      s += 2;
      if (s >= STAGES) {
        s -= STAGES;
        ph ^= 1;
      }
    }
    // the sums: four warps a lane quarter, which share the tiles and the blocks of 32 columns
    warp_wait(&sh->done, 0, wctx);
    tc_fence_after();
    const int quarter = warp & 3, share = wk >> 2;
    const int i = MT == 2 ? share & 1 : 0;
    const int o = m0 + i * 128 + quarter * 32 + lane;
    const uint32_t t = tmem_addr(sh->tmem, quarter * 32, i * 256);
    float* g = a.g + ((int64_t)range * a.outs + o - lane) * a.norm.cols;
#pragma unroll 1
    for (int c = 32 * (MT == 2 ? share >> 1 : share); c < a.norm.cols; c += MT == 2 ? 64 : 128) {
      uint32_t v[32];
      tmem_ld32(t + c, v);
      tmem_ld_wait();
      // (the stages and the buffers of xh~ are all used up)
      put_block(smem + wk * kBlockStaging, v, lane, [&](int r, int e, const float4& x) {
        if (o - lane + r < a.outs && c + e < a.norm.cols)
          *reinterpret_cast<float4*>(g + (int64_t)r * a.norm.cols + c + e) = x;
      });
    }
    if (share < MT) {
      uint32_t v[8];
      tmem_ld8(t + ones * 64, v);
      tmem_ld_wait();
      if (o < a.outs) a.s[(int64_t)range * a.outs + o] = __uint_as_float(v[0]);
    }
  }
}

// ---- dx ------------------------------------------------------------------------------------------
constexpr int kWBytes = 128 * 1024;  // most of the weight
constexpr int kATile = 128 * 128;    // 128 rows of 64 outputs
constexpr int kHalfTile = 1024;      // 32 rows of 16 columns of dx on their way out; 32 columns: twice as much
constexpr int kSmem = kSmemMax;      // all of it: one CTA an SM
template <bool CODES>
constexpr int kKept = CODES ? 128 * 128 : 2 * 128 * 128;  // 128 rows of 128 codes, or twice 64 bf16
static_assert(kSharedBytes + kWBytes + kWorkers * kHalfTile + kKept<false> + 3 * kATile <= kSmem, "");

// 32 columns of a kept row, as they lie in memory.
template <bool CODES>
struct KeptBlock {
  static constexpr int N = CODES ? 2 : 4;
  uint4 u[N];
  // Where 16-byte unit i of columns c0 .. c0 + 31 is in a tile (rows of 128 bytes, 128-byte swizzle).
  static __device__ __forceinline__ uint8_t* at(uint8_t* tile, int row, int c0, int i) {
    const int unit = CODES ? c0 / 16 + i : c0 % 64 / 8 + i;
    return tile + (CODES ? 0 : c0 / 64 * (128 * 128)) + row * 128 + ((unit ^ (row & 7)) << 4);
  }
  __device__ __forceinline__ void load(uint8_t* tile, int row, int c0) {
#pragma unroll
    for (int i = 0; i < N; ++i) u[i] = *reinterpret_cast<const uint4*>(at(tile, row, c0, i));
  }
  // xh of sixteen columns, in pairs
  __device__ __forceinline__ void get(int i, uint64_t f, uint64_t m, uint64_t (&x)[8]) const {
    if constexpr (CODES) {
      unpack_codes(u[i].x, x);
      unpack_codes(u[i].y, x + 2);
      unpack_codes(u[i].z, x + 4);
      unpack_codes(u[i].w, x + 6);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f2_fma(x[e], f, m);
    } else {
      const uint32_t v[8] = {u[2 * i].x, u[2 * i].y, u[2 * i].z, u[2 * i].w,
                             u[2 * i + 1].x, u[2 * i + 1].y, u[2 * i + 1].z, u[2 * i + 1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = f2_mul(f2_add(f2_pack_bits(v[e] << 16, v[e] & 0xffff0000u), m), f);
    }
  }
};

template <bool CODES>
__device__ __forceinline__ void dx_role(uint8_t* smem, Shared* sh, const WaitCtx& wctx, const CUtensorMap& tm_rows,
                                        const CUtensorMap& tm_w, const CUtensorMap& tm_kept, const CUtensorMap& tm_dx,
                                        const BwdArgs& a, int part, int range) {
  const int kb = a.w_blocks, cb = a.col_blocks, stages = a.dx_stages;
  uint8_t* w_buf = smem;
  uint8_t* ring = smem + kb * cb * kChunk;
  uint8_t* kept = ring + stages * kATile;
  uint8_t* staging = kept + a.dx_kept * kKept<CODES>;
  float* w_norm = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sh) + 512);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int64_t range_begin = range * a.rows_per_range;
  const int64_t range_end = min(a.norm.rows, range_begin + a.rows_per_range);
  const int64_t row_begin = range_begin + part * 128;
  const int64_t row_step = a.dx_ctas * 128;
  const int tiles = row_begin < range_end ? (int)((range_end - row_begin + row_step - 1) / row_step) : 0;

  if (warp == 0) {
    const uint32_t el = elect_one();
    mbar_expect_tx(el, &sh->w_full, kb * cb * kChunk);
    for (int k = 0; k < kb; ++k)
      for (int c = 0; c < cb; ++c)
        tma_load_3d(el, w_buf + (k * cb + c) * kChunk, &tm_w, &sh->w_full, c * 64, k * 64, 0);
    int s = 0;
    uint32_t ph = 1;
    for (int t = 0; t < tiles; ++t) {
      const int row = (int)(row_begin + t * row_step);
      for (int k = 0; k < kb; ++k) {
        warp_wait(&sh->empty[s], ph, wctx);
        mbar_expect_tx(el, &sh->full[s], kATile);
        tma_load_3d(el, ring + s * kATile, &tm_rows, &sh->full[s], k * 64, row, 0);
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 2 + kWorkers) {
    const uint32_t el = elect_one();
    int s = 0;
    uint32_t ph = 1;
    for (int t = 0; t < tiles; ++t) {
      warp_wait(&sh->kept_empty[s], ph, wctx);
      mbar_expect_tx(el, &sh->kept_full[s], kKept<CODES>);
#pragma unroll
      for (int c = 0; c < (CODES ? 1 : 2); ++c)
        tma_load_3d(el, kept + s * kKept<CODES> + c * (128 * 128), &tm_kept, &sh->kept_full[s], c * 64,
                    (int)(row_begin + t * row_step), 0);
      if (++s == a.dx_kept) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t el = elect_one();
    const uint32_t idesc = make_idesc_bf16(128, (a.norm.cols + 31) / 32 * 32, false, true);
    const uint64_t a_desc = make_smem_desc(smem_u32(ring), 16, 1024, swizzle_mode_for_bytes(128));
    const uint64_t b_desc = make_smem_desc(smem_u32(w_buf), kChunk, 1024, swizzle_mode_for_bytes(128));
    const uint32_t tmem = sh->tmem;
    warp_wait(&sh->w_full, 0, wctx);
    int s = 0;
    uint32_t ph = 0;
    for (int t = 0; t < tiles; ++t) {
      const int acc = t & 1;
      warp_wait(&sh->second_empty[acc], ((t >> 1) & 1) ^ 1, wctx);
      tc_fence_after();
      for (int k = 0; k < kb; ++k) {
        warp_wait(&sh->full[s], ph, wctx);
        tc_fence_after();
        const uint64_t ad = a_desc + ((s * kATile) >> 4), bd = b_desc + ((k * cb * kChunk) >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          umma_ss(el, tmem + acc * 128, ad + j * 2, bd + j * (16 * 128 >> 4), idesc, (k | j) != 0 ? 1u : 0u);
        umma_commit(el, &sh->empty[s]);
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
      umma_commit(el, &sh->second_full[acc]);
    }
  } else {
    // Four warps a lane quarter, 32 columns each of its 32 rows; a lane has a row.  The kept rows come by TMA: a lane's loads
    // of its own row touch 32 lines an instruction (twice as long a tile).  Two warps a quarter took 4.2 us a tile.
    const int wk = warp - 2, quarter = warp & 3, c0 = (wk >> 2) * 32, r = quarter * 32 + lane;
    uint8_t* tile = staging + wk * (a.dx_width / 16) * kHalfTile;
    const bool exists = c0 < a.norm.cols;
    float mean = 0.f, rstd = 0.f, down = 1.f;
    auto stats = [&](int t) {
      const int64_t row = min(row_begin + t * row_step + r, a.norm.rows - 1);
      mean = a.norm.mean[row];
      rstd = a.norm.rstd[row];
      if (CODES) down = a.norm.scales[row];
    };
    if (tiles > 0) stats(0);
    int ks = 0;
    uint32_t kph = 0;
    for (int t = 0; t < tiles; ++t) {
      const int acc = t & 1;
      const uint64_t f = f2_dup(CODES ? down * rstd : rstd), m = f2_dup(CODES ? -mean * rstd : -mean), rs = f2_dup(rstd);
      if (t + 1 < tiles) stats(t + 1);
      uint8_t* rows = kept + ks * kKept<CODES>;
      warp_wait2(&sh->second_full[acc], (t >> 1) & 1, &sh->kept_full[ks], kph, wctx);
      tc_fence_after();
      KeptBlock<CODES> x;
      uint64_t wd[16], s1 = 0, s2 = 0;
      if (exists) {
        uint32_t v[32];
        tmem_ld32(tmem_addr(sh->tmem, quarter * 32, acc * 128 + c0), v);
        x.load(rows, r, c0);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float4 w = *reinterpret_cast<const float4*>(w_norm + c0 + e * 2);
          wd[e] = f2_mul(f2_pack_bits(v[2 * e], v[2 * e + 1]), f2_pack(w.x, w.y));
          wd[e + 1] = f2_mul(f2_pack_bits(v[2 * e + 2], v[2 * e + 3]), f2_pack(w.z, w.w));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint64_t xh[8];
          x.get(h, f, m, xh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            s1 = f2_add(s1, wd[h * 8 + e]);
            s2 = f2_fma(wd[h * 8 + e], xh[e], s2);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->second_empty[acc]);
      // The four sums of a row meet where its kept columns were: every lane's own are in registers by now.
      *reinterpret_cast<float2*>(KeptBlock<CODES>::at(rows, r, c0, 0)) = make_float2(f2_sum(s1), f2_sum(s2));
      asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = *reinterpret_cast<const float2*>(KeptBlock<CODES>::at(rows, r, k * 32, 0));
        sum.x += v.x;
        sum.y += v.y;
      }
      fence_async_smem();  // the next tile's rows come through the asynchronous proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->kept_empty[ks]);
      if (++ks == a.dx_kept) {
        ks = 0;
        kph ^= 1;
      }
      if (!exists) continue;
      const uint64_t m1 = f2_dup(-sum.x * a.norm.inv_cols), m2 = f2_dup(-sum.y * a.norm.inv_cols);
      uint32_t pk[16];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint64_t xh[8];
        x.get(h, f, m, xh);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float lo, hi;
          f2_unpack(f2_mul(f2_fma(xh[e], m2, f2_add(wd[h * 8 + e], m1)), rs), lo, hi);
          pk[h * 8 + e] = pack_bf16x2(lo, hi);
        }
      }
      const int row0 = (int)(row_begin + t * row_step + quarter * 32);
      if (a.dx_width == 32) {
        int buf = 0;
        warp_tile_store_tma<1>(tile, buf, lane, pk, &tm_dx, c0, row0, 0);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // rows of 32 bytes, 32-byte swizzle
          bulk_wait_read<0>();
          __syncwarp();
          const int sw = (lane >> 2) & 1;
          *reinterpret_cast<uint4*>(tile + lane * 32 + (sw << 4)) = make_uint4(pk[8 * h], pk[8 * h + 1], pk[8 * h + 2], pk[8 * h + 3]);
          *reinterpret_cast<uint4*>(tile + lane * 32 + ((sw ^ 1) << 4)) =
              make_uint4(pk[8 * h + 4], pk[8 * h + 5], pk[8 * h + 6], pk[8 * h + 7]);
          fence_async_smem();
          __syncwarp();
          if (c0 + h * 16 < a.norm.cols) tma_store_3d(lane == 0, &tm_dx, tile, c0 + h * 16, row0, 0);
        }
      }
    }
    bulk_wait_all();
  }
}

template <int MT, bool CODES>
__global__ void __launch_bounds__(32 * kWarps, 1)
    nl_bwd_kernel(const __grid_constant__ CUtensorMap tm_cols, const __grid_constant__ CUtensorMap tm_rows,
                  const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_kept,
                  const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_dx,
                  const __grid_constant__ BwdArgs a, int* __restrict__ status) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using Grad = GradConfig<MT, CODES>;
  static_assert(Grad::SMEM <= kSmem, "");
  const int per = a.g_ctas + a.dx_ctas;
  const int range = blockIdx.x / per, part = blockIdx.x - range * per;
  const bool grad = part < a.g_ctas;
  Shared* sh = reinterpret_cast<Shared*>(smem + kSmem - kSharedBytes);
  const WaitCtx wctx{&sh->abort_flag, status};
  const int warp = warp_index();
  if (threadIdx.x == 0) {
    for (int s = 0; s < 8; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], grad ? 1 + kWorkers / 2 : 1);  // UMMAs; for G the warps that read the kept rows too
    }
    for (int b = 0; b < 2; ++b) {  // G: the xh~ buffers, dx: the accumulators
      mbar_init(&sh->second_full[b], grad ? kWorkers / 2 : 1);
      mbar_init(&sh->second_empty[b], grad ? 1 : kWorkers);
      mbar_init(&sh->kept_full[b], 1);
      mbar_init(&sh->kept_empty[b], kWorkers);
    }
    mbar_init(&sh->w_full, 1);
    mbar_init(&sh->done, 1);
    sh->abort_flag = 0;
    mbar_fence_init();
  }
  const int tmem_cols = grad ? Grad::TMEM : 256;
  if (warp == 1) {
    tmem_alloc(&sh->tmem, tmem_cols);
    tmem_relinquish();
  }
  griddep_wait();
  if (!grad && threadIdx.x >= 64 && threadIdx.x < 192) {
    float w;
    param_load<1, 1>(a.norm.w, threadIdx.x - 64, a.norm.cols, 1.f, &w);
    reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(sh) + 512)[threadIdx.x - 64] = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (grad) grad_role<MT, CODES>(smem, sh, wctx, tm_cols, tm_x, a, part, range);
  else dx_role<CODES>(smem, sh, wctx, tm_rows, tm_w, tm_kept, tm_dx, a, part - a.g_ctas, range);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(sh->tmem, tmem_cols);
  }
}

// One CTA an output: G_o and s_o over the ranges (in order), then dW_o = w G_o + b s_o and the output's terms
// terms[o] = (W_o G_o, W_o s_o) of dw and db.  32 lanes hold four columns each, eight warps a part of the ranges.
__global__ void __launch_bounds__(256) nl_fold_kernel(const BwdArgs a, int ranges, const bf16* __restrict__ w, ParamOut dw,
                                                      float* __restrict__ terms) {
  griddep_wait();
  __shared__ float4 red[8][32];
  __shared__ float red_s[8];
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, o = blockIdx.x, cols = a.norm.cols;
  const int per = (ranges + 7) / 8, k0 = g * per, k1 = min(ranges, k0 + per);
  const int c = lane * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  float t = 0.f;
  for (int k = k0; k < k1; k += 8) {
    float4 v[8];
    float q[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t at = (int64_t)(k + u) * a.outs + o;
      v[u] = c < cols && k + u < k1 ? *reinterpret_cast<const float4*>(a.g + at * cols + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      q[u] = k + u < k1 ? a.s[at] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      s.x += v[u].x;
      s.y += v[u].y;
      s.z += v[u].z;
      s.w += v[u].w;
      t += q[u];
    }
  }
  red[g][lane] = s;
  if (lane == 0) red_s[g] = t;
  __syncthreads();
  const int e = threadIdx.x;  // one column
  if (e >= cols) return;
  const float* r = reinterpret_cast<const float*>(&red[0][0]) + e;
  float G = r[0], S = red_s[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) {
    G += r[k * 128];
    S += red_s[k];
  }
  float gamma, beta;
  param_load<1, 1>(a.norm.w, e, cols, 1.f, &gamma);
  param_load<1, 1>(a.norm.b, e, cols, 0.f, &beta);
  if (dw.p != nullptr) param_put(dw, (int64_t)o * cols + e, fmaf(gamma, G, beta * S));
  if (terms != nullptr) {
    const float wo = __bfloat162float(w[(int64_t)o * cols + e]);
    terms[(int64_t)o * 2 * cols + e] = wo * G;
    terms[(int64_t)o * 2 * cols + cols + e] = wo * S;
  }
}

struct Plan {
  int mt, tiles, ranges, g_ctas, dx_ctas;
  int64_t rows_per_range;
};
Plan make_plan(int64_t rows, int64_t outs, bool want_g, bool want_dx) {
  Plan p;
  p.mt = outs > 128 ? 2 : 1;
  p.tiles = (int)((outs + p.mt * 128 - 1) / (p.mt * 128));
  p.g_ctas = want_g ? p.tiles : 0;
  // with 128 outputs or fewer a CTA for G is done in half the time of one for dx (500000 rows of 128: 97 us, 119 with one each)
  p.dx_ctas = want_dx ? (p.mt == 1 ? 2 : p.tiles) : 0;
  int64_t ranges = sm_count() / (p.g_ctas + p.dx_ctas);
  const int64_t most = (rows + 255) / 256;  // 256 rows at least: G's sums are written and read once more
  if (ranges > most) ranges = most;
  if (ranges < 1) ranges = 1;
  p.rows_per_range = ((rows + ranges - 1) / ranges + 127) / 128 * 128;
  p.ranges = (int)((rows + p.rows_per_range - 1) / p.rows_per_range);
  return p;
}
// The most ranges that any choice of gradients takes.
int64_t most_ranges(int64_t rows, int64_t outs) { return make_plan(rows, outs, true, false).ranges; }

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

template <int MT, bool CODES>
int launch_bwd(const BwdArgs& a, const Plan& p, const void* d_out, const void* w, void* dx, cudaStream_t stream) {
  CUtensorMap tm_cols, tm_rows, tm_x, tm_kept, tm_w, tm_dx;
  const int64_t R = a.norm.rows, C = a.norm.cols, O = a.outs;
  if (int rc = make_operand_tmap(&tm_cols, d_out, true, O, R, O, 1, 0, 128, 64, kRows)) return rc;
  if (int rc = make_operand_tmap(&tm_rows, d_out, false, R, O, O, 1, 0, 128, 128, 64)) return rc;
  if (int rc = make_operand_tmap(&tm_w, w, true, C, O, C, 1, 0, 128, 64, 64)) return rc;
  const int64_t pitch = CODES ? a.norm.code_pitch : a.norm.x_pitch * 2;  // bytes
  const uint64_t dims[3] = {(uint64_t)(CODES ? pitch : C), (uint64_t)R, 1}, strides[2] = {(uint64_t)pitch, 16};
  const uint32_t box[3] = {CODES ? 128u : 64u, (uint32_t)kRows, 1}, kept_box[3] = {CODES ? 128u : 64u, 128, 1};
  const auto type = CODES ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const void* kept = CODES ? static_cast<const void*>(a.norm.codes) : a.norm.x;
  if (int rc = make_tmap(&tm_x, type, kept, 3, dims, strides, box, 0)) return rc;
  if (int rc = make_tmap(&tm_kept, type, kept, 3, dims, strides, kept_box, 128)) return rc;
  if (dx != nullptr) {
    const uint64_t dx_dims[3] = {(uint64_t)C, (uint64_t)R, 1}, dx_strides[2] = {(uint64_t)C * 2, 16};
    const uint32_t dx_box[3] = {(uint32_t)a.dx_width, 32, 1};
    if (int rc = make_tmap_bf16(&tm_dx, dx, 3, dx_dims, dx_strides, dx_box, a.dx_width * 2)) return rc;
  } else {
    tm_dx = tm_w;  // not used
  }
  int* status = nullptr;
  static PerDeviceAddress status_at;
  if (int rc = device_symbol_address(g_nl_bwd_status, status_at, reinterpret_cast<void**>(&status))) return rc;
  const auto kern = nl_bwd_kernel<MT, CODES>;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(kern, kSmem, once, 1024)) return rc;
  launch_kernel(kern, dim3(p.ranges * (p.g_ctas + p.dx_ctas)), dim3(32 * kWarps), kSmem, stream, tm_cols, tm_rows, tm_x, tm_kept,
                tm_w, tm_dx, a, status);
  TPF_LAUNCH_OK();
  return TPF_OK;
}

}  // namespace

int norm_linear_bwd_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  TPF_CUDA_OK(cudaMemcpyFromSymbol(&v, g_nl_bwd_status, sizeof(int)));
  if (v) TPF_CUDA_OK(cudaMemcpyToSymbol(g_nl_bwd_status, &zero, sizeof(int)));
  *out = v;
  return TPF_OK;
}

bool norm_linear_narrow(int64_t cols, int64_t outs) {
  return cols <= 128 && (outs + 63) / 64 * ((cols + 63) / 64) * kChunk <= kWBytes;
}

int64_t norm_linear_narrow_bwd_workspace_bytes(int64_t rows, int64_t cols, int64_t outs) {
  const int64_t z = rows > 0 ? most_ranges(rows, outs) : 0;
  return up256(z * outs * cols * 4) + up256(z * outs * 4) + up256(outs * 2 * cols * 4);
}

int norm_linear_narrow_bwd(const NormArgs& norm, const void* w, int64_t outs, const NormLinearGrads& g, void* workspace,
                           cudaStream_t stream) {
  const int64_t R = norm.rows, C = norm.cols;
  const bool vectors = g.dweight != nullptr || g.dbias != nullptr, want_g = g.dw != nullptr || vectors;
  if (!want_g && g.dx == nullptr) return TPF_OK;
  const Plan p = make_plan(R, outs, want_g, g.dx != nullptr);
  const int64_t z = most_ranges(R, outs);
  char* base = static_cast<char*>(workspace);
  float* terms = reinterpret_cast<float*>(base + up256(z * outs * C * 4) + up256(z * outs * 4));
  const bool codes = norm.codes != nullptr;
  const int w_blocks = (int)((outs + 63) / 64), col_blocks = (int)((C + 63) / 64);
  // What the weight leaves: narrow staging where d_out would have two blocks (512 outputs from whole rows: 213 us, 307 with
  // two blocks; from codes it would be 199 in the place of 190), a second tile of kept rows where four blocks fit beside it.
  const int kept = codes ? kKept<true> : kKept<false>;
  const int left = kSmem - kSharedBytes - w_blocks * col_blocks * kChunk;
  const int dx_width = left - kWorkers * 2 * kHalfTile - kept >= 3 * kATile ? 32 : 16;
  const int room = left - kWorkers * (dx_width / 16) * kHalfTile;
  const int dx_kept = room - 2 * kept >= 4 * kATile ? 2 : 1;
  int dx_stages = (room - dx_kept * kept) / kATile;
  if (dx_stages > 8) dx_stages = 8;
  const BwdArgs a{norm, p.rows_per_range, (int)outs, p.g_ctas, p.dx_ctas, w_blocks, col_blocks, dx_stages, dx_kept,
                  dx_width, reinterpret_cast<float*>(base), reinterpret_cast<float*>(base + up256(z * outs * C * 4))};
  const int rc = p.mt == 2 ? (codes ? launch_bwd<2, true>(a, p, g.d_out, w, g.dx, stream)
                                    : launch_bwd<2, false>(a, p, g.d_out, w, g.dx, stream))
                           : (codes ? launch_bwd<1, true>(a, p, g.d_out, w, g.dx, stream)
                                    : launch_bwd<1, false>(a, p, g.d_out, w, g.dx, stream));
  if (rc || !want_g) return rc;
  launch_kernel(nl_fold_kernel, dim3((unsigned)outs), dim3(256), 0, stream, a, p.ranges, static_cast<const bf16*>(w),
                ParamOut{g.dw, g.dw_type}, vectors ? terms : nullptr);
  TPF_LAUNCH_OK();
  if (!vectors) return TPF_OK;
  return norm_fold(terms, (int)outs, (int)C, g.dweight, g.dweight_type, g.dbias, g.dbias_type, stream);
}

}  // namespace tpf

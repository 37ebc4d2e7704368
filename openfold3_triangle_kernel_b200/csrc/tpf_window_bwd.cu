// Window attention, backward, for sm_100a.
//
//   P = exp(S - lse) where a key is seen (0 elsewhere, and in rows that see nothing),  dP = dO V^T,  dS = P (dP - delta)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K,       delta = rowsum(dO out)
//
// `window_stats_kernel` makes -lse log2(e) and -delta of every query, padded to whole tiles; `window_bwd_kernel` then runs with the keys as
// rows (dK and dV), with the queries (dQ), and before these, for the queries that see few keys, to make delta again from P and dP.
// It makes S and dP each time: seven products a tile instead of five, but every gradient is summed by one CTA in a fixed order,
// without atomics and without partial sums of dQ in memory (at a window of 1024 keys those would be 9 times dQ in fp32).
//
// An item is 128 rows (keys: K and V; queries: Q and dO), kept in shared memory while the CTA walks over their tiles of 64 columns.  S and
// dP are made with the rows as TMEM lanes, so that P and dS, written over them as 16-bit numbers, are the A operands of the second
// products straight from TMEM; a thread has a row.  Two groups of four warps take turns with the tiles, three where heads of 64 elements
// leave room for a third S and dP in TMEM: while one computes, the products of the others run.  With the keys as rows the CTA goes through all query heads that share them.  The next item's rows are
// loaded, and its first tiles made, while the last item's gradients are still on their way out (an item a CTA left the tensor pipe idle
// for 4 us at its start and end: 8192 queries, 32 heads on 8 of 128, window 1024: dQ 224 us, now 187, dK and dV 250 to 267).
//
// What bounds it at 128 elements a head: the tensor pipe.  An UMMA of 64 columns with both operands in shared memory reads 6 KB, 48
// cycles, for 32 cycles of products, which makes 1280 cycles a tile with the keys as rows and 1024 with the queries (1345 and 1127
// measured without masks, starts and ends).  Q and dO as operands in TMEM were no faster (239 us for 224),
// nor were gradients that leave by TMA through the place of the item's rows (dQ 184 us for 186, at 64 elements a head 152 for 146).
//
// The sinks are seen by every later query, which would make the first keys' CTA walk over the whole sequence.  It does its window;
// the queries beyond are split over CTAs of their own, whose sums of the sinks' rows a last kernel adds up in a fixed order.
#include "tpf_window_kernels.h"

namespace tpf {

static __device__ int g_window_bwd_status;

int window_bwd_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  TPF_CUDA_OK(cudaMemcpyFromSymbol(&v, g_window_bwd_status, sizeof(int)));
  if (v) TPF_CUDA_OK(cudaMemcpyToSymbol(g_window_bwd_status, &zero, sizeof(int)));
  *out = v;
  return TPF_OK;
}

namespace {

constexpr int kTile = 64;  // columns of a tile
// delta from the stored output has the roundings of that and of the probabilities in it.  Beside a dS of many keys they do not show; where a
// query sees fewer than this, delta is made as the sum of P dP in fp32, tile by tile.  (Error of dQ and dK relative to their
// norms, bf16, roundings of dS and of the results alone 0.0023: with two keys 0.0043, nine 0.0028, 31 0.0025, 128 0.0024.)
// It costs a third S and dP of the items that have such a query (backward, us, without it and with it: 8192 tokens, 32 heads on 8 of 128,
// windows of 64, 100 and 127 keys 155 and 199, 183 and 232, 180 and 229, of 128, where only the first queries see fewer, 176 and 187; of 64
// elements a head, 64 keys 91 and 123; causal, 256 of 128 tokens 257 and 323).
constexpr int kFewKeys = 128;

// ---- stats ------------------------------------------------------------------------------------------------
// [B, H, NP] of -lse log2(e) (-inf: the row sees nothing, or lies behind the last one) and of -delta.
// A team of lanes, one for every eight elements of a head, has eight queries of a head (a query at a time it took 33 us at 8192 queries of
// 32 heads of 128 and 31 at 64, now 26 and 14; the bytes are 20 and 10).
template <typename T, int LANES>
__global__ void __launch_bounds__(256) window_stats_kernel(const T* __restrict__ out, const T* __restrict__ d_out,
                                                           const float* __restrict__ lse, float* __restrict__ nlse,
                                                           float* __restrict__ ndelta, int N, int NP, int H, int D, int64_t teams) {
  griddep_wait();
  const int lane = threadIdx.x % LANES;
  const int64_t team = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;  // (b, eight queries, h)
  const int64_t bi = team / H;
  const int h = (int)(team - bi * H);
  const int64_t b = bi / (NP / 8);
  const int i0 = (int)(bi - b * (NP / 8)) * 8;
  const bool on = team < teams && lane * 8 < D;
  const int64_t at = ((b * N + i0) * H + h) * D + lane * 8, pitch = (int64_t)H * D;
  float s[8];
#pragma unroll
  for (int half = 0; half < 8; half += 4) {
    Piece<T, 8> x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (on && i0 + half + k < N) {
        x[k].load(out + at + (half + k) * pitch);
        y[k].load(d_out + at + (half + k) * pitch);
      } else {
        x[k].zero();
        y[k].zero();
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float u[8], v[8], t = 0.f;
      x[k].get(u);
      y[k].get(v);
#pragma unroll
      for (int e = 0; e < 8; ++e) t = fmaf(u[e], v[e], t);
      s[half + k] = t;
    }
  }
  // eight sums over the team: the lanes share the queries out while they add
#pragma unroll
  for (int n = 4; n > 0; n >>= 1)
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const bool upper = (lane & n) != 0;
      s[k] = (upper ? s[k + n] : s[k]) + __shfl_xor_sync(0xffffffffu, upper ? s[k] : s[k + n], n);
    }
  if (LANES == 16) s[0] += __shfl_xor_sync(0xffffffffu, s[0], 8);
  if (lane < 8 && team < teams) {
    const int i = i0 + lane;
    const int64_t to = (b * H + h) * NP + i;
    const float l = i < N ? lse[(b * H + h) * N + i] : -INFINITY;
    nlse[to] = l == -INFINITY ? -INFINITY : -l * kWindowLog2e;
    ndelta[to] = -s[0];
  }
}

// ---- gradients --------------------------------------------------------------------------------------------
struct BwdArgs {
  const float *nlse, *ndelta;  // [B, H, NP]
  float* exact;                // ndelta, to be written
  int NP;
  void *g1, *g2;               // KEYS: dV and dK; else dQ and nothing
  float* parts;                // KEYS: [B, HK, 1 + far][2][sinks][D] of the sinks' rows, or nullptr
  int key_tiles, far, far_tiles;  // KEYS: items of far queries (of a head), and query tiles of each
  int row_items, heads, lists, items;    // items: (head, sequence, 128 rows), the heads fastest
  FastDiv div_heads, div_lists, div_g;  // (lists: heads of all sequences)
};

enum BwdRole { kKeyRows, kQueryRows, kDeltas };

template <typename T_, int DP_, BwdRole ROLE, bool TWICE_ = false>
struct BwdCfg {
  using T = T_;
  static constexpr bool TWICE = TWICE_;
  static constexpr int STEP = TWICE ? 16 : 8;                  // columns of TMEM from one 16 of an operand to the next
  static constexpr bool KEYS = ROLE == kKeyRows, DELTA = ROLE == kDeltas;
  static constexpr int DP = DP_, CHUNKS = DP / 64, NACC = KEYS ? 1 : 2;
  static constexpr int NS = DP == 64 ? 6 : 3, NR = 2;
  // Groups of compute warps, each with an S and a dP.  (Heads of 64, 8192 queries, 32 on 8 heads, window 1024: dQ 145 us with two, 118 with
  // three, dK and dV 193 and 169.)
  static constexpr int NG = DP == 64 ? 3 : 2;
  static constexpr int R_CHUNK = 128 * 128, C_CHUNK = kTile * 128;
  static constexpr int R_TILE = CHUNKS * R_CHUNK, C_TILE = CHUNKS * C_CHUNK;
  static constexpr int OFF_R = 0;                              // [NR] two tiles of rows
  static constexpr int OFF_C = OFF_R + NR * 2 * R_TILE;        // [NS] two tiles of columns
  static constexpr int OFF_VEC = OFF_C + NS * 2 * C_TILE;      // [NS] nlse and ndelta of the columns (KEYS)
  static constexpr int OFF_SUM = OFF_VEC + (KEYS ? NS * 2 * kTile * 4 : 0);  // [2][NG][128] fp32 (DELTA)
  static constexpr int OFF_BAR = OFF_SUM + (DELTA ? 2 * NG * 128 * 4 : 0);
  static constexpr int N_BAR = 2 * NR + 4 + 2 * NS + 2 * NG;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16;
  static constexpr int THREADS = 128 * NG + 64, WARP_TMA = 4 * NG, WARP_MMA = WARP_TMA + 1;
  static constexpr int TM_ACC = 128 * NG, TMEM_COLS = 512;          // KEYS: dV, dK; else dQ of two items in turn
  static_assert(SMEM + 1024 <= 233472 && TM_ACC + 2 * DP <= TMEM_COLS, "");
};

__device__ __forceinline__ void bulk_load(uint32_t elected, void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %4, 0;\n\t"
      "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "r"(elected)
      : "memory");
}

// The items of a CTA: one of every gridDim.x, from the front and from the back of them in turn, so that with the longest items first the
// CTAs get like sums.  (One stride for all: 8192 queries, causal, 16 heads on 4 of 128: 1090 us, now 770.)
struct BwdWalk {
  int item, step;
  __device__ __forceinline__ BwdWalk() : item(blockIdx.x), step(2 * (gridDim.x - 1 - blockIdx.x) + 1) {}
  __device__ __forceinline__ void next() {
    item += step;
    step = 2 * gridDim.x - step;
  }
};

// An item and its column tiles: for each of `heads` heads [a tile of the sinks,] tiles lo .. hi - 1.
template <class Cfg>
struct BwdItem {
  static constexpr bool KEYS = Cfg::KEYS;
  int r0, head, b, len, off;  // head: KEYS: a key head, else a query head
  int part;                   // KEYS: 0, or 1 + the number of far queries' item
  int extra, lo, heads, per_head, tiles;
  __device__ __forceinline__ BwdItem(int item, const WindowParams& p, const BwdArgs& a) {
    const int turn = (int)a.div_lists.div((uint32_t)item), list = item - turn * a.lists;
    b = (int)a.div_heads.div((uint32_t)list);
    head = list - b * a.heads;
    // the longest items first: the first keys, or the last queries, where the window is longer on the left
    const int x = (p.left > p.right) == KEYS ? turn : a.row_items - 1 - turn;
    len = p.length(b), off = p.first_position(b);
    part = KEYS && x >= a.key_tiles ? x - a.key_tiles + 1 : 0;
    r0 = part > 0 ? 0 : x * 128;
    extra = 0;
    int hi;
    if constexpr (KEYS) {
      heads = p.G;
      const int last = min(r0 + 127, len - 1);
      const int first = min(max(0, r0 - p.right - off), p.N), end = max(0, min(p.N, last + p.left - off + 1));
      lo = first / kTile;
      hi = r0 < len ? max(lo, (end + kTile - 1) / kTile) : lo;
      if (part > 0) {  // queries beyond the first key tile's window
        lo = max(hi, (part - 1) * a.far_tiles);
        hi = len > 0 ? min((p.N + kTile - 1) / kTile, part * a.far_tiles) : lo;
      }
    } else {
      heads = 1;
      const KeyRange kr = key_range(p, len, off + r0, off + min(r0 + 127, p.N - 1));
      extra = kr.lo >= kTile && kr.sink > 0 ? 1 : 0;
      lo = kr.sink > 0 && !extra ? 0 : kr.lo / kTile;
      hi = (kr.hi + kTile - 1) / kTile;
    }
    if (Cfg::DELTA) {  // (the fewest keys are those of a query at one of the ends)
      auto count = [&](int pos) { return __popcll(seen_keys(p, min(len, 64), pos, 0)) + max(0, min(len, pos + p.right + 1) - max(64, pos - p.left)); };
      if (min(count(off + r0), count(off + min(r0 + 127, p.N - 1))) >= kFewKeys) hi = lo, extra = 0;
    }
    per_head = extra + max(0, hi - lo);
    tiles = per_head * heads;
  }
  __device__ __forceinline__ int column(int u) const { return u < extra ? 0 : (lo + u - extra) * kTile; }  // of tile u of a head
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap tmR1, const __grid_constant__ CUtensorMap tmR2,
                  const __grid_constant__ CUtensorMap tmC1, const __grid_constant__ CUtensorMap tmC2, const WindowParams p,
                  const BwdArgs a, int* __restrict__ status) {
  griddep_wait();
  using T = typename Cfg::T;
  constexpr bool KEYS = Cfg::KEYS, DELTA = Cfg::DELTA, TWICE = Cfg::TWICE;
  constexpr int DP = Cfg::DP, NS = Cfg::NS, NR = Cfg::NR, NG = Cfg::NG, NACC = Cfg::NACC, CHUNKS = Cfg::CHUNKS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* r_full = bars;               // [NR]
  uint64_t* r_empty = r_full + NR;       // [NR]
  uint64_t* acc_full = r_empty + NR;     // [2]
  uint64_t* acc_free = acc_full + 2;     // [2]
  uint64_t* c_full = acc_free + 2;       // [NS]
  uint64_t* c_empty = c_full + NS;
  uint64_t* sdp_full = c_empty + NS;     // [NG]
  uint64_t* pds_ready = sdp_full + NG;   // [NG]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::N_BAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const WaitCtx wctx{abort_flag, status};
  const int warp = warp_index(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NR; ++s) {
      mbar_init(&r_full[s], 1);
      mbar_init(&r_empty[s], 1);
    }
    for (int s = 0; s < NS; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(&acc_full[g], 1);
      mbar_init(&acc_free[g], 8);
    }
    for (int g = 0; g < NG; ++g) {
      mbar_init(&sdp_full[g], 1);
      mbar_init(&pds_ready[g], 4);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmR1);
    tma_prefetch_desc(&tmR2);
    tma_prefetch_desc(&tmC1);
    tma_prefetch_desc(&tmC2);
  }
  if (warp == Cfg::WARP_MMA) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == Cfg::WARP_TMA) {
    const uint32_t el = elect_one();
    int s = 0, rs = 0;
    uint32_t ph = 1, rph = 1;
    for (BwdWalk walk; walk.item < a.items; walk.next()) {
      const BwdItem<Cfg> it(walk.item, p, a);
      if (it.tiles == 0) continue;
      warp_wait(&r_empty[rs], rph, wctx);
      mbar_expect_tx(el, &r_full[rs], 2 * Cfg::R_TILE);
      uint8_t* rows = smem + Cfg::OFF_R + rs * 2 * Cfg::R_TILE;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        tma_load_4d(el, rows + c * Cfg::R_CHUNK, &tmR1, &r_full[rs], 64 * c, it.r0, it.head, it.b);
        tma_load_4d(el, rows + Cfg::R_TILE + c * Cfg::R_CHUNK, &tmR2, &r_full[rs], 64 * c, it.r0, it.head, it.b);
      }
      if (++rs == NR) rs = 0, rph ^= 1;
      for (int hh = 0; hh < it.heads; ++hh) {
        const int ch = KEYS ? it.head * p.G + hh : (int)a.div_g.div((uint32_t)it.head);
        const int64_t vec = ((int64_t)it.b * p.H + ch) * a.NP;
        for (int u = 0; u < it.per_head; ++u) {
          const int c0 = it.column(u);
          warp_wait(&c_empty[s], ph, wctx);
          mbar_expect_tx(el, &c_full[s], 2 * Cfg::C_TILE + (KEYS ? 2 * kTile * 4 : 0));
          uint8_t* dst = smem + Cfg::OFF_C + s * 2 * Cfg::C_TILE;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            tma_load_4d(el, dst + c * Cfg::C_CHUNK, &tmC1, &c_full[s], 64 * c, c0, ch, it.b);
            tma_load_4d(el, dst + Cfg::C_TILE + c * Cfg::C_CHUNK, &tmC2, &c_full[s], 64 * c, c0, ch, it.b);
          }
          if constexpr (KEYS) {
            uint8_t* v = smem + Cfg::OFF_VEC + s * 2 * kTile * 4;
            bulk_load(el, v, a.nlse + vec + c0, kTile * 4, &c_full[s]);
            bulk_load(el, v + kTile * 4, a.ndelta + vec + c0, kTile * 4, &c_full[s]);
          }
          if (++s == NS) s = 0, ph ^= 1;
        }
      }
    }
  } else if (warp == Cfg::WARP_MMA) {
    const uint32_t el = elect_one();
    constexpr uint32_t idesc_s = window_idesc<T>(128, kTile, false), idesc_acc = window_idesc<T>(128, DP, true);
    constexpr uint32_t hi = smem_desc_hi(1024, swizzle_mode_for_bytes(128));
    const uint32_t d_r = smem_desc_lo(smem_u32(smem + Cfg::OFF_R), 16);
    const uint32_t d_c = smem_desc_lo(smem_u32(smem + Cfg::OFF_C), 16);
    const uint32_t d_cmn = smem_desc_lo(smem_u32(smem + Cfg::OFF_C), Cfg::C_CHUNK);
    constexpr uint32_t kRows = 2 * Cfg::R_TILE >> 4, kStage = 2 * Cfg::C_TILE >> 4, kSecond = Cfg::C_TILE >> 4;
    // The issuing thread is what the tensor pipe waits for first: its loop over an item's tiles holds nothing but counters.  (As a walk over
    // the tiles of all items that finds the next item by itself it made the kernel of the keys 270 us in the place of 250.)
    int s = 0, rs = 0, bs = 0, ab = 0;
    uint32_t ph = 0, rph = 0, pph = 0, aph = 1;
    auto issue_sdp = [&](int buf) {
      warp_wait(&c_full[s], ph, wctx);
      tc_fence_after();
      const uint32_t r1 = NR > 1 ? d_r + rs * kRows : d_r, r2 = r1 + (Cfg::R_TILE >> 4);
      const uint32_t d1 = d_c + s * kStage, d2 = d1 + kSecond, to = tmem + 128 * buf;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        umma_ss_w<hi, hi, idesc_s>(el, to, r1 + ((d / 4 * Cfg::R_CHUNK + d % 4 * 32) >> 4),
                                   d1 + ((d / 4 * Cfg::C_CHUNK + d % 4 * 32) >> 4), d != 0);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        umma_ss_w<hi, hi, idesc_s>(el, to + 64, r2 + ((d / 4 * Cfg::R_CHUNK + d % 4 * 32) >> 4),
                                   d2 + ((d / 4 * Cfg::C_CHUNK + d % 4 * 32) >> 4), d != 0);
      umma_commit(el, &sdp_full[buf]);
      if (++s == NS) s = 0, ph ^= 1;
    };
    auto rows_used = [&] {  // by all S and dP of the item
      umma_commit(el, &r_empty[rs]);
      if (++rs == NR) rs = 0, rph ^= 1;
    };
    auto tiles_from = [&](BwdWalk& w) {  // of the next item that has any
      int n = 0;
      while (w.item < a.items && (n = BwdItem<Cfg>(w.item, p, a).tiles) == 0) w.next();
      return __shfl_sync(0xffffffffu, n, 0);
    };
    BwdWalk walk;
    int buf = 0, lead = 0;  // lead: tiles of the item whose S and dP were made while the one before was finished
    int tiles = tiles_from(walk);
    while (walk.item < a.items) {
      if (lead == 0) warp_wait(&r_full[rs], rph, wctx);
      for (; lead < NG && lead < tiles; ++lead) issue_sdp(buf + lead < NG ? buf + lead : buf + lead - NG);
      if (tiles <= NG) rows_used();
      walk.next();
      const int next_tiles = tiles_from(walk);
      lead = 0;
      for (int t = 0; t < tiles; ++t) {
        if (t == 0 && !DELTA) warp_wait2(&pds_ready[buf], pph, &acc_free[ab], aph, wctx);
        else warp_wait(&pds_ready[buf], pph, wctx);
        tc_fence_after();
        const uint32_t d1 = d_cmn + bs * kStage, d2 = d1 + kSecond, from = tmem + 128 * buf, sums = tmem + Cfg::TM_ACC + (NACC > 1 ? ab * DP : 0);
        if constexpr (KEYS) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma_ts_w<hi, idesc_acc>(el, sums, from + Cfg::STEP * k, d2 + k * 128, (k | t) != 0);
            if constexpr (TWICE) umma_ts_w<hi, idesc_acc>(el, sums, from + Cfg::STEP * k + 8, d2 + k * 128, true);
          }
        }
        if constexpr (!DELTA) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma_ts_w<hi, idesc_acc>(el, KEYS ? sums + DP : sums, from + 64 + Cfg::STEP * k, d1 + k * 128, (k | t) != 0);
            if constexpr (TWICE)
              umma_ts_w<hi, idesc_acc>(el, KEYS ? sums + DP : sums, from + 64 + Cfg::STEP * k + 8, d1 + k * 128, true);
          }
        }
        umma_commit(el, &c_empty[bs]);
        if (++bs == NS) bs = 0;
        // S and dP of NG tiles ahead go over P and dS, which the products just issued have to read: the UMMAs of a thread go through the
        // tensor pipe in order (as in the triangle attention's backward pass)
        if (t + NG < tiles) {
          issue_sdp(buf);
          if (t + NG + 1 == tiles) rows_used();
        } else {
          if (t + 1 == tiles) umma_commit(el, &acc_full[ab]);
          if (NR > 1 && tiles >= NG && lead < next_tiles) {  // of the next item (beside fewer tiles, its first one is not due yet)
            if (lead == 0) warp_wait(&r_full[rs], rph, wctx);
            issue_sdp(buf);
            ++lead;
          }
        }
        if (++buf == NG) buf = 0, pph ^= 1;
      }
      if (++ab == NACC) ab = 0, aph ^= 1;
      tiles = next_tiles;
    }
  } else {
    // ------------------------------------------------------------------ compute warps: one thread per row
    const int g = warp >> 2, lane_base = 32 * (warp & 3), row = lane_base + lane;
    const uint32_t t_s = tmem_addr(tmem, lane_base, 128 * g), t_dp = t_s + 64;
    const float c2 = p.scale * kWindowLog2e;
    const uint64_t c22 = f2_pack(c2, c2);
    const int rows = KEYS ? p.M : p.N, heads = KEYS ? p.HK : p.H;

    // KEYS: group 0 stores dV and group 1 dK; else each a half of dQ's columns (a third group nothing).  The sums of an item leave after
    // the group's first tile of a later one has been handed over.
    const int cb = KEYS ? 0 : g * (DP / 2), ce = KEYS ? DP : cb + DP / 2;
    const bool stores = g < 2 && !DELTA;
    constexpr int PART = KEYS && NG == 3 ? 16 : 32;  // columns in registers at a time
    const float mul = KEYS && g == 0 ? 1.f : p.scale;
    bool pending = false;
    int d_row = 0, d_head = 0, d_b = 0, d_part = 0, ab = 0;
    uint32_t aph = 0;
    auto store_rows = [&](bool any) {
      // the sinks' rows are finished by the last kernel
      const bool part = KEYS && a.parts != nullptr && d_row == row && row < min(p.sinks, p.M);
      T* out = static_cast<T*>(KEYS && g == 1 ? a.g2 : a.g1) + (((int64_t)d_b * rows + d_row) * heads + d_head) * p.D;
      float* sums = nullptr;
      if (part) sums = a.parts + (((((int64_t)d_b * p.HK + d_head) * (1 + a.far) + d_part) * 2 + g) * p.sinks + row) * p.D;
      const uint32_t src = tmem_addr(tmem, lane_base, Cfg::TM_ACC + (KEYS ? g : ab) * DP);
#pragma unroll 1
      for (int c = cb; c < ce; c += 16) {
        uint32_t r[16];
        if (any) {
          tmem_ld16(src + c, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) r[e] = 0u;
        }
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[e]) * mul;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (c + 8 * k >= p.D) continue;
          if (part) {
            *reinterpret_cast<float4*>(sums + c + 8 * k) = make_float4(v[8 * k], v[8 * k + 1], v[8 * k + 2], v[8 * k + 3]);
            *reinterpret_cast<float4*>(sums + c + 8 * k + 4) = make_float4(v[8 * k + 4], v[8 * k + 5], v[8 * k + 6], v[8 * k + 7]);
          } else if (d_part == 0 && d_row < rows) {
            store_vec<T, 8>(out + c + 8 * k, v + 8 * k);
          }
        }
      }
    };
    auto finish = [&] {
      warp_wait(&acc_full[ab], aph, wctx);
      tc_fence_after();
      store_rows(true);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_free[ab]);
      if (++ab == NACC) ab = 0, aph ^= 1;
      pending = false;
    };

    int turn = g;   // tiles until the group's next one
    [[maybe_unused]] int which = 0;
    int s = 0;      // stage of the item's first tile
    uint32_t ph = 0;
    for (BwdWalk walk; walk.item < a.items; walk.next()) {
      const BwdItem<Cfg> it(walk.item, p, a);
      const int mine = it.r0 + row;
      if (it.tiles == 0) {
        if (pending) finish();
        d_row = mine, d_head = it.head, d_b = it.b, d_part = it.part;
        if (stores) store_rows(false);
        continue;
      }
      float nl = 0.f, nd = 0.f;
      if (!KEYS && mine < p.N) {
        const int64_t at = ((int64_t)it.b * p.H + it.head) * a.NP + mine;
        nl = __ldg(a.nlse + at);
        if (!DELTA) nd = __ldg(a.ndelta + at);
      }
      const uint64_t nl2 = f2_pack(nl, nl), nd2 = f2_pack(nd, nd);
      [[maybe_unused]] uint64_t delta2 = 0;
      const int w0 = it.r0 + lane_base, w1 = w0 + 31, len = it.len, off = it.off;  // the warp's rows
      int u = turn, t = turn, st = s + turn;
      while (u >= it.per_head && t < it.tiles) u -= it.per_head;
      while (st >= NS) st -= NS;
      for (; t < it.tiles; t += NG) {
        const int c0 = it.column(u);
        warp_wait(&sdp_full[g], ph, wctx);
        ph ^= 1;
        tc_fence_after();
        uint64_t seen;
        bool whole;
        if constexpr (KEYS) {
          seen = seeing_queries(p, len, mine, off + c0);
          whole = w1 < len && off + c0 >= w1 - p.right && off + c0 + kTile - 1 <= w0 + p.left;
        } else {
          seen = seen_keys(p, len, off + mine, c0);
          whole = c0 + kTile <= min(len, off + w0 + p.right + 1) && c0 >= off + w1 - p.left;
        }
        const float* vec = reinterpret_cast<const float*>(smem + Cfg::OFF_VEC + st * 2 * kTile * 4);
        auto tile = [&](auto masked) {
          constexpr bool MASKED = decltype(masked)::value;
#pragma unroll
          for (int half = 0; half < kTile / PART; ++half) {
            uint32_t rs[PART], rd[PART];
            if constexpr (PART == 32) {
              tmem_ld32(t_s + 32 * half, rs);
              tmem_ld32(t_dp + 32 * half, rd);
            } else {
              tmem_ld16(t_s + 16 * half, rs);
              tmem_ld16(t_dp + 16 * half, rd);
            }
            tmem_ld_wait();
            const uint32_t bits = (uint32_t)(seen >> (PART * half));
#pragma unroll
            for (int q = 0; q < PART / 16; ++q) {
              uint32_t pk[8], dk[8];
              [[maybe_unused]] uint32_t pl[8], dl[8];  // what the rounding of these leaves over
              [[maybe_unused]] float4 x4, y4;  // of four columns
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int c = 16 * q + 2 * e;
                uint64_t l2 = nl2, de2 = nd2;
                if constexpr (KEYS) {
                  if (e % 2 == 0) {
                    x4 = *reinterpret_cast<const float4*>(vec + PART * half + c);
                    y4 = *reinterpret_cast<const float4*>(vec + kTile + PART * half + c);
                  }
                  l2 = e % 2 == 0 ? f2_pack(x4.x, x4.y) : f2_pack(x4.z, x4.w);
                  de2 = e % 2 == 0 ? f2_pack(y4.x, y4.y) : f2_pack(y4.z, y4.w);
                }
                float a0, a1;
                f2_unpack(f2_fma(f2_pack_bits(rs[c], rs[c + 1]), c22, l2), a0, a1);
                float p0 = ex2_approx(a0), p1 = ex2_approx(a1), d0, d1;
                f2_unpack(f2_mul(f2_pack(p0, p1), f2_add(f2_pack_bits(rd[c], rd[c + 1]), de2)), d0, d1);
                if (MASKED) {  // (what is masked may be a NaN)
                  if (!(bits >> c & 1u)) p0 = d0 = 0.f;
                  if (!(bits >> (c + 1) & 1u)) p1 = d1 = 0.f;
                }
                if constexpr (DELTA) {
                  delta2 = f2_add(delta2, f2_pack(d0, d1));
                } else {
                  // 16 bits, as operands of the products
                  pk[e] = pack2<T>(p0, p1);
                  dk[e] = pack2<T>(d0, d1);
                  if constexpr (TWICE) {
                    const float2 ph = unpack2<T>(pk[e]), dh = unpack2<T>(dk[e]);
                    pl[e] = pack2<T>(p0 - ph.x, p1 - ph.y);
                    dl[e] = pack2<T>(d0 - dh.x, d1 - dh.y);
                  }
                }
              }
              const int at = (PART * half + 16 * q) / 16 * Cfg::STEP;
              if (KEYS) tmem_st8(t_s + at, pk);
              if (!DELTA) tmem_st8(t_dp + at, dk);
              if constexpr (TWICE) {
                if (KEYS) tmem_st8(t_s + at + 8, pl);
                tmem_st8(t_dp + at + 8, dl);
              }
            }
          }
        };
        if (whole) tile(std::false_type{});
        else tile(std::true_type{});
        if constexpr (!KEYS && !DELTA) {
          // Keys behind the last one are anything, and a dS of zero times a NaN is one (S has been made from them, and masked).
          if (c0 + kTile > len) {
            uint8_t* kt = smem + Cfg::OFF_C + st * 2 * Cfg::C_TILE;
            for (int e = threadIdx.x & 127; e < CHUNKS * kTile * 8; e += 128) {
              const int r = e / 8 % kTile;
              if (c0 + r >= len)
                *reinterpret_cast<uint4*>(kt + e / (8 * kTile) * Cfg::C_CHUNK + r * 128 + e % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pds_ready[g]);
        if (pending) finish();
        u += NG;
        while (u >= it.per_head) u -= it.per_head;
        st += NG;
        while (st >= NS) st -= NS;
      }
      turn = t - it.tiles;
      s = (s + it.tiles) % NS;
      if constexpr (DELTA) {
        // the groups' parts of the rows' sums, added in their order
        float* sums = reinterpret_cast<float*>(smem + Cfg::OFF_SUM) + which * NG * 128;
        which ^= 1;  // (so that what the first group reads stays until everybody has come here again)
        sums[g * 128 + row] = f2_sum(delta2);
        asm volatile("bar.sync 1, %0;" ::"n"(NG * 128) : "memory");
        if (g == 0 && mine < p.N) {
          float sum = sums[row];
#pragma unroll
          for (int k = 1; k < NG; ++k) sum += sums[k * 128 + row];
          a.exact[((int64_t)it.b * p.H + it.head) * a.NP + mine] = -sum;
        }
      }
      if (pending) finish();  // (the item had no tile for the group)
      d_row = mine, d_head = it.head, d_b = it.b, d_part = it.part;
      pending = stores;
    }
    if (pending) finish();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::WARP_MMA) {
    __syncwarp();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
}

// ---- the sinks' rows ----------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) window_sinks_kernel(const float* __restrict__ parts, int count, int sinks, int D, int M, int HK,
                                                           T* __restrict__ dv, T* __restrict__ dk) {
  griddep_wait();
  __shared__ float4 red[8][32];
  const int row = blockIdx.x >> 1, which = blockIdx.x & 1, head = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const float* from = parts + (((int64_t)b * HK + head) * count * 2 + which) * sinks * D + row * D + 4 * lane;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (4 * lane < D)
    for (int k = w; k < count; k += 8) {
      const float4 x = *reinterpret_cast<const float4*>(from + (int64_t)k * 2 * sinks * D);
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
  red[w][lane] = s;
  __syncthreads();
  if (w == 0 && 4 * lane < D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      const float4 x = red[k][lane];
      s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
    }
    *reinterpret_cast<uint2*>((which == 0 ? dv : dk) + (((int64_t)b * M + row) * HK + head) * D + 4 * lane) =
        make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
  }
}

// Query tiles of a CTA of far queries: as many as a key tile's window has.
void far_plan(const WindowCall& c, int* far, int* far_tiles) {
  *far = 0;
  *far_tiles = 1;
  if (c.sinks == 0 || c.left == kWindowUnlimited) return;
  if (c.offsets == nullptr && c.offset + c.N - 1 <= c.left) return;  // every query's window reaches key 0
  const int64_t all = (c.N + kTile - 1) / kTile;
  int64_t window = ((int64_t)c.left + (c.right == kWindowUnlimited ? 0 : c.right) + 128) / kTile + 1;
  if (window < 8) window = 8;
  if (window > all) window = all;
  *far_tiles = (int)window;
  *far = (int)((all + window - 1) / window);
}
int64_t padded(int64_t n) { return (n + kTile - 1) / kTile * kTile; }
int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

template <class Cfg>
int launch(const CUtensorMap& r1, const CUtensorMap& r2, const CUtensorMap& c1, const CUtensorMap& c2, const WindowParams& p,
           BwdArgs a, const WindowCall& c, cudaStream_t stream) {
  a.row_items = Cfg::KEYS ? a.key_tiles + a.far : (int)((c.N + 127) / 128);
  a.heads = (int)(Cfg::KEYS ? c.HK : c.H);
  const int64_t items = (int64_t)a.row_items * a.heads * c.B;
  TPF_REQUIRE(items < (1ll << 31) - 65536, TPF_ERR_UNSUPPORTED, "window_attn_bwd: too many rows");
  a.items = (int)items;
  TPF_REQUIRE((int64_t)a.heads * c.B < (1ll << 31), TPF_ERR_UNSUPPORTED, "window_attn_bwd: too many heads");
  a.lists = a.heads * (int)c.B;
  a.div_lists = FastDiv::make((uint32_t)a.lists);
  a.div_heads = FastDiv::make((uint32_t)a.heads);
  a.div_g = FastDiv::make((uint32_t)p.G);
  const int grid = a.items < sm_count() ? a.items : sm_count();
  auto kern = window_bwd_kernel<Cfg>;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(kern, Cfg::SMEM, once, 1024)) return rc;
  int* status = nullptr;
  static PerDeviceAddress cache;
  if (int rc = device_symbol_address(g_window_bwd_status, cache, reinterpret_cast<void**>(&status))) return rc;
  launch_kernel(kern, dim3(grid), dim3(Cfg::THREADS), Cfg::SMEM, stream, r1, r2, c1, c2, p, a, status);
  TPF_LAUNCH_OK();
  return TPF_OK;
}

template <typename T, int DP>
int run(const WindowCall& c, const WindowParams& p, uint8_t* ws, cudaStream_t stream) {
  const int64_t NP = padded(c.N), stat = round256(c.B * c.H * NP * 4);
  BwdArgs a = {};
  float* nlse = reinterpret_cast<float*>(ws);
  float* ndelta = reinterpret_cast<float*>(ws + stat);
  a.nlse = nlse, a.ndelta = ndelta;
  a.NP = (int)NP;
  constexpr int LANES = DP / 8;
  const int64_t teams = c.B * c.H * (NP / 8);
  launch_kernel(window_stats_kernel<T, LANES>, dim3((unsigned)((teams + 256 / LANES - 1) / (256 / LANES))), dim3(256), 0, stream,
                static_cast<const T*>(c.out), static_cast<const T*>(c.d_out), static_cast<const float*>(c.lse), nlse, ndelta, (int)c.N,
                (int)NP, (int)c.H, (int)c.D, teams);
  TPF_LAUNCH_OK();
  const int64_t os[3] = {c.N * c.H * c.D, c.H * c.D, c.D};
  int rc;
  // Short sequences take P and dS in two parts, which together have 16 bits of mantissa (22 in fp16), so that the result's own rounding is
  // what is left of the error: 0.42 half steps of the gradient's norm for 0.60 with one part, at any length.  What differs is the
  // price, since longer sequences wait for the tensor pipe (backward, us, one part and two: 16.9 and 18.5 for three of 4
  // tokens, 303 and 322 for 256 of 128, 16 heads on 4 of 128, 71 and 82 for 64 of 128, 16 heads of 64; beyond: 327 and 359 for 128 of
  // 256, 63 and 75 for two of 2053, 128 on both sides, 480 and 597 for 8192, 32 heads on 8, window 1024).
  const bool twice = c.N <= 128 && c.M <= 128;
  // (without a bound on either side, and with enough keys, every query sees enough of them)
  if (c.lengths != nullptr || c.left != kWindowUnlimited || c.right != kWindowUnlimited || c.M < kFewKeys) {
    CUtensorMap tk, tv, tq, tg;
    if ((rc = make_window_tmap(&tq, c.q, c.type, c.B, c.N, c.H, c.D, c.qs, 128))) return rc;
    if ((rc = make_window_tmap(&tg, c.d_out, c.type, c.B, c.N, c.H, c.D, os, 128))) return rc;
    if ((rc = make_window_tmap(&tk, c.k, c.type, c.B, c.M, c.HK, c.D, c.ks, kTile))) return rc;
    if ((rc = make_window_tmap(&tv, c.v, c.type, c.B, c.M, c.HK, c.D, c.vs, kTile))) return rc;
    a.exact = ndelta;
    if ((rc = launch<BwdCfg<T, DP, kDeltas>>(tq, tg, tk, tv, p, a, c, stream))) return rc;
  }
  if (c.dk != nullptr) {
    CUtensorMap tk, tv, tq, tg;
    if ((rc = make_window_tmap(&tk, c.k, c.type, c.B, c.M, c.HK, c.D, c.ks, 128))) return rc;
    if ((rc = make_window_tmap(&tv, c.v, c.type, c.B, c.M, c.HK, c.D, c.vs, 128))) return rc;
    if ((rc = make_window_tmap(&tq, c.q, c.type, c.B, c.N, c.H, c.D, c.qs, kTile))) return rc;
    if ((rc = make_window_tmap(&tg, c.d_out, c.type, c.B, c.N, c.H, c.D, os, kTile))) return rc;
    a.g1 = c.dv, a.g2 = c.dk;
    a.key_tiles = (int)((c.M + 127) / 128);
    far_plan(c, &a.far, &a.far_tiles);
    if (a.far > 0) a.parts = reinterpret_cast<float*>(ws + 2 * stat);
    if ((rc = twice ? launch<BwdCfg<T, DP, kKeyRows, true>>(tk, tv, tq, tg, p, a, c, stream)
                    : launch<BwdCfg<T, DP, kKeyRows>>(tk, tv, tq, tg, p, a, c, stream)))
      return rc;
    if (a.far > 0) {
      launch_kernel(window_sinks_kernel<T>, dim3(2 * (unsigned)(c.sinks < c.M ? c.sinks : c.M), (unsigned)c.HK, (unsigned)c.B), dim3(256),
                    0, stream, static_cast<const float*>(a.parts), 1 + a.far, c.sinks, (int)c.D, (int)c.M, (int)c.HK,
                    static_cast<T*>(c.dv), static_cast<T*>(c.dk));
      TPF_LAUNCH_OK();
    }
  }
  if (c.dq != nullptr) {
    CUtensorMap tk, tv, tq, tg;
    if ((rc = make_window_tmap(&tq, c.q, c.type, c.B, c.N, c.H, c.D, c.qs, 128))) return rc;
    if ((rc = make_window_tmap(&tg, c.d_out, c.type, c.B, c.N, c.H, c.D, os, 128))) return rc;
    if ((rc = make_window_tmap(&tk, c.k, c.type, c.B, c.M, c.HK, c.D, c.ks, kTile))) return rc;
    if ((rc = make_window_tmap(&tv, c.v, c.type, c.B, c.M, c.HK, c.D, c.vs, kTile))) return rc;
    a.g1 = c.dq, a.g2 = nullptr;
    a.parts = nullptr;
    if ((rc = twice ? launch<BwdCfg<T, DP, kQueryRows, true>>(tq, tg, tk, tv, p, a, c, stream)
                    : launch<BwdCfg<T, DP, kQueryRows>>(tq, tg, tk, tv, p, a, c, stream)))
      return rc;
  }
  return TPF_OK;
}

}  // namespace

int64_t window_bwd_workspace_bytes(const WindowCall& c) {
  WindowCall any = c;
  static const int some = 0;
  any.offsets = &some;  // (the plan for positions that only the device knows is the larger one)
  int far, far_tiles;
  far_plan(any, &far, &far_tiles);
  return 2 * round256(c.B * c.H * padded(c.N) * 4) + (far > 0 ? c.B * c.HK * (1 + far) * 2 * c.sinks * c.D * 4 : 0);
}

int window_bwd(const WindowCall& c, const WindowParams& p, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  TPF_REQUIRE(workspace != nullptr && workspace_bytes >= window_bwd_workspace_bytes(c), TPF_ERR_WORKSPACE,
              "window_attn_bwd: the workspace is too small");
  TPF_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, TPF_ERR_INVALID_ARGUMENT,
              "window_attn_bwd: the workspace must be 256-byte aligned");
  TPF_REQUIRE(c.H <= 65535 && c.B * c.H * padded(c.N) < (1ll << 34), TPF_ERR_UNSUPPORTED, "window_attn_bwd: extent too large");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (c.type == kRowBF16) return c.D <= 64 ? run<bf16, 64>(c, p, ws, stream) : run<bf16, 128>(c, p, ws, stream);
  return c.D <= 64 ? run<__half, 64>(c, p, ws, stream) : run<__half, 128>(c, p, ws, stream);
}

}  // namespace tpf

// Window attention of many queries for sm_100a: a CTA has 128 queries of one head and walks over the tiles of 64 keys that they reach.
//
// Four softmax warps, a thread per query (= TMEM lane); a warp that loads by TMA and one that issues UMMAs.  S = Q K^T of two tiles is
// in TMEM at a time; a thread takes its 64 logits into registers, raises its maximum only when a tile exceeds it by more than
// a fixed gap, writes the probabilities over its logits as 16-bit numbers, and P V takes them from there; O stays in TMEM.
// Two CTAs share an SM, so that one computes exponentials while the other's products run.
// Tiles that every query of a warp sees whole take a way without masks.  The sinks, when they lie before the window, are a
// tile of their own, of as many steps of 16 keys as there are sinks.
// What bounds it at 128 elements a head: the tensor pipe.  S = Q K^T is made 64 columns at a time, of 6 KB from shared memory, 48
// cycles for 32 cycles of products, so a tile takes it 640 cycles; the two CTAs of an SM need 1600 for a tile each, which leaves it
// 80 % busy.  The exponentials (16 a clock and SM) are 1024 of them, beside the products.
// Measured (B200, bf16, 32 heads on 8 of 128, 8192 queries, window 1024): 139 us, 0.93 PFLOP/s; causal 1.2.  Tiles of 128 keys with one S at a
// time (187 us), two threads a row (188), a part of the exponentials as polynomials (160) and a persistent walk (154) gained nothing.
#include "tpf_window_kernels.h"

namespace tpf {

static __device__ int g_window_fwd_status;

int window_fwd_status_fetch_and_clear(int* out) {
  int v = 0, zero = 0;
  TPF_CUDA_OK(cudaMemcpyFromSymbol(&v, g_window_fwd_status, sizeof(int)));
  if (v) TPF_CUDA_OK(cudaMemcpyToSymbol(g_window_fwd_status, &zero, sizeof(int)));
  *out = v;
  return TPF_OK;
}

int make_window_tmap(CUtensorMap* tm, const void* base, int type, int64_t B, int64_t rows, int64_t heads, int64_t D,
                     const int64_t* strides, int box_rows) {
  auto bytes = [&](int64_t n, int64_t stride) { return n > 1 ? (uint64_t)stride * 2 : (uint64_t)256; };  // (any, where it is unused)
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)rows, (uint64_t)heads, (uint64_t)B};
  uint64_t s[3] = {bytes(rows, strides[1]), bytes(heads, strides[2]), bytes(B, strides[0])};
  uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
  return make_tmap(tm, type == kRowBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, base, 4, dims, s, box,
                   128);
}

namespace {

template <typename T_, int DP_>
struct FwdCfg {
  using T = T_;
  static constexpr int DP = DP_, CHUNKS = DP / 64;   // elements of a head in steps of 64: a swizzled row of 128 bytes
  static constexpr int KEYS = 64, NK = 3, NV = 2;
  static constexpr int Q_CHUNK = 128 * 128, KV_CHUNK = KEYS * 128, KV_TILE = CHUNKS * KV_CHUNK;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + CHUNKS * Q_CHUNK;
  static constexpr int OFF_V = OFF_K + NK * KV_TILE;
  static constexpr int OFF_BAR = OFF_V + NV * KV_TILE;
  static constexpr int N_BAR = 1 + 2 * NK + 2 * NV + 6;
  static constexpr int SMEM = OFF_BAR + N_BAR * 8 + 16;
  static constexpr int THREADS = 192, WARP_TMA = 4, WARP_MMA = 5;
  static constexpr int S_COLS = 128, O_COLS = DP;
  static_assert((SMEM + 1024) * 2 <= 233472, "two CTAs an SM");
};

struct FwdArgs {
  float* lse;
  int tiles;  // of queries
  FastDiv div_heads;
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 2)
window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const WindowParams p, const FwdArgs a,
                  int* __restrict__ status) {
  griddep_wait();
  using T = typename Cfg::T;
  constexpr int DP = Cfg::DP, KEYS = Cfg::KEYS, NK = Cfg::NK, NV = Cfg::NV, CHUNKS = Cfg::CHUNKS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::OFF_BAR);
  uint64_t* q_full = bars;
  uint64_t* k_full = q_full + 1;        // [NK]
  uint64_t* k_empty = k_full + NK;
  uint64_t* v_full = k_empty + NK;      // [NV]
  uint64_t* v_empty = v_full + NV;
  uint64_t* s_full = v_empty + NV;      // [2]
  uint64_t* p_ready = s_full + 2;       // [2]
  uint64_t* pv_done = p_ready + 2;      // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Cfg::N_BAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);
  const WaitCtx wctx{abort_flag, status};
  const int warp = warp_index(), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < NK; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_ready[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == Cfg::WARP_MMA) {
    tmem_alloc(tmem_slot, Cfg::S_COLS);
    tmem_alloc(tmem_slot + 1, Cfg::O_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_s = tmem_slot[0], tmem_o = tmem_slot[1];

  // The queries that reach the most keys come first, the last ones where the window is longer on the left, and the heads beside one
  // another.  (Tile by tile of head by head, in their order: 8192 queries, 16 heads of 128, causal 300 us, now 230.)
  const int turn = (int)a.div_heads.div(blockIdx.x), h = (int)blockIdx.x - turn * p.H;
  const int i0 = (p.left > p.right ? a.tiles - 1 - turn : turn) * 128, b = blockIdx.y, hk = h / p.G;
  const int len = p.length(b), p0 = p.first_position(b) + i0;
  const KeyRange kr = key_range(p, len, p0, p0 + min(127, p.N - 1 - i0));
  // tile t: keys from first(t) on, steps(t) groups of 16 of them
  const int extra = kr.lo >= KEYS && kr.sink > 0 ? 1 : 0;   // the sinks as a tile of their own
  const int lo_tile = kr.sink > 0 && !extra ? 0 : kr.lo / KEYS;
  const int tiles = extra + (kr.hi > lo_tile * KEYS ? (kr.hi + KEYS - 1) / KEYS - lo_tile : 0);
  auto first = [&](int t) { return t < extra ? 0 : (lo_tile + t - extra) * KEYS; };
  auto steps = [&](int t) { return t < extra ? (kr.sink + 15) / 16 : min(4, (kr.hi - first(t) + 15) / 16); };

  if (warp == Cfg::WARP_TMA) {
    const uint32_t el = elect_one();
    if (tiles > 0) {
      mbar_expect_tx(el, q_full, CHUNKS * Cfg::Q_CHUNK);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) tma_load_4d(el, smem + Cfg::OFF_Q + c * Cfg::Q_CHUNK, &tmQ, q_full, 64 * c, i0, h, b);
    }
    int ks = 0, vs = 0;
    uint32_t kph = 1, vph = 1;
    for (int t = 0; t < tiles; ++t) {
      const int j0 = first(t);
      warp_wait(&k_empty[ks], kph, wctx);
      mbar_expect_tx(el, &k_full[ks], Cfg::KV_TILE);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        tma_load_4d(el, smem + Cfg::OFF_K + ks * Cfg::KV_TILE + c * Cfg::KV_CHUNK, &tmK, &k_full[ks], 64 * c, j0, hk, b);
      if (++ks == NK) ks = 0, kph ^= 1;
      warp_wait(&v_empty[vs], vph, wctx);
      mbar_expect_tx(el, &v_full[vs], Cfg::KV_TILE);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        tma_load_4d(el, smem + Cfg::OFF_V + vs * Cfg::KV_TILE + c * Cfg::KV_CHUNK, &tmV, &v_full[vs], 64 * c, j0, hk, b);
      if (++vs == NV) vs = 0, vph ^= 1;
    }
  } else if (warp == Cfg::WARP_MMA) {
    const uint32_t el = elect_one();
    constexpr uint32_t idesc_pv = window_idesc<T>(128, DP, true);
    const uint64_t q_desc = make_smem_desc(smem_u32(smem + Cfg::OFF_Q), 16, 1024, swizzle_mode_for_bytes(128));
    const uint64_t k_desc = make_smem_desc(smem_u32(smem + Cfg::OFF_K), 16, 1024, swizzle_mode_for_bytes(128));
    const uint64_t v_desc = make_smem_desc(smem_u32(smem + Cfg::OFF_V), Cfg::KV_CHUNK, 1024, swizzle_mode_for_bytes(128));
    int ks = 0;
    uint32_t kph = 0;
    auto issue_qk = [&](int t) {
      warp_wait(&k_full[ks], kph, wctx);
      tc_fence_after();
      const uint32_t idesc = window_idesc<T>(128, 0, false) | (uint32_t)(2 * steps(t)) << 17;
      const uint64_t kd = k_desc + (uint64_t)(ks * Cfg::KV_TILE >> 4);
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        umma_ss(el, tmem_s + 64 * (t & 1), q_desc + (uint64_t)((d / 4 * Cfg::Q_CHUNK + d % 4 * 32) >> 4),
                kd + (uint64_t)((d / 4 * Cfg::KV_CHUNK + d % 4 * 32) >> 4), idesc, d != 0);
      umma_commit(el, &s_full[t & 1]);
      umma_commit(el, &k_empty[ks]);
      if (++ks == NK) ks = 0, kph ^= 1;
    };
    if (tiles > 0) {
      warp_wait(q_full, 0, wctx);
      issue_qk(0);
      if (tiles > 1) issue_qk(1);
    }
    for (int t = 0; t < tiles; ++t) {
      const int buf = t & 1;
      const uint32_t ph = (t >> 1) & 1;
      warp_wait2(&p_ready[buf], ph, &v_full[buf], ph, wctx);
      tc_fence_after();
      const uint64_t vd = v_desc + (uint64_t)(buf * Cfg::KV_TILE >> 4);
      const int n = steps(t);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (s < n)
          umma_ts(el, tmem_o, tmem_s + 64 * buf + 8 * s, vd + (uint64_t)(s * 128), idesc_pv, (s | t) != 0);
      umma_commit(el, &pv_done[buf]);
      umma_commit(el, &v_empty[buf]);
      // S of tile t + 2 goes over P of this one, which the products just issued have to read: one thread's UMMAs go through the
      // tensor pipe in the order of issue (as in the triangle attention's backward pass).
      if (t + 2 < tiles) issue_qk(t + 2);
    }
  } else {
    // ------------------------------------------------------------------ softmax: one thread per query
    const int row = 32 * warp + lane, i = i0 + row, pos = p0 + row;
    const uint32_t t_s = tmem_addr(tmem_s, 32 * warp, 0), t_o = tmem_addr(tmem_o, 32 * warp, 0);
    const float c2 = p.scale * kWindowLog2e;  // logits -> exponents of two
    const uint64_t c22 = f2_pack(c2, c2);
    // largest exponent of two a probability may have relative to m: P is held in 16 bits, fp16 ends at 2^16
    constexpr float kGap = std::is_same<T, bf16>::value ? 16.f : 8.f;
    float m = -INFINITY, l = 0.f;  // m in units of S
    const bool live = i0 + 32 * warp < p.N;
    const int w0 = p0 + 32 * warp, w1 = w0 + 31;  // positions of the warp
    for (int t = 0; t < tiles; ++t) {
      const int buf = t & 1;
      const uint32_t ph = (t >> 1) & 1;
      const int j0 = first(t), n = steps(t);
      const bool whole = n == 4 && j0 + KEYS <= min(len, w0 + p.right + 1) && j0 >= w1 - p.left;
      const uint64_t seen = whole ? 0 : seen_keys(p, len, pos, j0) & low_bits(16 * n);
      const bool some = whole || __any_sync(0xffffffffu, seen != 0);
      warp_wait(&s_full[buf], ph, wctx);
      tc_fence_after();
      auto tile = [&](auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        uint32_t raw[64];
        tmem_ld32(t_s + 64 * buf, *reinterpret_cast<uint32_t(*)[32]>(raw));
        if (!MASKED || n > 2) tmem_ld32(t_s + 64 * buf + 32, *reinterpret_cast<uint32_t(*)[32]>(raw + 32));
        tmem_ld_wait();
        if (MASKED) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t bits = (uint32_t)(seen >> (16 * c)) & 0xffffu;
            if (__all_sync(0xffffffffu, bits == 0xffffu)) continue;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (!(bits >> e & 1u)) raw[16 * c + e] = 0xff800000u;
          }
        }
        float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          m0 = max3(m0, __uint_as_float(raw[e]), __uint_as_float(raw[e + 1]));
          m1 = max3(m1, __uint_as_float(raw[e + 2]), __uint_as_float(raw[e + 3]));
        }
        const float top = fmaxf(m0, m1);
        const bool grow = (m == -INFINITY && top != -INFINITY) || (top - m) * c2 > kGap;
        if (__any_sync(0xffffffffu, grow)) {
          // rows that need it get a new maximum (f = 1 for the others), and what they have summed is rescaled
          const float f = grow ? ex2_approx((m - top) * c2) : 1.f;  // m = -inf gives 0
          const bool held = __any_sync(0xffffffffu, grow && m != -INFINITY);  // (rows that have seen nothing yet have sums of zeros: 143 us, now 139)
          if (grow) m = top;
          l *= f;
          if (t > 0 && held) {
            warp_wait(&pv_done[buf ^ 1], ((t - 1) >> 1) & 1, wctx);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DP; c += 8) {
              uint32_t ro[8];
              tmem_ld8(t_o + c, ro);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) ro[e] = __float_as_uint(__uint_as_float(ro[e]) * f);
              tmem_st8(t_o + c, ro);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.f : -m * c2;
        const uint64_t shift2 = f2_pack(shift, shift);
        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (MASKED && c >= n) break;
          uint32_t pk[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a0, a1;
            f2_unpack(f2_fma(f2_pack_bits(raw[16 * c + 2 * e], raw[16 * c + 2 * e + 1]), c22, shift2), a0, a1);
            const float e0 = ex2_approx(a0), e1 = ex2_approx(a1);
            if (e & 1) sum1 = f2_add(sum1, f2_pack(e0, e1));
            else sum0 = f2_add(sum0, f2_pack(e0, e1));
            pk[e] = pack2<T>(e0, e1);  // an operand of the products: 16 bits; the sum takes it unrounded
          }
          tmem_st8(t_s + 64 * buf + 8 * c, pk);
        }
        float r0, r1;
        f2_unpack(f2_add(sum0, sum1), r0, r1);
        l += r0 + r1;
      };
      if (live && whole) {
        tile(std::false_type{});
      } else if (live && some) {
        tile(std::true_type{});
      } else if (live) {  // none of the warp's queries sees any of them
        const uint32_t zero[8] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st8(t_s + 64 * buf + 8 * c, zero);
      }
      if (j0 + 16 * n > len) {
        // Values behind the last key are anything (the rest of a cache), and a probability of zero times a NaN is one.
        warp_wait(&v_full[buf], ph, wctx);
        for (int e = threadIdx.x; e < CHUNKS * KEYS * 8; e += 128) {
          const int r = e / 8 % KEYS;
          if (j0 + r >= len)
            *reinterpret_cast<uint4*>(smem + Cfg::OFF_V + buf * Cfg::KV_TILE + e / (8 * KEYS) * Cfg::KV_CHUNK + r * 128 + e % 8 * 16) =
                make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[buf]);
    }
    if (tiles > 0) {
      warp_wait(&pv_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, wctx);
      tc_fence_after();
    }
    if (live) {
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // (a NaN stays one)
      // The warp's rows leave through the place of Q, which every S has been made from: written row by row from here they
      // took the address path 2048 cycles (8192 queries, 32 heads, window 1024: 151 us, now 143).
      uint8_t* mine = smem + Cfg::OFF_Q + row * 128;
#pragma unroll
      for (int c = 0; c < DP; c += 16) {
        uint32_t ro[16];
        if (tiles > 0) {
          tmem_ld16(t_o + c, ro);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) ro[e] = 0u;
        }
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(ro[e]) * inv;
        uint8_t* chunk = mine + c / 64 * Cfg::Q_CHUNK;
        store_vec<T, 8>(reinterpret_cast<T*>(chunk + ((c % 64 / 8) ^ (row & 7)) * 16), v);
        store_vec<T, 8>(reinterpret_cast<T*>(chunk + ((c % 64 / 8 + 1) ^ (row & 7)) * 16), v + 8);
      }
      fence_async_smem();
      __syncwarp();
      const uint32_t el = elect_one();
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c)
        tma_store_4d(el, &tmO, smem + Cfg::OFF_Q + c * Cfg::Q_CHUNK + warp * 32 * 128, 64 * c, i0 + 32 * warp, h, b);
      if (i < p.N && a.lse != nullptr)
        a.lse[((int64_t)b * p.H + h) * p.N + i] =
            l == 0.f ? -INFINITY : (m * c2 + log2f(l)) * 0.6931471805599453f;
      bulk_wait_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::WARP_MMA) {
    __syncwarp();
    tmem_dealloc(tmem_s, Cfg::S_COLS);
    tmem_dealloc(tmem_o, Cfg::O_COLS);
  }
}

template <typename T, int DP>
int launch(const WindowCall& c, const WindowParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
           const CUtensorMap& to, cudaStream_t stream) {
  using Cfg = FwdCfg<T, DP>;
  auto kern = window_fwd_kernel<Cfg>;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(kern, Cfg::SMEM, once, 1024)) return rc;
  int* status = nullptr;
  static PerDeviceAddress cache;
  if (int rc = device_symbol_address(g_window_fwd_status, cache, reinterpret_cast<void**>(&status))) return rc;
  const int64_t tiles = (c.N + 127) / 128;
  TPF_REQUIRE(tiles * c.H < (1ll << 31), TPF_ERR_UNSUPPORTED, "window_attn_fwd: too many queries and heads");
  launch_kernel(kern, dim3((unsigned)(tiles * c.H), (unsigned)c.B), dim3(Cfg::THREADS), Cfg::SMEM, stream, tq, tk, tv, to, p,
                FwdArgs{c.lse, (int)tiles, FastDiv::make((uint32_t)c.H)}, status);
  TPF_LAUNCH_OK();
  return TPF_OK;
}

}  // namespace

int window_many(const WindowCall& c, const WindowParams& p, cudaStream_t stream) {
  CUtensorMap tq, tk, tv, to;
  const int64_t out_strides[3] = {c.N * c.H * c.D, c.H * c.D, c.D};
  int rc;
  if ((rc = make_window_tmap(&tq, c.q, c.type, c.B, c.N, c.H, c.D, c.qs, 128))) return rc;
  if ((rc = make_window_tmap(&tk, c.k, c.type, c.B, c.M, c.HK, c.D, c.ks, 64))) return rc;
  if ((rc = make_window_tmap(&tv, c.v, c.type, c.B, c.M, c.HK, c.D, c.vs, 64))) return rc;
  if ((rc = make_window_tmap(&to, c.out, c.type, c.B, c.N, c.H, c.D, out_strides, 32))) return rc;
  if (c.type == kRowBF16)
    return c.D <= 64 ? launch<bf16, 64>(c, p, tq, tk, tv, to, stream) : launch<bf16, 128>(c, p, tq, tk, tv, to, stream);
  return c.D <= 64 ? launch<__half, 64>(c, p, tq, tk, tv, to, stream) : launch<__half, 128>(c, p, tq, tk, tv, to, stream);
}

}  // namespace tpf

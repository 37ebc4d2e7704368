// Window attention of few queries over many keys: single tokens over their caches.
//
// Rows are the queries of all heads that share a key head: a tile is 16 of them (queries times heads of the group), so a key
// is read once for the group.  The keys of a tile are split over the CTAs of a cluster and over the warps of each; a warp walks over
// blocks of 16 keys with a running maximum and sum, and the partial results are joined in shared memory, within a CTA and then over the
// cluster, in a fixed order.
//
// What bounds it: the bytes of the keys and values that are seen (10 MFLOP a megabyte at 8 heads a group: the products need the
// tensor cores, but a small part of them, so mma.sync does).  Loads: every warp brings its own blocks by cp.async, kStages deep.
// Measured (B200, bf16, 8 key heads of 128): 18.4 us for 16 sequences that see 1024 keys each (67 MB, 3.7 TB/s), of which 5 are the
// launch, the first loads and the joining; 8 warps, 2 warps or 6 stages were no faster.
#include <cooperative_groups.h>

#include "tpf_window_kernels.h"

namespace tpf {

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 3, kBlock = 16;
constexpr int kMostSplits = 16;  // CTAs of a cluster

template <int DP>
struct FewCfg {
  static constexpr int PITCH = DP * 2 + 16;                 // bytes of a row in shared memory: ldmatrix without conflicts
  static constexpr int TILE = kBlock * PITCH;
  static constexpr int OFF_KV = 0;                          // [warp][stage][K, V]
  static constexpr int OFF_Q = kWarps * kStages * 2 * TILE;
  static constexpr int OFF_O = 0;                           // [16][DP] fp32 a warp, over the keys when they have been used
  static constexpr int OFF_ML = OFF_Q + 16 * PITCH;         // [warp][16] x {m, l}
  static constexpr int OFF_MINE = OFF_ML + kWarps * 16 * 8;  // the CTA's {m, l} [16]
  static constexpr int SMEM = OFF_MINE + 16 * 8;
  static_assert(kWarps * 16 * DP * 4 <= OFF_Q, "");
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, bf16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct FewArgs {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  void* out;
  float* lse;
  int rows, row_tiles, splits;
  FastDiv div_g;
};

// Key of position `i` in the list of a tile's keys: the sinks, then the window.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) window_few_kernel(const WindowParams p, const FewArgs a) {
  griddep_wait();
  using Cfg = FewCfg<DP>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int row0 = tile * 16;
  const int off = p.first_position(b), len = p.length(b);
  const int i0 = (int)a.div_g.div(row0), i1 = (int)a.div_g.div(min(row0 + 15, a.rows - 1));
  const KeyRange kr = key_range(p, len, off + i0, off + i1);
  const int keys = kr.sink + (kr.hi - kr.lo);
  const int blocks = (keys + kBlock - 1) / kBlock;
  const int workers = a.splits * kWarps, me = warp * a.splits + split;  // worker w takes blocks w, w + workers, ...
  const uint32_t s_kv = smem_u32(smem) + Cfg::OFF_KV + warp * kStages * 2 * Cfg::TILE;
  const uint32_t s_q = smem_u32(smem) + Cfg::OFF_Q;
  constexpr int CHUNKS = DP / 8;  // 16-byte pieces of a row

  const T* kbase = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vbase = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  auto load = [&](int block, int stage) {
    uint8_t* dst = smem + Cfg::OFF_KV + (warp * kStages + stage) * 2 * Cfg::TILE;
#pragma unroll
    for (int c = lane; c < kBlock * CHUNKS; c += 32) {
      const int r = c / CHUNKS, col = c % CHUNKS * 8;
      const int i = block * kBlock + r;
      const int key = i < kr.sink ? i : kr.lo + i - kr.sink;
      const bool on = i < keys && col < p.D;  // the rest is zeros: P is zero there, and zero times what lies behind could be a NaN
      const int64_t at = on ? key : 0;
      const int d = on ? col : 0;
      cp_async_16(dst + r * Cfg::PITCH + col * 2, kbase + at * a.ks[1] + d, on);
      cp_async_16(dst + Cfg::TILE + r * Cfg::PITCH + col * 2, vbase + at * a.vs[1] + d, on);
    }
  };

  // queries
  for (int c = threadIdx.x; c < 16 * CHUNKS; c += kThreads) {
    const int r = c / CHUNKS, col = c % CHUNKS * 8;
    const int row = row0 + r;
    const bool on = row < a.rows && col < p.D;
    const int i = on ? (int)a.div_g.div(row) : 0, h = hk * p.G + (on ? row - i * p.G : 0);
    cp_async_16(smem + Cfg::OFF_Q + r * Cfg::PITCH + col * 2,
                static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + (on ? col : 0), on);
  }
  cp_async_commit();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (me + s * workers < blocks) load(me + s * workers, s);
    cp_async_commit();
  }
  cp_async_wait<kStages - 1>();
  __syncthreads();
  uint32_t qf[DP / 16][4];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d)
    ldmatrix_x4(qf[d], s_q + (lane & 15) * Cfg::PITCH + d * 32 + (lane >> 4) * 16);

  // a thread's rows: g and g + 8; their positions
  const int g = lane >> 2, t4 = lane & 3;
  int pos[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) pos[r] = off + (int)a.div_g.div(min(row0 + g + 8 * r, a.rows - 1));
  const float c2 = p.scale * 1.4426950408889634f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[d][e] = 0.f;

  int stage = 0;
  for (int block = me; block < blocks; block += workers) {
    const int ahead = block + (kStages - 1) * workers;
    const int next_stage = stage == 0 ? kStages - 1 : stage - 1;
    __syncwarp();  // every lane has used what lay there
    if (ahead < blocks) load(ahead, next_stage);
    cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const uint32_t sk = s_kv + stage * 2 * Cfg::TILE, sv = sk + Cfg::TILE;
    float s[2][4] = {};
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t kf[4];  // keys 0-7 and 8-15, d 0-7 and 8-15 each
      ldmatrix_x4(kf, sk + ((lane & 7) + (lane >> 4) * 8) * Cfg::PITCH + d * 32 + (lane >> 3 & 1) * 16);
      mma16816<T>(s[0], qf[d], kf[0], kf[1]);
      mma16816<T>(s[1], qf[d], kf[2], kf[3]);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = block * kBlock + n * 8 + 2 * t4 + (e & 1), r = e >> 1;
        const int key = i < kr.sink ? i : kr.lo + i - kr.sink;
        const bool seen = i < keys && key <= pos[r] + p.right && (key >= pos[r] - p.left || key < p.sinks);
        s[n][e] = seen ? s[n][e] * c2 : -INFINITY;
        top[r] = fmaxf(top[r], s[n][e]);
      }
    uint32_t pf[4], pl[4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float now = fmaxf(m[r], top[r]);
      const float base = now == -INFINITY ? 0.f : now;
      const float f = ex2_approx(m[r] - base);
      m[r] = now;
      float e0 = ex2_approx(s[0][2 * r] - base), e1 = ex2_approx(s[0][2 * r + 1] - base);
      float e2 = ex2_approx(s[1][2 * r] - base), e3 = ex2_approx(s[1][2 * r + 1] - base);
      l[r] = l[r] * f + ((e0 + e1) + (e2 + e3));
      // P as an operand of the matrix instructions: two numbers of v's type, the second what the rounding to the first leaves over
      // (of a few values the sum would show it: error of the output relative to its norm 0.0021 for 0.0017, 17.9 us for 18.4 at 16
      // sequences that see 1024 keys)
      pf[r] = pack2<T>(e0, e1);
      pf[2 + r] = pack2<T>(e2, e3);
      const float2 h0 = unpack2<T>(pf[r]), h1 = unpack2<T>(pf[2 + r]);
      pl[r] = pack2<T>(e0 - h0.x, e1 - h0.y);
      pl[2 + r] = pack2<T>(e2 - h1.x, e3 - h1.y);
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        o[d][2 * r] *= f;
        o[d][2 * r + 1] *= f;
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t vf[4];  // keys 0-7, 8-15 of d 0-7, then of d 8-15
      ldmatrix_x4_trans(vf, sv + (lane & 15) * Cfg::PITCH + d * 32 + (lane >> 4) * 16);
      mma16816<T>(o[2 * d], pf, vf[0], vf[1]);
      mma16816<T>(o[2 * d + 1], pf, vf[2], vf[3]);
      mma16816<T>(o[2 * d], pl, vf[0], vf[1]);
      mma16816<T>(o[2 * d + 1], pl, vf[2], vf[3]);
    }
    if (++stage == kStages) stage = 0;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  cp_async_wait<0>();
  __syncthreads();  // the keys' memory is free
  float* so = reinterpret_cast<float*>(smem + Cfg::OFF_O) + warp * 16 * DP;
  float2* ml = reinterpret_cast<float2*>(smem + Cfg::OFF_ML);
  float2* mine = reinterpret_cast<float2*>(smem + Cfg::OFF_MINE);
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(so + (g + 8 * r) * DP + d * 8 + 2 * t4) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
  if (t4 == 0) {
    ml[warp * 16 + g] = make_float2(m[0], l[0]);
    ml[warp * 16 + g + 8] = make_float2(m[1], l[1]);
  }
  __syncthreads();
  // the warps' parts -> the CTA's, over warp 0's
  for (int e = threadIdx.x; e < 16 * DP / 4; e += kThreads) {
    const int r = e / (DP / 4);
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[w * 16 + r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    float4* all = reinterpret_cast<float4*>(smem + Cfg::OFF_O);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 x = ml[w * 16 + r];
      const float f = ex2_approx(x.x - base);
      const float4 y = all[w * 16 * DP / 4 + e];
      acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w;
      sum += f * x.y;
    }
    all[e] = acc;
    if (e % (DP / 4) == 0) mine[r] = make_float2(top, sum);
  }
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  // the CTAs' parts -> the output: CTA `split` does every splits-th piece
  for (int e = threadIdx.x + split * kThreads; e < 16 * DP / 4; e += a.splits * kThreads) {
    const int r = e / (DP / 4), d = e % (DP / 4) * 4;
    float top = -INFINITY;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, cluster.map_shared_rank(mine, s)[r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const float2 x = cluster.map_shared_rank(mine, s)[r];
      const float f = ex2_approx(x.x - base);
      const float4 y = cluster.map_shared_rank(reinterpret_cast<float4*>(smem + Cfg::OFF_O), s)[e];
      acc.x += f * y.x, acc.y += f * y.y, acc.z += f * y.z, acc.w += f * y.w;
      sum += f * x.y;
    }
    const int row = row0 + r;
    if (row < a.rows) {
      const int i = (int)a.div_g.div(row), h = hk * p.G + row - i * p.G;
      const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;  // (a NaN stays one)
      if (d < p.D)
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (((int64_t)b * p.N + i) * p.H + h) * p.D + d) =
            make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      if (d == 0 && a.lse != nullptr)
        a.lse[((int64_t)b * p.H + h) * p.N + i] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
  }
  cluster.sync();  // nobody leaves while its memory is read
}

template <typename T, int DP>
int launch(const WindowParams& p, const FewArgs& a, cudaStream_t stream) {
  using Cfg = FewCfg<DP>;
  auto kern = window_few_kernel<T, DP>;
  static PerDeviceOnce once;
  if (int rc = ensure_dynamic_smem(kern, Cfg::SMEM, once)) return rc;
  if (a.splits > 8) {  // more than a cluster has everywhere
    static PerDeviceOnce wide;
    int dev = 0;
    if (int rc = current_device(&dev)) return rc;
    if (!wide.done[dev].load(std::memory_order_acquire)) {
      TPF_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      wide.done[dev].store(true, std::memory_order_release);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.splits * a.row_tiles, p.HK, p.B);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)a.splits, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, kern, p, a);  // the error is read by TPF_LAUNCH_OK()
  TPF_LAUNCH_OK();
  return TPF_OK;
}

}  // namespace

int window_few(const WindowCall& c, const WindowParams& p, cudaStream_t stream) {
  FewArgs a = {};
  a.q = c.q, a.k = c.k, a.v = c.v;
  for (int i = 0; i < 3; ++i) a.qs[i] = c.qs[i], a.ks[i] = c.ks[i], a.vs[i] = c.vs[i];
  a.out = c.out, a.lse = c.lse;
  TPF_REQUIRE(c.N * p.G < (1ll << 31), TPF_ERR_UNSUPPORTED, "window_attn_fwd: too many queries");
  a.rows = (int)(c.N * p.G);
  a.row_tiles = (a.rows + 15) / 16;
  a.div_g = FastDiv::make((uint32_t)p.G);
  // Keys are split over a cluster of up to sixteen CTAs, while no more of them come than find room on the SMs at once (two an SM), and a
  // split keeps at least two blocks a warp.  (One sequence of 32768 keys, 8 key heads: 57 us with eight, 44 with sixteen.)
  const int64_t ctas = c.B * c.HK * a.row_tiles;
  int64_t keys = (int64_t)c.left + c.right + c.N + c.sinks;
  if (keys > c.M) keys = c.M;
  a.splits = 1;
  while (a.splits < kMostSplits && ctas * a.splits * 2 <= 2 * sm_count() && keys >= a.splits * 2 * kWarps * kBlock * 2) a.splits *= 2;
  if (c.type == kRowBF16) return c.D <= 64 ? launch<bf16, 64>(p, a, stream) : launch<bf16, 128>(p, a, stream);
  return c.D <= 64 ? launch<__half, 64>(p, a, stream) : launch<__half, 128>(p, a, stream);
}

}  // namespace tpf

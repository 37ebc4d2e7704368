// Position rotation of the heads of q and k, with or without an RMS norm of every head in the same pass; forward and backward.
//
//   y = x rsqrt(mean(x^2) + eps) w             (y = x without a norm)
//   pair i of the first R elements:  (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = position * f_i
//   backward: g = the inverse rotation of dz (times m);  t = g w;  dx = r (t - x r^2 sum(t x) / D);  dw = sum of g x r
//
// Angles: f_i comes as turns a position in 64-bit fixed point, the product with the position modulo 2^64 is the phase modulo a
// turn, exactly, and its upper 32 bits go to sincospi.  So a position of a million is as exact as position one, without a
// table in memory and without arithmetic in 64-bit floats.
//
// Mapping: a team of TL lanes takes a token and a run of its heads.  A lane holds two pieces of eight elements: in the half
// order the two that are rotated into one another, so nothing is exchanged, and its sines and cosines stay in registers for
// all heads of the run (sincospi costs as much as a head).  What bounds it: memory (the smallest calls: the launch).
// Head sizes that are no multiple of eight, and halves that no piece fits, take a warp per head with single elements and pass
// partners through shared memory.
#include "tpf_rotary.h"

#include "tpf_rows.cuh"
#include "tpf_rows.h"

namespace tpf {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct RotaryParams {
  struct Tensor {
    const void *x, *dy;
    void* out;
    int64_t sb, sn, sh;
    int heads, runs, run;       // runs of `run` heads
    int64_t first_item;         // items: (token, run)
    ParamVec w;
    bool want_dw;
  } t[2];
  int64_t items, rows;          // rows = batch * tokens
  int tokens, dim, rot;
  const int64_t* turns;
  const int64_t* positions;
  int64_t first;
  float magnitude, eps, inv_dim;
  float* terms;                 // [grid][2][dim]
};

// A lane's elements: VEC = 8: pieces at at[0] and at[1], eight each; VEC = 1: element lane + 32 i.
template <int VEC, int TL, bool HALF>
struct Place {
  static constexpr int E = VEC == 8 ? 16 : 8, PIECES = VEC == 8 ? 2 : 8;
  int at[PIECES];
  bool on[PIECES];
  __device__ __forceinline__ Place(int lane, const RotaryParams& p) {
    if constexpr (VEC == 8) {
      // half order: lanes up to R / 16 hold partners, the rest of the head follows two pieces a lane
      const int pairs = p.rot / 16, pieces = p.dim / 8;
      const int a = !HALF || lane < pairs ? lane : 2 * lane;
      const int b = !HALF ? lane + TL : lane < pairs ? lane + pairs : a + 1;
      on[0] = a < pieces;
      on[1] = b < pieces;
      at[0] = on[0] ? 8 * a : 0;
      at[1] = on[1] ? 8 * b : 0;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        on[i] = lane + 32 * i < p.dim;
        at[i] = on[i] ? lane + 32 * i : 0;
      }
    }
  }
};

__device__ __forceinline__ void cos_sin(uint64_t turns, int64_t position, float magnitude, float& c, float& s) {
  const uint64_t phase = turns * (uint64_t)position;
  sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);  // half turns, -1 .. 1
  c *= magnitude;
  s *= magnitude;
}

// Cosines and sines of a lane's elements: VEC = 8: of the eight pairs it holds (HALF: element j of both pieces; else pairs 0-3 in the
// first piece, 4-7 in the second); VEC = 1: of each element.
template <int VEC, int TL, bool HALF>
struct Angles {
  float c[8], s[8];
  uint32_t turned;  // bit j: pair (element) j is rotated
  __device__ __forceinline__ void make(const Place<VEC, TL, HALF>& pl, const RotaryParams& p, int64_t position) {
    turned = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      int pair;
      if constexpr (VEC == 8) pair = HALF ? pl.at[0] + j : (pl.at[j >> 2] >> 1) + (j & 3);
      else pair = HALF ? (pl.at[j] < p.rot / 2 ? pl.at[j] : pl.at[j] - p.rot / 2) : pl.at[j] >> 1;
      const bool is = VEC == 8 ? pl.on[HALF ? 0 : j >> 2] && pair < p.rot / 2 : pl.on[j] && pl.at[j] < p.rot;
      c[j] = 1.f;
      s[j] = 0.f;
      if (is) {
        turned |= 1u << j;
        cos_sin((uint64_t)__ldg(p.turns + pair), position, p.magnitude, c[j], s[j]);
      }
    }
  }
};

// Rotates a lane's elements; SIGN = -1: back.  `row`: 256 floats of the warp (VEC = 1 only).
template <int VEC, int TL, bool HALF, int SIGN>
__device__ __forceinline__ void turn(float (&y)[Place<VEC, TL, HALF>::E], const Place<VEC, TL, HALF>& pl,
                                     const Angles<VEC, TL, HALF>& an, const RotaryParams& p, float* row) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int ia = HALF ? j : 2 * j, ib = HALF ? j + 8 : 2 * j + 1;
      const float a = y[ia], b = y[ib], s = SIGN * an.s[j];
      const float na = a * an.c[j] - b * s, nb = fmaf(a, s, b * an.c[j]);
      if (an.turned >> j & 1u) {  // (an infinity next to elements that stay must not reach them)
        y[ia] = na;
        y[ib] = nb;
      }
    }
  } else {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) row[lane + 32 * i] = y[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(an.turned >> i & 1u)) continue;
      const bool is_a = HALF ? pl.at[i] < p.rot / 2 : (pl.at[i] & 1) == 0;
      const int partner = HALF ? (is_a ? pl.at[i] + p.rot / 2 : pl.at[i] - p.rot / 2) : pl.at[i] ^ 1;
      const float o = row[partner], s = SIGN * an.s[i];
      y[i] = is_a ? y[i] * an.c[i] - o * s : fmaf(o, s, y[i] * an.c[i]);
    }
  }
}

template <typename T, int VEC, int TL, bool HALF>
struct Head {  // a lane's part of a head as it lies in memory
  using Pl = Place<VEC, TL, HALF>;
  Piece<T, VEC> p[Pl::PIECES];
  __device__ __forceinline__ void load(const T* x, const Pl& pl) {
#pragma unroll
    for (int i = 0; i < Pl::PIECES; ++i) p[i].load(x + pl.at[i]);
  }
  __device__ __forceinline__ void get(float (&v)[Pl::E], const Pl& pl) const {
#pragma unroll
    for (int i = 0; i < Pl::PIECES; ++i) {
      p[i].get(v + i * VEC);
      if (!pl.on[i])
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i * VEC + j] = 0.f;
    }
  }
};
template <typename T, int VEC, class Pl>
__device__ __forceinline__ void put(T* out, const float* v, const Pl& pl) {
#pragma unroll
  for (int i = 0; i < Pl::PIECES; ++i)
    if (pl.on[i]) store_vec<T, VEC>(out + pl.at[i], v + i * VEC);
}
template <int VEC, class Pl>
__device__ __forceinline__ void weights(const ParamVec& w, float (&v)[Pl::E], const Pl& pl, int dim) {
#pragma unroll
  for (int i = 0; i < Pl::PIECES; ++i) {
    param_load<VEC, 1>(w, pl.at[i], dim, 1.f, v + i * VEC);
    if (!pl.on[i])
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i * VEC + j] = 0.f;
  }
}

struct Item {
  int64_t row;
  int head, heads;
};
__device__ __forceinline__ Item item_of(const RotaryParams::Tensor& t, int64_t i) {
  const uint32_t row = (uint32_t)i / (uint32_t)t.runs, run = (uint32_t)i - row * t.runs;
  const int h = (int)run * t.run;
  return {(int64_t)row, h, min(t.run, t.heads - h)};
}
__device__ __forceinline__ int64_t position_of(const RotaryParams& p, int64_t row) {
  return p.positions != nullptr ? __ldg(p.positions + row) : p.first + (int64_t)((uint32_t)row % (uint32_t)p.tokens);
}

template <typename T, int VEC, int TL, bool HALF, bool NORM>
__global__ void __launch_bounds__(kThreads) rotary_fwd_kernel(const RotaryParams p) {
  griddep_wait();
  using Pl = Place<VEC, TL, HALF>;
  __shared__ float exchange[VEC == 1 ? kThreads / 32 : 1][VEC == 1 ? 256 : 1];
  float* row_mem = exchange[VEC == 1 ? threadIdx.x >> 5 : 0];
  const int lane = threadIdx.x % TL;
  const Pl pl(lane, p);
  constexpr int TEAMS = kThreads / TL;
  // (the teams of a warp go through the shuffles together: those without an item repeat the last one)
  const int64_t mine = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TL;
  const bool real = mine < p.items;
  const int64_t i = real ? mine : p.items - 1;
  const bool second = i >= p.t[1].first_item;
  const RotaryParams::Tensor& t = p.t[second ? 1 : 0];
  const Item it = item_of(t, i - t.first_item);
  const int64_t b = (int64_t)((uint32_t)it.row / (uint32_t)p.tokens), n = it.row - b * p.tokens;
  const T* x = static_cast<const T*>(t.x) + b * t.sb + n * t.sn + it.head * t.sh;
  T* out = static_cast<T*>(t.out) + (it.row * t.heads + it.head) * p.dim;
  Head<T, VEC, TL, HALF> cur, next;
  cur.load(x, pl);
  Angles<VEC, TL, HALF> an;
  an.make(pl, p, position_of(p, it.row));
  float w[Pl::E];
  if (NORM) weights<VEC, Pl>(t.w, w, pl, p.dim);
  const int heads = __reduce_max_sync(0xffffffffu, it.heads);
  for (int h = 0; h < heads; ++h) {
    const bool live = h < it.heads;
    if (h + 1 < it.heads) next.load(x + t.sh, pl);
    float y[Pl::E];
    cur.get(y, pl);
    if (NORM) {
      float ss[1] = {0.f};
#pragma unroll
      for (int e = 0; e < Pl::E; ++e) ss[0] = fmaf(y[e], y[e], ss[0]);
      warp_sum(ss, TL);
      const float r = rsqrtf(fmaf(ss[0], p.inv_dim, p.eps));
#pragma unroll
      for (int e = 0; e < Pl::E; ++e) y[e] = y[e] * r * w[e];
    }
    turn<VEC, TL, HALF, 1>(y, pl, an, p, row_mem);
    if (real && live) put<T, VEC>(out, y, pl);
    cur = next;
    x += t.sh;
    out += p.dim;
  }
}

// A block walks over the items of one tensor after the other, so that a thread's sums of dw belong to one weight at a time; the teams'
// sums are added in shared memory in the order of the teams and leave as one term a block, which norm_fold adds up.
template <typename T, int VEC, int TL, bool HALF, bool NORM>
__global__ void __launch_bounds__(kThreads, NORM ? 2 : 3) rotary_bwd_kernel(const RotaryParams p) {
  griddep_wait();
  using Pl = Place<VEC, TL, HALF>;
  __shared__ float exchange[VEC == 1 ? kThreads / 32 : 1][VEC == 1 ? 256 : 1];
  __shared__ float sums[NORM ? kThreads / 32 : 1][NORM ? kMaxDim : 1];
  float* row_mem = exchange[VEC == 1 ? threadIdx.x >> 5 : 0];
  const int lane = threadIdx.x % TL;
  const Pl pl(lane, p);
  constexpr int TEAMS = kThreads / TL;
  for (int k = 0; k < 2; ++k) {
    const RotaryParams::Tensor& t = p.t[k];
    const int64_t items = k == 0 ? p.t[1].first_item : p.items - p.t[1].first_item;
    float w[Pl::E], dw[Pl::E];
#pragma unroll
    for (int e = 0; e < Pl::E; ++e) dw[e] = 0.f;
    if (NORM) weights<VEC, Pl>(t.w, w, pl, p.dim);
    for (int64_t base = (int64_t)blockIdx.x * TEAMS; base < items; base += (int64_t)gridDim.x * TEAMS) {
      const int64_t mine = base + threadIdx.x / TL;
      const bool real = mine < items;
      const Item it = item_of(t, real ? mine : items - 1);
      const int64_t b = (int64_t)((uint32_t)it.row / (uint32_t)p.tokens), n = it.row - b * p.tokens;
      const T* x = NORM ? static_cast<const T*>(t.x) + b * t.sb + n * t.sn + it.head * t.sh : nullptr;
      const int64_t at = (it.row * t.heads + it.head) * p.dim;
      const T* dy = static_cast<const T*>(t.dy) + at;
      T* out = static_cast<T*>(t.out) + at;
      Head<T, VEC, TL, HALF> cx, cg, nx, ng;
      if (NORM) cx.load(x, pl);
      cg.load(dy, pl);
      Angles<VEC, TL, HALF> an;
      an.make(pl, p, position_of(p, it.row));
      const int heads = __reduce_max_sync(0xffffffffu, it.heads);
      for (int h = 0; h < heads; ++h) {
        const bool live = real && h < it.heads;
        if (h + 1 < it.heads) {
          if (NORM) nx.load(x + t.sh, pl);
          ng.load(dy + p.dim, pl);
        }
        float g[Pl::E];
        cg.get(g, pl);
        turn<VEC, TL, HALF, -1>(g, pl, an, p, row_mem);
        if (NORM) {
          float v[Pl::E], s[2] = {0.f, 0.f};
          cx.get(v, pl);
#pragma unroll
          for (int e = 0; e < Pl::E; ++e) {
            s[0] = fmaf(v[e], v[e], s[0]);
            s[1] = fmaf(g[e] * w[e], v[e], s[1]);
          }
          warp_sum(s, TL);
          const float r = rsqrtf(fmaf(s[0], p.inv_dim, p.eps)), m = s[1] * p.inv_dim * r * r;
#pragma unroll
          for (int e = 0; e < Pl::E; ++e) {
            if (live) dw[e] = fmaf(g[e], v[e] * r, dw[e]);
            g[e] = r * fmaf(-v[e], m, g[e] * w[e]);
          }
        }
        if (live) put<T, VEC>(out, g, pl);
        if (NORM) cx = nx;
        cg = ng;
        if (NORM) x += t.sh;
        dy += p.dim;
        out += p.dim;
      }
    }
    if constexpr (NORM) {
      if (p.terms != nullptr) {
        // teams of a warp by shuffles, then the warps
#pragma unroll
        for (int off = 16; off >= TL; off >>= 1)
#pragma unroll
          for (int e = 0; e < Pl::E; ++e) dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], off);
        if ((threadIdx.x & 31) < TL) {
#pragma unroll
          for (int i = 0; i < Pl::PIECES; ++i)
            if (pl.on[i])
#pragma unroll
              for (int j = 0; j < VEC; ++j) sums[threadIdx.x >> 5][pl.at[i] + j] = dw[i * VEC + j];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.dim; c += kThreads) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < kThreads / 32; ++i) s += sums[i][c];
          p.terms[((int64_t)blockIdx.x * 2 + k) * p.dim + c] = s;
        }
        __syncthreads();
      }
    }
  }
}

constexpr int kTermBlocks = 2 * 148;  // blocks of a backward pass with a norm

template <typename T, int VEC, int TL, bool HALF>
int launch(const RotaryCall& c, RotaryParams& p, bool back, cudaStream_t stream) {
  constexpr int TEAMS = kThreads / TL;
  // Runs of heads: as long as there are about a thousand threads an SM left, so that sines and cosines are used often.
  const int64_t want = (int64_t)sm_count() * 1024 / TL;
  int64_t items = 0;
  for (int k = 0; k < 2; ++k) {
    RotaryParams::Tensor& t = p.t[k];
    const int64_t total = c.t[0].heads + c.t[1].heads;
    int64_t runs_all = (want + p.rows - 1) / p.rows;  // a token is cut into this many
    if (runs_all > total) runs_all = total;
    t.run = (int)((total + runs_all - 1) / runs_all);
    if (t.heads > 0 && t.run > t.heads) t.run = t.heads;
    t.runs = t.heads > 0 ? (t.heads + t.run - 1) / t.run : 1;
    t.first_item = items;
    items += t.heads > 0 ? p.rows * t.runs : 0;
  }
  p.items = items;
  TPF_REQUIRE(items < (1ll << 31) - kThreads, TPF_ERR_UNSUPPORTED, "rotary: too many heads");
  const int64_t blocks = (items + TEAMS - 1) / TEAMS;
  if (!back) {
    if (c.norm) launch_kernel(rotary_fwd_kernel<T, VEC, TL, HALF, true>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
    else launch_kernel(rotary_fwd_kernel<T, VEC, TL, HALF, false>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
    TPF_LAUNCH_OK();
    return TPF_OK;
  }
  if (!c.norm) {
    launch_kernel(rotary_bwd_kernel<T, VEC, TL, HALF, false>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
    TPF_LAUNCH_OK();
    return TPF_OK;
  }
  const int grid = blocks < kTermBlocks ? (int)blocks : kTermBlocks;
  launch_kernel(rotary_bwd_kernel<T, VEC, TL, HALF, true>, dim3(grid), dim3(kThreads), 0, stream, p);
  TPF_LAUNCH_OK();
  if (p.terms == nullptr) return TPF_OK;
  return norm_fold(p.terms, grid, p.dim, c.t[0].dweight, c.t[0].weight_type, c.t[1].dweight, c.t[1].weight_type, stream);
}
template <typename T, int VEC, int TL>
int launch(const RotaryCall& c, RotaryParams& p, bool back, cudaStream_t stream) {
  return c.half ? launch<T, VEC, TL, true>(c, p, back, stream) : launch<T, VEC, TL, false>(c, p, back, stream);
}
template <typename T>
int launch(const RotaryCall& c, RotaryParams& p, bool vec, bool back, cudaStream_t stream) {
  if (!vec) return launch<T, 1, 32>(c, p, back, stream);
  const int lanes = (int)(c.dim / 8 + 1) / 2;
  if (lanes <= 2) return launch<T, 8, 2>(c, p, back, stream);
  if (lanes <= 4) return launch<T, 8, 4>(c, p, back, stream);
  if (lanes <= 8) return launch<T, 8, 8>(c, p, back, stream);
  return launch<T, 8, 16>(c, p, back, stream);
}

int run(const RotaryCall& c, void* workspace, int64_t workspace_bytes, bool back, cudaStream_t stream) {
  const char* who = back ? "rotary_bwd" : "rotary_fwd";
  TPF_REQUIRE(row_type_ok(c.type), TPF_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", who, c.type);
  TPF_REQUIRE(c.batch >= 0 && c.tokens >= 0 && c.t[0].heads >= 0 && c.t[1].heads >= 0, TPF_ERR_INVALID_ARGUMENT,
              "%s: extents must not be negative", who);
  TPF_REQUIRE(c.dim >= 2 && c.dim <= kMaxDim, TPF_ERR_UNSUPPORTED, "%s: heads of 2 to %d elements", who, kMaxDim);
  TPF_REQUIRE(c.rot >= 2 && c.rot % 2 == 0 && c.rot <= c.dim, TPF_ERR_INVALID_ARGUMENT,
              "%s: the rotated part must be even and at most a head", who);
  const int64_t total = c.t[0].heads + c.t[1].heads;
  const bool none = c.batch == 0 || c.tokens == 0 || total == 0;
  bool want_dw = false;
  for (int k = 0; k < 2; ++k) {
    TPF_REQUIRE(c.t[k].weight == nullptr || row_type_ok(c.t[k].weight_type), TPF_ERR_INVALID_ARGUMENT,
                "%s: unknown type of a weight", who);
    want_dw = want_dw || (back && c.t[k].dweight != nullptr);
    TPF_REQUIRE(c.t[k].dweight == nullptr || (c.norm && row_type_ok(c.t[k].weight_type)), TPF_ERR_INVALID_ARGUMENT,
                "%s: a weight's gradient without a norm", who);
  }
  if (none) {
    for (int k = 0; k < 2; ++k)
      if (back && c.t[k].dweight != nullptr)
        TPF_CUDA_OK(cudaMemsetAsync(c.t[k].dweight, 0, (size_t)c.dim * row_type_size(c.t[k].weight_type), stream));
    return TPF_OK;
  }
  TPF_REQUIRE(c.batch < (1ll << 31) && c.tokens < (1ll << 31) && total < (1 << 24) && c.batch * c.tokens < (1ll << 31),
              TPF_ERR_UNSUPPORTED, "%s: too many tokens", who);
  TPF_REQUIRE(c.turns != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  RotaryParams p = {};
  p.rows = c.batch * c.tokens;
  p.tokens = (int)c.tokens, p.dim = (int)c.dim, p.rot = (int)c.rot;
  p.turns = c.turns, p.positions = c.positions, p.first = c.first;
  p.magnitude = c.magnitude, p.eps = c.eps, p.inv_dim = 1.f / (float)c.dim;
  bool vec = c.dim % 8 == 0 && (!c.half || c.rot % 16 == 0);
  for (int k = 0; k < 2; ++k) {
    const RotaryTensor& s = c.t[k];
    RotaryParams::Tensor& t = p.t[k];
    t.heads = (int)s.heads;
    if (s.heads == 0) continue;
    const bool reads_x = !back || c.norm;
    TPF_REQUIRE((s.x != nullptr || !reads_x) && s.out != nullptr && (s.dy != nullptr || !back), TPF_ERR_INVALID_ARGUMENT,
                "%s: null pointer", who);
    t.x = s.x, t.dy = s.dy, t.out = s.out;
    t.sb = s.strides[0], t.sn = s.strides[1], t.sh = s.strides[2];
    t.w = {s.weight, s.weight_type};
    vec = vec && vec_ok(s.out, c.type) && (!back || vec_ok(s.dy, c.type));
    if (reads_x)
      vec = vec && vec_ok(s.x, c.type) && (c.batch == 1 || t.sb % 8 == 0) && (c.tokens == 1 || t.sn % 8 == 0) &&
            (s.heads == 1 || t.sh % 8 == 0);
  }
  if (want_dw) {
    TPF_REQUIRE(workspace != nullptr && workspace_bytes >= rotary_bwd_workspace_bytes(c.dim), TPF_ERR_WORKSPACE,
                "%s: the workspace is too small", who);
    TPF_REQUIRE_ALIGNED16(workspace, who, "workspace");
    p.terms = static_cast<float*>(workspace);
  }
  if (c.type == kRowF32) return launch<float>(c, p, vec, back, stream);
  if (c.type == kRowBF16) return launch<bf16>(c, p, vec, back, stream);
  return launch<__half>(c, p, vec, back, stream);
}

}  // namespace

int rotary_fwd(const RotaryCall& c, cudaStream_t stream) { return run(c, nullptr, 0, false, stream); }
int64_t rotary_bwd_workspace_bytes(int64_t dim) { return dim > 0 && dim <= kMaxDim ? (int64_t)kTermBlocks * 2 * dim * 4 : 0; }
int rotary_bwd(const RotaryCall& c, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  return run(c, workspace, workspace_bytes, true, stream);
}

}  // namespace tpf

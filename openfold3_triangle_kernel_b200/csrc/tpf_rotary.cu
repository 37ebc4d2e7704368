// Position rotation of the heads of q and k, with or without an RMS norm of every head in the same pass; forward and backward.
//
//   y = x rsqrt(mean(x^2) + eps) w             (y = x without a norm)
//   pair i of the first R elements:  (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = position * f_i
//   backward: g = the inverse rotation of dz (times m);  t = g w;  dx = r (t - x r^2 sum(t x) / D);  dw = sum of g x r
//
// Angles: f_i comes as turns a position in 64-bit fixed point, the product with the position modulo 2^64 is the phase modulo a
// turn, exactly, and its upper 32 bits, rounded to fp32 (by 2^-26 of a turn at most), go to sincospi.  So a position of a million is as
// exact as position one, without a table in memory and without arithmetic in 64-bit floats.
//
// Mapping: a block has a stretch of tokens, as long as any other block's.  It makes their sines and cosines, in shared memory, and goes
// through the heads of q and then through those of k: a team of TL lanes has a few of them in succession, loaded two ahead.  With the
// sines as registers of each team they were made several times over, and took the place of loads in flight (8192 tokens, 32 + 8
// heads of 128, bf16, with norms, forward and backward: 44 and 75 us, now 36 and 51; 32 heads without norms 32, now 23).  A lane holds two pieces of eight elements, in the half order the two that are
// rotated into one another, so nothing is exchanged.
// What bounds it: memory (the smallest calls: the launch).
// Halves that no piece of eight fits pass partners through shared memory, element by element; head sizes that are no multiple of eight and
// misaligned tensors take a warp per head, with single elements.  Both are served, not fast (bf16, norms, forward and backward, us, in
// brackets the bytes at the rate of a copy): 4099 tokens of 16 + 8 heads of 96, R = 24: 20 and 29 (5.8 and 8.7); 8192 of 16 + 4 heads
// of 126: 88 and 121 (12.6 and 18.9), of 128 from an odd element on 87 and 150.
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
    int heads;
    ParamVec w;
  } t[2];
  uint32_t all;                 // tokens of all batches
  uint32_t per_block, step;     // tokens of a block, and of a step of it
  int tokens, dim, rot, pairs;  // pairs = rot / 2
  const int64_t* turns;
  const int64_t* positions;
  int64_t first;
  float magnitude, eps, inv_dim;
  float* terms;                 // [grid][2][dim]
  FastDiv div_pairs;
};

// How a head is rotated, and by whom:
//   kInterleaved, kHalf  a lane has both elements of its pairs (kHalf: rot / 16 lanes with a piece of either half)
//   kHalfAny             halves that no piece of eight fits: pieces in order, partners through shared memory
enum Mode : int { kInterleaved = 0, kHalf = 1, kHalfAny = 2 };

// A lane's elements: VEC = 8: pieces at at[0] and at[1], eight each; VEC = 1: element lane + 32 i.
template <int VEC, int TL, int MODE>
struct Place {
  static constexpr int E = VEC == 8 ? 16 : 8, PIECES = VEC == 8 ? 2 : 8;
  int at[PIECES];
  bool on[PIECES];
  __device__ __forceinline__ Place(int lane, const RotaryParams& p) {
    if constexpr (VEC == 8) {
      // kHalf: lanes up to R / 16 hold partners, the rest of the head follows two pieces a lane
      const int pairs = p.rot / 16, pieces = p.dim / 8;
      const int a = MODE != kHalf || lane < pairs ? lane : 2 * lane;
      const int b = MODE != kHalf ? lane + TL : lane < pairs ? lane + pairs : a + 1;
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

__device__ __forceinline__ float2 cos_sin(uint64_t turns, int64_t position, float magnitude) {
  const uint64_t phase = turns * (uint64_t)position;
  float c, s;
  sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &s, &c);  // half turns, -1 .. 1
  return make_float2(c * magnitude, s * magnitude);
}

// Sines and cosines of a token in shared memory: all cosines, then all sines, `pitch` numbers each.  In the half order a lane takes
// eight pairs at once: those of even fours lie before those of odd ones, so that the 16-byte reads of neighbours meet no bank twice.
__host__ __device__ constexpr int angle_pitch(int pairs) { return (pairs + 7) / 8 * 8; }
template <int VEC, int MODE>
__device__ __forceinline__ int angle_slot(int pair, int pitch) {
  return VEC == 8 && MODE == kHalf ? (pair >> 2 & 1) * (pitch / 2) + (pair >> 3) * 4 + (pair & 3) : pair;
}

// Rotates a lane's elements; SIGN = -1: back.  `angles`: of the token; `row`: 256 floats of the team, where partners are exchanged.
template <int VEC, int TL, int MODE, int SIGN>
__device__ __forceinline__ void turn(float (&y)[Place<VEC, TL, MODE>::E], const Place<VEC, TL, MODE>& pl, const RotaryParams& p,
                                     const float* angles, float* row) {
  const int pitch = angle_pitch(p.pairs);
  if constexpr (VEC == 8 && MODE == kHalf) {
    if (pl.on[0] && pl.at[0] < p.pairs) {
#pragma unroll
      for (int f = 0; f < 2; ++f) {  // four pairs, two at a time
        const int slot = angle_slot<VEC, MODE>(pl.at[0] + 4 * f, pitch);
        const float4 c = *reinterpret_cast<const float4*>(angles + slot);
        const float4 s = *reinterpret_cast<const float4*>(angles + pitch + slot);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* a = y + 4 * f + 2 * j;
          float* b = a + 8;
          const uint64_t a2 = f2_pack(a[0], a[1]), b2 = f2_pack(b[0], b[1]);
          const uint64_t c2 = j == 0 ? f2_pack(c.x, c.y) : f2_pack(c.z, c.w);
          const uint64_t s2 = SIGN > 0 ? (j == 0 ? f2_pack(s.x, s.y) : f2_pack(s.z, s.w))
                                       : (j == 0 ? f2_pack(-s.x, -s.y) : f2_pack(-s.z, -s.w));
          const uint64_t n2 = SIGN > 0 ? (j == 0 ? f2_pack(-s.x, -s.y) : f2_pack(-s.z, -s.w))
                                       : (j == 0 ? f2_pack(s.x, s.y) : f2_pack(s.z, s.w));
          f2_unpack(f2_fma(b2, n2, f2_mul(a2, c2)), a[0], a[1]);
          f2_unpack(f2_fma(a2, s2, f2_mul(b2, c2)), b[0], b[1]);
        }
      }
    }
  } else if constexpr (VEC == 8 && MODE == kInterleaved) {
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int pair = pl.at[f] >> 1;
      if (!pl.on[f] || pair >= p.pairs) continue;
      const float4 c4 = *reinterpret_cast<const float4*>(angles + pair);
      const float4 s4 = *reinterpret_cast<const float4*>(angles + pitch + pair);
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float &a = y[8 * f + 2 * j], &b = y[8 * f + 2 * j + 1];
        const float na = fmaf(a, c[j], -SIGN * (b * s[j])), nb = fmaf(a, SIGN * s[j], b * c[j]);
        if (pair + j < p.pairs) {  // (an infinity next to elements that stay must not reach them)
          a = na;
          b = nb;
        }
      }
    }
  } else {
    __syncwarp();
    if constexpr (VEC == 8) {
#pragma unroll
      for (int f = 0; f < 4; ++f)
        if (pl.on[f / 2])
          *reinterpret_cast<float4*>(row + pl.at[f / 2] + f % 2 * 4) = make_float4(y[4 * f], y[4 * f + 1], y[4 * f + 2], y[4 * f + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (pl.on[i]) row[pl.at[i]] = y[i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < Place<VEC, TL, MODE>::E; ++i) {
      const int at = pl.at[i / VEC] + i % VEC;
      if (!pl.on[i / VEC] || at >= p.rot) continue;
      const bool is_a = MODE == kInterleaved ? (at & 1) == 0 : at < p.pairs;
      const int pair = MODE == kInterleaved ? at >> 1 : is_a ? at : at - p.pairs;
      const float c = angles[pair], s = SIGN * angles[pitch + pair];
      const float o = row[MODE == kInterleaved ? at ^ 1 : is_a ? at + p.pairs : pair];
      y[i] = is_a ? fmaf(y[i], c, -(o * s)) : fmaf(o, s, y[i] * c);
    }
  }
}

template <typename T, int VEC, int TL, int MODE>
struct Head {  // a lane's part of a head as it lies in memory
  using Pl = Place<VEC, TL, MODE>;
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
// The weights in shared memory, even fours before odd ones (as the angles of the half order).
template <int VEC>
__device__ __forceinline__ int weight_slot(int c) {
  return VEC == 8 ? (c >> 2 & 1) * (kMaxDim / 2) + (c >> 3) * 4 + (c & 3) : c;
}
template <int VEC, class Pl>
__device__ __forceinline__ void weights(const float* mem, float (&w)[Pl::E], const Pl& pl) {
  if constexpr (VEC == 8) {
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const float4 x = *reinterpret_cast<const float4*>(mem + weight_slot<VEC>(pl.at[f / 2] + f % 2 * 4));
      w[4 * f] = x.x, w[4 * f + 1] = x.y, w[4 * f + 2] = x.z, w[4 * f + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = mem[pl.at[i]];
  }
}

__device__ __forceinline__ int64_t position_of(const RotaryParams& p, uint32_t token) {
  return p.positions != nullptr ? __ldg(p.positions + token) : p.first + (int64_t)(token % (uint32_t)p.tokens);
}

// Where a team's rows lie in a strided tensor, one after the other.
template <typename T>
struct Walk {
  const T* x;
  int64_t row0;    // offset of the token
  int n, head;
  const RotaryParams::Tensor& t;
  const int tokens;
  __device__ __forceinline__ Walk(const RotaryParams::Tensor& t_, int tokens_, uint32_t token, int head_)
      : head(head_), t(t_), tokens(tokens_) {
    const uint32_t b = token / (uint32_t)tokens;
    n = (int)(token - b * tokens);
    row0 = (int64_t)b * t.sb + (int64_t)n * t.sn;
    x = static_cast<const T*>(t.x) + row0 + head * t.sh;
  }
  __device__ __forceinline__ void next() {
    x += t.sh;
    if (++head < t.heads) return;
    head = 0;
    row0 += t.sn;
    if (++n == tokens) {
      n = 0;
      row0 += t.sb - (int64_t)tokens * t.sn;
    }
    x = static_cast<const T*>(t.x) + row0;
  }
};

template <typename T>
constexpr int blocks_per_sm(bool norm) {
  return sizeof(T) == 4 || norm ? 2 : 3;
}

// BACK, with a norm: a block's sums of dw leave as one term for each tensor (the teams' sums are added in their order), which
// norm_fold adds up.
template <typename T, int VEC, int TL, int MODE, bool NORM, bool BACK>
__global__ void __launch_bounds__(kThreads, blocks_per_sm<T>(NORM)) rotary_kernel(const RotaryParams p) {
  griddep_wait();
  using Pl = Place<VEC, TL, MODE>;
  using Hd = Head<T, VEC, TL, MODE>;
  constexpr int TEAMS = kThreads / TL;
  constexpr bool READ_X = NORM || !BACK;
  constexpr int AHEAD = sizeof(T) == 4 || (NORM && BACK) ? 1 : 2;  // rows on their way, as many as find registers
  extern __shared__ __align__(16) float angles[];
  constexpr bool EXCHANGE = VEC == 1 || MODE == kHalfAny;
  __shared__ __align__(16) float exchange[EXCHANGE ? TEAMS : 1][EXCHANGE ? (VEC == 1 ? 256 : 16 * TL) : 4];
  __shared__ float sums[NORM && BACK ? kThreads / 32 : 1][NORM && BACK ? kMaxDim : 1];
  __shared__ __align__(16) float wsm[NORM ? kMaxDim : 4];
  float* row_mem = exchange[EXCHANGE ? threadIdx.x / TL : 0];
  const int lane = threadIdx.x % TL, team = threadIdx.x / TL;
  const Pl pl(lane, p);
  const int pitch = angle_pitch(p.pairs);
  const uint32_t begin = min(p.all, blockIdx.x * p.per_block), end = min(p.all, begin + p.per_block);
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const RotaryParams::Tensor& t = p.t[k];
    if (t.heads == 0) continue;
    float dw[Pl::E];
#pragma unroll
    for (int e = 0; e < Pl::E; ++e) dw[e] = 0.f;
    if (NORM) {
      __syncthreads();
      for (int c = threadIdx.x; c < p.dim; c += kThreads) {
        float x[1];
        param_load<1, 1>(t.w, c, p.dim, 1.f, x);
        wsm[weight_slot<VEC>(c)] = x[0];
      }
    }
#pragma unroll 1
    for (uint32_t token0 = begin; token0 < end; token0 += p.step) {
      const uint32_t tokens = min(end - token0, p.step), rows = tokens * t.heads;
      const uint32_t run = (rows + TEAMS - 1) / TEAMS;  // rows of a team
      const uint32_t mine = min(team * run, rows - 1);   // a team without rows stands at the last one
      const int count = team * run < rows ? (int)min(run, rows - mine) : 0;
      const uint32_t token = mine / (uint32_t)t.heads;
      int head = (int)(mine - token * t.heads);
      // the first rows are on their way while the angles are made
      Walk<T> walk(t, p.tokens, token0 + token, head);
      const int64_t at = ((int64_t)token0 * t.heads + mine) * p.dim;
      const T* dy = BACK ? static_cast<const T*>(t.dy) + at : nullptr;
      Hd xs[AHEAD + 1], gs[AHEAD + 1];
      auto load = [&](Hd& x, Hd& g, int i) {
        if (i >= count) return;
        if (READ_X) {
          x.load(walk.x, pl);
          walk.next();
        }
        if (BACK) {
          g.load(dy, pl);
          dy += p.dim;
        }
      };
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) load(xs[i], gs[i], i);
      if (k == 0 || p.t[0].heads == 0 || p.step < p.per_block) {  // (the angles of a block's only step serve q and k)
        __syncthreads();                                          // those of the step before have been used
        for (uint32_t i = threadIdx.x; i < tokens * p.pairs; i += kThreads) {
          const uint32_t n = p.div_pairs.div(i), pair = i - n * p.pairs;
          const float2 cs = cos_sin((uint64_t)__ldg(p.turns + pair), position_of(p, token0 + n), p.magnitude);
          float* to = angles + n * 2 * pitch + angle_slot<VEC, MODE>(pair, pitch);
          to[0] = cs.x;
          to[pitch] = cs.y;
        }
      }
      __syncthreads();
      const float* an = angles + token * 2 * pitch;
      T* out = static_cast<T*>(t.out) + at;
      const int most = __reduce_max_sync(0xffffffffu, count);
      auto row = [&](const Hd& x, const Hd& g, int i) {
        float y[Pl::E];
        if constexpr (!BACK) {
          x.get(y, pl);
          if (NORM) {
            uint64_t sq = 0;
#pragma unroll
            for (int e = 0; e < Pl::E; e += 2) {
              const uint64_t v = f2_pack(y[e], y[e + 1]);
              sq = f2_fma(v, v, sq);
            }
            float ss[1] = {f2_sum(sq)};
            warp_sum(ss, TL);
            const float r = rsqrtf(fmaf(ss[0], p.inv_dim, p.eps));
            const uint64_t r2 = f2_dup(r);
            float w[Pl::E];
            weights<VEC, Pl>(wsm, w, pl);
#pragma unroll
            for (int e = 0; e < Pl::E; e += 2)
              f2_unpack(f2_mul(f2_mul(f2_pack(y[e], y[e + 1]), r2), f2_pack(w[e], w[e + 1])), y[e], y[e + 1]);
          }
          turn<VEC, TL, MODE, 1>(y, pl, p, an, row_mem);
        } else {
          g.get(y, pl);
          turn<VEC, TL, MODE, -1>(y, pl, p, an, row_mem);
          if (NORM) {
            float v[Pl::E], w[Pl::E];
            x.get(v, pl);
            weights<VEC, Pl>(wsm, w, pl);
            uint64_t sq = 0, tx = 0;
#pragma unroll
            for (int e = 0; e < Pl::E; e += 2) {
              const uint64_t x2 = f2_pack(v[e], v[e + 1]);
              sq = f2_fma(x2, x2, sq);
              tx = f2_fma(f2_mul(f2_pack(y[e], y[e + 1]), f2_pack(w[e], w[e + 1])), x2, tx);
            }
            float s[2] = {f2_sum(sq), f2_sum(tx)};
            warp_sum(s, TL);
            const float r = rsqrtf(fmaf(s[0], p.inv_dim, p.eps)), m = s[1] * p.inv_dim * r * r;
            const uint64_t r2 = f2_dup(r), m2 = f2_dup(-m);
#pragma unroll
            for (int e = 0; e < Pl::E; e += 2) {
              const uint64_t x2 = f2_pack(v[e], v[e + 1]), g2 = f2_pack(y[e], y[e + 1]);
              if (i < count) f2_unpack(f2_fma(g2, f2_mul(x2, r2), f2_pack(dw[e], dw[e + 1])), dw[e], dw[e + 1]);
              f2_unpack(f2_mul(r2, f2_fma(x2, m2, f2_mul(g2, f2_pack(w[e], w[e + 1])))), y[e], y[e + 1]);
            }
          }
        }
        if (i < count) put<T, VEC>(out, y, pl);
        out += p.dim;
        if (++head == t.heads) {
          head = 0;
          if (i + 1 < count) an += 2 * pitch;
        }
      };
#pragma unroll 1
      for (int i = 0; i < most; i += AHEAD + 1) {
#pragma unroll
        for (int d = 0; d <= AHEAD; ++d) {
          load(xs[(d + AHEAD) % (AHEAD + 1)], gs[(d + AHEAD) % (AHEAD + 1)], i + d + AHEAD);
          if (d == 0 || i + d < most) row(xs[d], gs[d], i + d);
        }
      }
    }
    if constexpr (NORM && BACK) {
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

constexpr int kTermBlocks = 2 * 148;    // blocks of a backward pass with a norm
constexpr int kAngleBytes = 60 * 1024;  // of a step

template <typename T, int VEC, int TL, int MODE, bool NORM, bool BACK>
struct Kernel {
  static constexpr auto kernel() { return rotary_kernel<T, VEC, TL, MODE, NORM, BACK>; }
};

template <typename T, int VEC, int TL, int MODE>
int launch(const RotaryCall& c, RotaryParams& p, bool back, cudaStream_t stream) {
  constexpr int TEAMS = kThreads / TL;
  // One wave of blocks (as many as find room on the SMs together), or fewer with a row a team.  A block takes its tokens at
  // once, or in steps whose angles find room.
  int most = blocks_per_sm<T>(c.norm) * sm_count();
  if (back && c.norm && most > kTermBlocks) most = kTermBlocks;
  const int64_t heads = c.t[0].heads + c.t[1].heads;
  int64_t grid = ((int64_t)p.all * heads + TEAMS - 1) / TEAMS;
  if (grid > most) grid = most;
  if (grid > p.all) grid = p.all;
  p.per_block = (uint32_t)((p.all + grid - 1) / grid);
  grid = (p.all + p.per_block - 1) / p.per_block;
  const uint32_t fit = kAngleBytes / (2 * angle_pitch(p.pairs) * 4);
  p.step = p.per_block < fit ? p.per_block : fit;
  const size_t smem = (size_t)p.step * 2 * angle_pitch(p.pairs) * 4;
  auto go = [&](auto tag) {
    auto kern = decltype(tag)::kernel();
    static PerDeviceOnce once;  // per kernel
    if (int rc = ensure_dynamic_smem(kern, kAngleBytes, once)) return rc;
    launch_kernel(kern, dim3((unsigned)grid), dim3(kThreads), smem, stream, p);
    TPF_LAUNCH_OK();
    return TPF_OK;
  };
  if (!back) {
    if (c.norm) return go(Kernel<T, VEC, TL, MODE, true, false>{});
    return go(Kernel<T, VEC, TL, MODE, false, false>{});
  }
  if (!c.norm) return go(Kernel<T, VEC, TL, MODE, false, true>{});
  if (int rc = go(Kernel<T, VEC, TL, MODE, true, true>{})) return rc;
  if (p.terms == nullptr) return TPF_OK;
  return norm_fold(p.terms, (int)grid, p.dim, c.t[0].dweight, c.t[0].weight_type, c.t[1].dweight, c.t[1].weight_type, stream);
}
template <typename T, int VEC, int TL>
int launch(const RotaryCall& c, RotaryParams& p, bool back, cudaStream_t stream) {
  if (!c.half) return launch<T, VEC, TL, kInterleaved>(c, p, back, stream);
  if (VEC == 8 && c.rot % 16 != 0) return launch<T, VEC, TL, kHalfAny>(c, p, back, stream);
  return launch<T, VEC, TL, kHalf>(c, p, back, stream);
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

int run(RotaryCall c, void* workspace, int64_t workspace_bytes, bool back, cudaStream_t stream) {
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
  p.all = (uint32_t)(c.batch * c.tokens);
  p.tokens = (int)c.tokens, p.dim = (int)c.dim, p.rot = (int)c.rot, p.pairs = (int)(c.rot / 2);
  p.div_pairs = FastDiv::make((uint32_t)p.pairs);
  p.turns = c.turns, p.positions = c.positions, p.first = c.first;
  p.magnitude = c.magnitude, p.eps = c.eps, p.inv_dim = 1.f / (float)c.dim;
  bool vec = c.dim % 8 == 0;
  for (int k = 0; k < 2; ++k) {
    const RotaryTensor& s = c.t[k];
    RotaryParams::Tensor& t = p.t[k];
    t.heads = (int)s.heads;
    if (s.heads == 0) {
      if (s.dweight != nullptr)
        TPF_CUDA_OK(cudaMemsetAsync(s.dweight, 0, (size_t)c.dim * row_type_size(s.weight_type), stream));
      c.t[k].dweight = nullptr;
      continue;
    }
    TPF_REQUIRE(c.batch * c.tokens * s.heads < (1ll << 31), TPF_ERR_UNSUPPORTED, "%s: too many heads", who);
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

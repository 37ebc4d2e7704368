// Dropout whose mask is never stored: every element's random bits are a function of a seed and of the element's index, so the
// backward pass makes them again.
//
//   out = residual + (kept ? x * 65536 / (65536 - T) : 0)        T = round(65536 p): an element is dropped where its 16 bits are < T
//
// The bits: Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), key = seed,
// counter = (m >> 3, offset), both 64 bits; element m of the mask has half word m & 7 of the four words, the low half first.
// m is the row-major index in the shape of the mask: the shape of x, with 1 in the place of a shared dimension.  So the bits
// depend neither on strides nor on the launch, and eight elements share one evaluation (a 32-bit word each would double its
// cost; 16 bits resolve p to 2^-16, and the scale uses the probability that is really used).
//
// What bounds it: memory where the mask is shared: it is made once by a thread that then walks along the shared dimension.  Instructions
// where every element has its own: 225 of them for eight elements without a residual (ten rounds are twenty 32 x 32 -> 64 bit
// products, with their keys about 90), and 72 % of all issue slots are taken, with the ALU and the multiplier at 57 and 58 %.
// Measured (B200, bf16, 1 x 384 x 384 x 128, with a residual and without): 17.0 and 10.9 us with a mask shared along the rows (6.7 and
// 6.9 TB/s, the rate of a copy), 23.1 and 21.1 us with bits for every element.  Rows at any address are slower, most of all with a shared
// mask, where a thread has two-byte loads of up to four rows (257 x 257 x 97 with a residual: 9.9 us for every element, 19.7 shared, 5.9 at
// the rate of a copy), and so are short mask rows over a long shared dimension, where a run has a block to itself (200000 x 64:
// 51 us for 11.7; 300001 x 33: 1390 for 9.1).
#include "tpf_dropout.h"

#include "tpf_rows.cuh"

namespace tpf {

namespace {

struct DropoutParams {
  const void *x, *r;
  void* out;
  int64_t xp, xq, xs, rp, rq, rs, op, oq, os;  // element strides of the outer dimensions
  int64_t inner;
  uint32_t P, Q, S;
  int s_in_mask;                // 0: the mask is shared along S
  uint32_t border;              // the threshold times 2^16
  int none;                     // the threshold is 2^16: nothing is kept
  float scale;
  const int64_t* seed_ptr;      // (seed, offset) on the device, or nullptr
  uint64_t seed, offset;
  uint32_t cells;               // vectors of a row
  FastDiv div_cells, div_q, div_inner;
};

struct Philox {
  uint32_t k0, k1, o0, o1;
  __device__ __forceinline__ explicit Philox(const DropoutParams& p) {
    uint64_t seed = p.seed, offset = p.offset;
    if (p.seed_ptr != nullptr) {
      seed = (uint64_t)p.seed_ptr[0];
      offset = (uint64_t)p.seed_ptr[1];
    }
    k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    o0 = (uint32_t)offset, o1 = (uint32_t)(offset >> 32);
  }
  __device__ __forceinline__ void words(uint64_t group, uint32_t (&w)[4]) const {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = o0, c3 = o1, a = k0, b = k1;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t l = (uint64_t)c0 * 0xD2511F53u, r = (uint64_t)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(r >> 32) ^ c1 ^ a;
      c1 = (uint32_t)r;
      c2 = (uint32_t)(l >> 32) ^ c3 ^ b;
      c3 = (uint32_t)l;
      a += 0x9E3779B9u;
      b += 0xBB67AE85u;
    }
    w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
  }
};
// Is element h of a group kept?  `border`: the threshold in the upper half word; 2^16 does not fit there, and `none` says it.
__device__ __forceinline__ bool is_kept(const uint32_t (&w)[4], int h, uint32_t border, bool none) {
  return (h & 1 ? w[h >> 1] : w[h >> 1] << 16) >= border && !none;
}
__device__ __forceinline__ uint32_t kept_bits(const uint32_t (&w)[4], uint32_t border, bool none) {
  uint32_t bits = 0;
#pragma unroll
  for (int h = 0; h < 8; ++h) bits |= is_kept(w, h, border, none) ? 1u << h : 0u;
  return bits;
}

constexpr int kThreads = 256;
// The first index along S of a block's run.  (Runs lie along the grid's y, and along z where there are more of them than y takes.)
template <int RUN>
__device__ __forceinline__ uint32_t run_start() {
  return (blockIdx.z * gridDim.y + blockIdx.y) * RUN;
}
template <typename T, bool RES>
__device__ __forceinline__ void drop_vec(const Piece<T, 8>& x, const Piece<T, 8>& r, const bool (&kept)[8], float scale, T* out) {
  float v[8], w[8];
  x.get(v);
  if (RES) r.get(w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = kept[i] ? v[i] * scale : 0.f;  // (a dropped infinity is a zero)
    v[i] = RES ? y + w[i] : y;
  }
  store_vec<T, 8>(out, v);
}

// Rows that start on vector boundaries and on groups of the mask: a thread per vector of the mask and run of the shared dimension.
// (Without a shared dimension: four vectors a thread, with their keys made once, took as long, 21 us, and with a residual 28 for 23.)
template <typename T, bool RES, int RUN>
__global__ void __launch_bounds__(kThreads) dropout_vec_kernel(const DropoutParams p) {
  griddep_wait();
  const uint32_t cell = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = p.div_cells.div(cell), vec = cell - row * p.cells;
  const uint32_t pi = p.div_q.div(row), qi = row - pi * p.Q;
  const uint32_t s0 = run_start<RUN>();
  if (pi >= p.P || s0 >= p.S) return;
  const int64_t e = (int64_t)vec * 8;
  const T* x = static_cast<const T*>(p.x) + pi * p.xp + qi * p.xq + s0 * p.xs + e;
  const T* r = RES ? static_cast<const T*>(p.r) + pi * p.rp + qi * p.rq + s0 * p.rs + e : nullptr;
  T* out = static_cast<T*>(p.out) + pi * p.op + qi * p.oq + s0 * p.os + e;
  const uint64_t m = ((uint64_t)row * (p.s_in_mask ? p.S : 1u) + (p.s_in_mask ? s0 : 0u)) * (uint64_t)p.inner + (uint64_t)e;
  const Philox gen(p);
  uint32_t words[4];
  if (p.inner - e < 8) {  // the tail of a single row
    gen.words(m >> 3, words);
    const uint32_t bits = kept_bits(words, p.border, p.none);
    for (int i = 0; i < (int)(p.inner - e); ++i) {
      const float y = bits >> i & 1u ? to_f32(x[i]) * p.scale : 0.f;
      out[i] = from_f32<T>(RES ? y + to_f32(r[i]) : y);
    }
    return;
  }
  Piece<T, 8> px[RUN], pr[RUN];
  const int n = RUN == 1 ? 1 : min(RUN, (int)(p.S - s0));
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int k = min(i, n - 1);
    px[i].load(x + k * p.xs);
    if (RES) pr[i].load(r + k * p.rs);
  }
  gen.words(m >> 3, words);  // while the loads are on their way
  bool kept[8];
#pragma unroll
  for (int h = 0; h < 8; ++h) kept[h] = is_kept(words, h, p.border, p.none);
#pragma unroll
  for (int i = 0; i < RUN; ++i)
    if (i < n) drop_vec<T, RES>(px[i], pr[i], kept, p.scale, out + i * p.os);
}

// Rows at any address: a warp takes 32 groups of the mask, whatever rows they belong to; each lane makes the bits of one, and the
// elements, which lie side by side over the lanes, take theirs by a shuffle.
template <typename T, bool RES, int RUN>
__global__ void __launch_bounds__(kThreads) dropout_any_kernel(const DropoutParams p) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t s0 = run_start<RUN>();  // (of a shared dimension; else 0)
  if (s0 >= p.S) return;
  const uint64_t m0 = ((uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * 256;
  const uint64_t row0 = m0 / (uint64_t)p.inner, e0 = m0 - row0 * p.inner;
  const int n = RUN == 1 ? 1 : min(RUN, (int)(p.S - s0));
  T v[RUN][8], w[RUN][8];
  T* out[8];
  uint64_t row_i = row0;
  int64_t e = (int64_t)e0 + lane;
#pragma unroll
  for (int i = 0; i < 8; ++i, e += 32) {
    if (e >= p.inner) {  // (rows of 32 elements and more end once at most)
      const uint32_t rows = p.inner >= 32 ? 1u : p.div_inner.div((uint32_t)e);
      row_i += rows;
      e -= rows * p.inner;
    }
    uint64_t row = row_i;
    int64_t xs = s0 * p.xs, rs = s0 * p.rs, os = s0 * p.os;
    if (p.s_in_mask && p.S > 1) {
      const uint32_t pq = (uint32_t)(row / p.S), s = (uint32_t)(row - (uint64_t)pq * p.S);
      xs = s * p.xs, rs = s * p.rs, os = s * p.os;
      row = pq;
    }
    const bool on = row < (uint64_t)p.P * p.Q;
    const uint32_t pi = on ? p.div_q.div((uint32_t)row) : 0u, qi = on ? (uint32_t)row - pi * p.Q : 0u;
    const T* x = static_cast<const T*>(p.x) + pi * p.xp + qi * p.xq + xs + e;
    const T* r = RES ? static_cast<const T*>(p.r) + pi * p.rp + qi * p.rq + rs + e : nullptr;
    out[i] = on ? static_cast<T*>(p.out) + pi * p.op + qi * p.oq + os + e : nullptr;
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      v[k][i] = on && k < n ? x[k * p.xs] : T(0.f);
      if (RES) w[k][i] = on && k < n ? r[k * p.rs] : T(0.f);
    }
  }
  const Philox gen(p);
  uint32_t words[4];
  gen.words((m0 >> 3) + lane, words);
  const uint32_t bits = kept_bits(words, p.border, p.none);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool kept = __shfl_sync(0xffffffffu, bits, 4 * i + (lane >> 3)) >> (lane & 7) & 1u;
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      const float y = kept ? to_f32(v[k][i]) * p.scale : 0.f;
      if (out[i] != nullptr && k < n) out[i][k * p.os] = from_f32<T>(RES ? y + to_f32(w[k][i]) : y);
    }
  }
}

// `cells`: vectors or, where there are none, groups of 256 elements of the mask.
template <typename T, bool RES, int RUN>
int launch(const DropoutParams& p, bool vec, int64_t cells, cudaStream_t stream) {
  const int64_t per_block = vec ? kThreads : kThreads / 32;
  const uint32_t runs = p.s_in_mask && !vec ? 1 : (p.S + RUN - 1) / RUN, z = (runs + 65534) / 65535;
  const dim3 grid((unsigned)((cells + per_block - 1) / per_block), (runs + z - 1) / z, z);
  if (vec) launch_kernel(dropout_vec_kernel<T, RES, RUN>, grid, dim3(kThreads), 0, stream, p);
  else if constexpr (RUN <= 4) launch_kernel(dropout_any_kernel<T, RES, RUN>, grid, dim3(kThreads), 0, stream, p);
  TPF_LAUNCH_OK();
  return TPF_OK;
}
template <typename T, bool RES>
int launch(const DropoutParams& p, bool vec, int64_t cells, cudaStream_t stream) {
  // Long runs make few masks, and few threads: a run is shortened while there would be fewer blocks than eight an SM (two, where
  // a thread has eight elements of every row).
  const int64_t enough = (vec ? 8ll : 2ll) * sm_count(), per_block = vec ? kThreads : kThreads / 32;
  const int64_t blocks = (cells + per_block - 1) / per_block;
  const int64_t s = p.s_in_mask ? 1 : p.S;
  if (s >= 8 && vec && blocks * (s / 8) >= enough) return launch<T, RES, 8>(p, vec, cells, stream);
  if (s >= 4 && blocks * (s / 4) >= enough) return launch<T, RES, 4>(p, vec, cells, stream);
  if (s >= 2) return launch<T, RES, 2>(p, vec, cells, stream);
  return launch<T, RES, 1>(p, vec, cells, stream);
}
template <typename T>
int launch(const DropoutParams& p, bool vec, int64_t cells, cudaStream_t stream) {
  return p.r != nullptr ? launch<T, true>(p, vec, cells, stream) : launch<T, false>(p, vec, cells, stream);
}

}  // namespace

int dropout(const DropoutCall& c, cudaStream_t stream) {
  TPF_REQUIRE(row_type_ok(c.type), TPF_ERR_INVALID_ARGUMENT, "dropout: unknown element type %d", c.type);
  for (int i = 0; i < 4; ++i)
    TPF_REQUIRE(c.sizes[i] >= 0, TPF_ERR_INVALID_ARGUMENT, "dropout: sizes must not be negative");
  TPF_REQUIRE(c.threshold >= 0 && c.threshold <= 65536, TPF_ERR_INVALID_ARGUMENT, "dropout: the threshold must be in 0 .. 65536");
  const int64_t P = c.sizes[0], Q = c.sizes[1], S = c.sizes[2], I = c.sizes[3];
  if (P == 0 || Q == 0 || S == 0 || I == 0) return TPF_OK;
  TPF_REQUIRE(c.x && c.out, TPF_ERR_INVALID_ARGUMENT, "dropout: null pointer");
  constexpr int64_t kMost = 1ll << 31;
  TPF_REQUIRE(P < kMost && Q < kMost && S < kMost && P * Q < kMost && P * Q * S < (1ll << 62) / I, TPF_ERR_UNSUPPORTED,
              "dropout: too many rows");
  DropoutParams p = {};
  p.x = c.x, p.r = c.residual, p.out = c.out;
  p.xp = c.x_strides[0], p.xq = c.x_strides[1], p.xs = c.x_strides[2];
  if (c.residual != nullptr) p.rp = c.residual_strides[0], p.rq = c.residual_strides[1], p.rs = c.residual_strides[2];
  p.os = c.out_strides[2], p.oq = c.out_strides[1], p.op = c.out_strides[0];
  p.inner = I;
  p.P = (uint32_t)P, p.Q = (uint32_t)Q, p.S = (uint32_t)S;
  p.s_in_mask = c.shared ? 0 : 1;
  p.none = c.threshold == 65536;
  p.border = p.none ? 0xffffffffu : (uint32_t)c.threshold << 16;
  p.scale = c.threshold < 65536 ? (float)(65536.0 / (65536 - c.threshold)) : 0.f;
  p.seed_ptr = c.seed_ptr;
  p.seed = (uint64_t)c.seed, p.offset = (uint64_t)c.offset;
  auto whole = [&](int64_t n, int64_t stride) { return n == 1 || stride % 8 == 0; };
  const bool aligned = vec_ok(c.x, c.type) && vec_ok(c.out, c.type) && (c.residual == nullptr || vec_ok(c.residual, c.type));
  bool vec = aligned && (I % 8 == 0 || P * Q * S == 1);
  for (int d = 0; d < 3; ++d)
    vec = vec && whole(c.sizes[d], c.x_strides[d]) && whole(c.sizes[d], c.out_strides[d]) &&
          (c.residual == nullptr || whole(c.sizes[d], c.residual_strides[d]));
  TPF_REQUIRE(!(vec && p.s_in_mask) || S <= 65535, TPF_ERR_UNSUPPORTED, "dropout: the third dimension is too long without a shared mask");
  int64_t cells = P * Q * ((I + 7) / 8);
  vec = vec && cells < kMost - kThreads;  // (more of them have indices beyond 32 bits, which the kernel of any rows has)
  if (vec) {
    p.cells = (uint32_t)((I + 7) / 8);
    p.div_cells = FastDiv::make(p.cells);
  } else {
    cells = (P * Q * (p.s_in_mask ? S : 1) * I + 255) / 256;
    TPF_REQUIRE(cells < (1ll << 36) / 256, TPF_ERR_UNSUPPORTED, "dropout: too many elements");  // (two such tensors fit no device)
    p.div_inner = FastDiv::make((uint32_t)(I < 32 ? I : 32));
  }
  p.div_q = FastDiv::make((uint32_t)Q);
  if (c.type == kRowF32) return launch<float>(p, vec, cells, stream);
  if (c.type == kRowBF16) return launch<bf16>(p, vec, cells, stream);
  return launch<__half>(p, vec, cells, stream);
}

}  // namespace tpf

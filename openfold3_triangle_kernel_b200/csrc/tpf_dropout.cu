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
// What bounds it: memory.  Ten rounds are twenty 32 x 32 -> 64 bit products, about 90 instructions for eight elements; a
// shared mask is made once by a thread that then walks along the shared dimension.
// Measured (B200, bf16, mask shared along dimension -3 of 1 x 384 x 384 x 128, forward with a residual and backward): see kRun.
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
  uint32_t threshold;
  float scale;
  const int64_t* seed_ptr;      // (seed, offset) on the device, or nullptr
  uint64_t seed, offset;
  uint32_t cells;               // vectors (or chunks of 32 groups) of a row
  FastDiv div_cells, div_q;
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
  // Bit h: element h of a group of eight is kept.
  __device__ __forceinline__ uint32_t kept(uint64_t group, uint32_t threshold) const {
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
    const uint32_t w[4] = {c0, c1, c2, c3};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bits |= ((w[i] & 0xffffu) >= threshold ? 1u : 0u) << (2 * i);
      bits |= ((w[i] >> 16) >= threshold ? 1u : 0u) << (2 * i + 1);
    }
    return bits;
  }
};

constexpr int kThreads = 256;
// Elements of the shared dimension that a thread walks with one mask.
constexpr int kRun = 8;

template <typename T, bool RES>
__device__ __forceinline__ void drop_vec(const Piece<T, 8>& x, const Piece<T, 8>& r, uint32_t bits, float scale, T* out) {
  float v[8], w[8];
  x.get(v);
  if (RES) r.get(w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = bits >> i & 1u ? v[i] * scale : 0.f;  // (a dropped infinity is a zero)
    v[i] = RES ? y + w[i] : y;
  }
  store_vec<T, 8>(out, v);
}

// Rows that start on vector boundaries and on groups of the mask: a thread per vector of the mask and run of the shared dimension.
template <typename T, bool RES, int RUN>
__global__ void __launch_bounds__(kThreads) dropout_vec_kernel(const DropoutParams p) {
  griddep_wait();
  const uint32_t cell = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t row = p.div_cells.div(cell), vec = cell - row * p.cells;
  const uint32_t pi = p.div_q.div(row), qi = row - pi * p.Q;
  if (pi >= p.P) return;
  const uint32_t s0 = blockIdx.y * RUN;
  const int64_t e = (int64_t)vec * 8;
  const T* x = static_cast<const T*>(p.x) + pi * p.xp + qi * p.xq + s0 * p.xs + e;
  const T* r = RES ? static_cast<const T*>(p.r) + pi * p.rp + qi * p.rq + s0 * p.rs + e : nullptr;
  T* out = static_cast<T*>(p.out) + pi * p.op + qi * p.oq + s0 * p.os + e;
  const Philox gen(p);
  const uint64_t m = ((uint64_t)row * (p.s_in_mask ? p.S : 1u) + (p.s_in_mask ? s0 : 0u)) * (uint64_t)p.inner + (uint64_t)e;
  if (p.inner - e < 8) {  // the tail of a single row
    const uint32_t bits = gen.kept(m >> 3, p.threshold);
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
  const uint32_t bits = gen.kept(m >> 3, p.threshold);  // while the loads are on their way
#pragma unroll
  for (int i = 0; i < RUN; ++i)
    if (i < n) drop_vec<T, RES>(px[i], pr[i], bits, p.scale, out + i * p.os);
}

// Rows at any address: a warp takes 32 groups of the mask, each lane makes the bits of one, and the elements, which lie side by side
// over the lanes, take theirs by a shuffle.
template <typename T, bool RES, int RUN>
__global__ void __launch_bounds__(kThreads) dropout_any_kernel(const DropoutParams p) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t cell = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const uint32_t row = p.div_cells.div(cell), chunk = cell - row * p.cells;
  const uint32_t pi = p.div_q.div(row), qi = row - pi * p.Q;
  if (pi >= p.P) return;
  const uint32_t s0 = blockIdx.y * RUN;
  const T* x = static_cast<const T*>(p.x) + pi * p.xp + qi * p.xq + s0 * p.xs;
  const T* r = RES ? static_cast<const T*>(p.r) + pi * p.rp + qi * p.rq + s0 * p.rs : nullptr;
  T* out = static_cast<T*>(p.out) + pi * p.op + qi * p.oq + s0 * p.os;
  const Philox gen(p);
  const uint64_t m = ((uint64_t)row * (p.s_in_mask ? p.S : 1u) + (p.s_in_mask ? s0 : 0u)) * (uint64_t)p.inner;
  const uint64_t first = (m >> 3) + 32ull * chunk;  // group of lane 0
  const int64_t at = (int64_t)(first * 8 - m);      // element of that group's first bit; negative at the start of a row
  const uint32_t bits = gen.kept(first + lane, p.threshold);
  const int n = RUN == 1 ? 1 : min(RUN, (int)(p.S - s0));
  for (int k = 0; k < n; ++k, x += p.xs, r += RES ? p.rs : 0, out += p.os) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t e = at + 32 * i + lane;
      const bool on = e >= 0 && e < p.inner;
      const float v = on ? to_f32(x[e]) : 0.f, w = RES && on ? to_f32(r[e]) : 0.f;
      const uint32_t b = __shfl_sync(0xffffffffu, bits, 4 * i + (lane >> 3)) >> (lane & 7);
      const float y = b & 1u ? v * p.scale : 0.f;
      if (on) out[e] = from_f32<T>(RES ? y + w : y);
    }
  }
}

template <typename T, bool RES, int RUN>
int launch(const DropoutParams& p, bool vec, uint32_t blocks, cudaStream_t stream) {
  const dim3 grid(blocks, (p.S + RUN - 1) / RUN);
  TPF_REQUIRE(grid.y <= 65535, TPF_ERR_UNSUPPORTED, "dropout: the shared dimension is too long");
  if (vec) launch_kernel(dropout_vec_kernel<T, RES, RUN>, grid, dim3(kThreads), 0, stream, p);
  else launch_kernel(dropout_any_kernel<T, RES, RUN>, grid, dim3(kThreads), 0, stream, p);
  TPF_LAUNCH_OK();
  return TPF_OK;
}
template <typename T>
int launch(const DropoutParams& p, bool vec, uint32_t blocks, bool run, cudaStream_t stream) {
  if (p.r != nullptr) return run ? launch<T, true, kRun>(p, vec, blocks, stream) : launch<T, true, 1>(p, vec, blocks, stream);
  return run ? launch<T, false, kRun>(p, vec, blocks, stream) : launch<T, false, 1>(p, vec, blocks, stream);
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
  p.threshold = (uint32_t)c.threshold;
  p.scale = c.threshold < 65536 ? (float)(65536.0 / (65536 - c.threshold)) : 0.f;
  p.seed_ptr = c.seed_ptr;
  p.seed = (uint64_t)c.seed, p.offset = (uint64_t)c.offset;
  auto whole = [&](int64_t n, int64_t stride) { return n == 1 || stride % 8 == 0; };
  const bool aligned = vec_ok(c.x, c.type) && vec_ok(c.out, c.type) && (c.residual == nullptr || vec_ok(c.residual, c.type));
  bool vec = aligned && (I % 8 == 0 || P * Q * S == 1);
  for (int d = 0; d < 3; ++d)
    vec = vec && whole(c.sizes[d], c.x_strides[d]) && whole(c.sizes[d], c.out_strides[d]) &&
          (c.residual == nullptr || whole(c.sizes[d], c.residual_strides[d]));
  const int64_t cells = vec ? (I + 7) / 8 : (I / 8 + 2 + 31) / 32;  // (a row touches at most I / 8 + 2 groups)
  const int64_t total = P * Q * cells, per_block = vec ? kThreads : kThreads / 32;
  TPF_REQUIRE(cells < kMost && total < kMost - kThreads, TPF_ERR_UNSUPPORTED, "dropout: too many elements");
  p.cells = (uint32_t)cells;
  p.div_cells = FastDiv::make((uint32_t)cells);
  p.div_q = FastDiv::make((uint32_t)Q);
  const uint32_t blocks = (uint32_t)((total + per_block - 1) / per_block);
  const bool run = c.shared && S > 1;
  if (c.type == kRowF32) return launch<float>(p, vec, blocks, run, stream);
  if (c.type == kRowBF16) return launch<bf16>(p, vec, blocks, run, stream);
  return launch<__half>(p, vec, blocks, run, stream);
}

}  // namespace tpf

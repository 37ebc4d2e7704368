// Row-wise pieces shared by the layer norm, the 8-bit checkpoint and the normalised projection: element types, how the
// threads of a team share a row, sums over a team, and the 8-bit format.
//
// 8-bit format.  Groups of 128 consecutive elements of a row (the last one ragged) share a scale.  With a = max |x| of
// the group, f = fl32(127 / a) and s = fl32(a / 127): code = rint(x f), value = code s.  The product x f is exact in the
// FMA that rounds it (ties to even), so the codes do not depend on the order of any operation.  |x f| <= 127 (1 + 2^-24)
// rounds to at most 127.  s is the largest value with a finite 127 s at most (FLT_MAX / 127 rounds up, so that FLT_MAX, a common
// fill of masks, would come back as infinity; no other a is touched).  a < 2^-119 (where f would overflow): the group is kept as zeros.  A group that holds an
// infinity or a NaN has the scale NaN and codes 0, and comes back as NaN.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "tpf_host.cuh"
#include "tpf_ptx.cuh"

namespace tpf {

typedef __nv_bfloat16 bf16;

constexpr int kGroup = 128;             // elements of a row that share one scale
constexpr float kTiny = 0x1p-119f;      // smallest amax that is kept
constexpr float kMaxScale = 0x1.020406p121f;  // 127 times this is finite, of the next float it is not
constexpr int64_t kMaxNormCols = 8192;  // widest row of the layer norm: 256 threads with 32 elements each

enum RowType : int { kRowF32 = 0, kRowBF16 = 1, kRowF16 = 2 };
inline bool row_type_ok(int type) { return type >= kRowF32 && type <= kRowF16; }
inline int row_type_size(int type) { return type == kRowF32 ? 4 : 2; }
inline int64_t row_groups(int64_t cols) { return (cols + kGroup - 1) / kGroup; }

// ---- element access ------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (std::is_same<T, bf16>::value) return __bfloat162float(v);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, bf16>::value) return __float2bfloat16_rn(v);
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, bf16>::value) {
    return pack_bf16x2(lo, hi);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (std::is_same<T, bf16>::value) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// VEC consecutive elements as they lie in memory, VEC = 8 or 1.  Eight are one 16-byte access, or one of 32 bytes in fp32
// (sm_100 has 256-bit loads and stores).  Loads and conversions are apart so that a kernel issues all its loads, without a
// branch around any, before it waits for the first: with `if (row < rows) x = convert(load)` the rows of a thread were
// loaded one after the other, and the backward of 768 * 768 rows of 128 channels took 155 us.
template <typename T, int VEC>
struct Piece {
  using Raw = std::conditional_t<VEC == 1, T, std::conditional_t<sizeof(T) == 4, float, uint32_t>>;
  static constexpr int N = VEC == 1 ? 1 : sizeof(T) == 4 ? 8 : 4;
  Raw v[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      v[0] = *p;
    } else if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                   : "l"(p)
                   : "memory");
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      v[0] = u.x;
      v[1] = u.y;
      v[2] = u.z;
      v[3] = u.w;
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Raw(0.f);
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (VEC == 1) {
      x[0] = to_f32(v[0]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<T, bf16>::value) {
          x[2 * i] = __uint_as_float(v[i] << 16);
          x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      }
    }
  }
  // Largest magnitude, NaN if one is; in 16-bit types two elements an instruction.
  __device__ __forceinline__ float amax() const {
    if constexpr (VEC == 1) {
      return fabsf(to_f32(v[0]));
    } else if constexpr (sizeof(T) == 4) {
      return max3_nan(max3_nan(fabsf(v[0]), fabsf(v[1]), fabsf(v[2])), max3_nan(fabsf(v[3]), fabsf(v[4]), fabsf(v[5])),
                      max_nan(fabsf(v[6]), fabsf(v[7])));
    } else {
      using T2 = std::conditional_t<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>;
      const T2* w = reinterpret_cast<const T2*>(v);
      const T2 m = __hmax2_nan(__hmax2_nan(__habs2(w[0]), __habs2(w[1])), __hmax2_nan(__habs2(w[2]), __habs2(w[3])));
      return max_nan(to_f32(m.x), to_f32(m.y));
    }
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(x[0]);
  } else if constexpr (sizeof(T) == 4) {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                 "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}
inline bool vec_ok(const void* p, int type) {  // may the address be accessed eight elements at a time?
  return (reinterpret_cast<uintptr_t>(p) & (type == kRowF32 ? 31 : 15)) == 0;
}

// Vectors of parameters in the caller's type; nullptr means `absent` everywhere.
struct ParamVec {
  const void* p;
  int type;
};
// N values, `stride` apart, from element c on; those at `cols` and behind are 0.
template <int N, int STRIDE>
__device__ __forceinline__ void param_load(const ParamVec& v, int c, int cols, float absent, float* x) {
  auto all = [&](auto* p) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = c + e * STRIDE < cols ? to_f32(p[c + e * STRIDE]) : 0.f;
  };
  if (v.p == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = c + e * STRIDE < cols ? absent : 0.f;
  } else if (v.type == kRowF32) {
    all(static_cast<const float*>(v.p));
  } else if (v.type == kRowBF16) {
    all(static_cast<const bf16*>(v.p));
  } else {
    all(static_cast<const __half*>(v.p));
  }
}
struct ParamOut {
  void* p;
  int type;
};
__device__ __forceinline__ void param_put(const ParamOut& v, int64_t i, float x) {
  if (v.type == kRowF32) static_cast<float*>(v.p)[i] = x;
  else if (v.type == kRowBF16) static_cast<bf16*>(v.p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(v.p)[i] = __float2half_rn(x);
}

// Four in a row, i a multiple of 4, p on a 16-byte boundary.
__device__ __forceinline__ void param_put4(const ParamOut& v, int64_t i, const float4& x) {
  if (v.type == kRowF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(v.p) + i) = x;
  } else {
    union {
      bf16 b[4];
      __half h[4];
      uint2 u;
    } o;
    if (v.type == kRowBF16) {
      o.b[0] = __float2bfloat16_rn(x.x), o.b[1] = __float2bfloat16_rn(x.y);
      o.b[2] = __float2bfloat16_rn(x.z), o.b[3] = __float2bfloat16_rn(x.w);
    } else {
      o.h[0] = __float2half_rn(x.x), o.h[1] = __float2half_rn(x.y);
      o.h[2] = __float2half_rn(x.z), o.h[3] = __float2half_rn(x.w);
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(v.p) + i) = o.u;
  }
}

// ---- 8-bit format --------------------------------------------------------------------------------
struct GroupScale {
  float up, down;  // code = rint(x up), value = code down; up is NaN where down is
};
__device__ __forceinline__ GroupScale group_scale(float amax) {
  const float nan = __int_as_float(0x7fc00000);
  if (!(amax <= 3.402823466e38f)) return {nan, nan};  // (NaN compares false)
  if (amax < kTiny) return {0.f, 0.f};
  return {__fdiv_rn(127.f, amax), fminf(__fdiv_rn(amax, 127.f), kMaxScale)};
}
// The factors of N groups (1, 2 or 4) that LANES lanes hold together, each lane with every amax: the quotients cost more than
// all else, so each lane computes those of one group, and they are handed round.  Returns the `down` of group
// (lane % N), the lane's own.
template <int N, int LANES>
__device__ __forceinline__ float group_scales(const float (&amax)[N], float (&up)[N]) {
  static_assert(N <= LANES && (N & (N - 1)) == 0, "");
  const int lane = threadIdx.x & 31, mine = lane & (N - 1);
  float a = amax[0];
#pragma unroll
  for (int n = 1; n < N; ++n) a = mine == n ? amax[n] : a;
  const GroupScale s = group_scale(a);
  if constexpr (N == 1) {
    up[0] = s.up;
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n) up[n] = __shfl_sync(0xffffffffu, s.up, (lane & ~(N - 1)) + n);
  }
  return s.down;
}
// The code in the low byte.  1.5 * 2^23 + n has n in its low bits, two's complement; the FMA rounds the exact product.
__device__ __forceinline__ uint32_t code_bits(float x, float up) { return __float_as_uint(__fmaf_rn(x, up, 12582912.f)); }
__device__ __forceinline__ int8_t code_of(float x, float up) { return up == up ? (int8_t)(code_bits(x, up) & 0xff) : (int8_t)0; }
// Four codes from two pairs.
__device__ __forceinline__ uint32_t pack_codes(uint64_t a, uint64_t b, uint64_t up2, bool good) {
  const uint64_t magic = f2_pack(12582912.f, 12582912.f);
  float x0, x1, x2, x3;
  f2_unpack(f2_fma(a, up2, magic), x0, x1);
  f2_unpack(f2_fma(b, up2, magic), x2, x3);
  const uint32_t lo = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(x2), __float_as_uint(x3), 0x0040);
  return good ? __byte_perm(lo, hi, 0x5410) : 0u;
}
// Four codes -> whole numbers, in two pairs.  With the sign bit flipped a code is 0 .. 255, and 2^23 + that is put together
// from bytes: conversions from integers run at a quarter of the rate.
__device__ __forceinline__ void unpack_codes(uint32_t w, uint64_t* x) {
  w ^= 0x80808080u;
  uint32_t f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __byte_perm(w, 0x4b000000u, 0x7440 + i);
  const uint64_t bias = f2_pack(-8388736.f, -8388736.f);
  x[0] = f2_add(f2_pack_bits(f[0], f[1]), bias);
  x[1] = f2_add(f2_pack_bits(f[2], f[3]), bias);
}
__device__ __forceinline__ uint64_t f2_dup(float x) { return f2_pack(x, x); }
__device__ __forceinline__ float f2_sum(uint64_t v) {
  float lo, hi;
  f2_unpack(v, lo, hi);
  return lo + hi;
}

// ---- a team of threads on a row ------------------------------------------------------------------
// A thread owns ITEMS pieces of VEC consecutive elements.  The pieces of one item lie side by side over the lanes of a
// warp (coalesced accesses), the items of a warp follow one another, the warps of a team as well.  So a group of 128
// elements is always inside one warp: 16 lanes of an item (VEC = 8), or 128 / TS items of all lanes (VEC = 1).
// TS = 4 .. 32: teams of TS lanes, 256 threads a block.  TS = 0: the block is the team, up to MAXB threads.
template <int VEC_, int TS_, int ITEMS_, int MAXB_ = 256>
struct Team {
  static constexpr int VEC = VEC_, TS = TS_, ITEMS = ITEMS_, E = VEC * ITEMS, MAXB = MAXB_;
  static constexpr bool BLOCK = TS == 0;
  static constexpr int TEAMS = BLOCK ? 1 : MAXB / TS;
  static constexpr int COLS = BLOCK ? MAXB * E : TS * E;  // widest row
  static_assert(VEC == 8 || (VEC == 1 && ITEMS % 4 == 0 && (BLOCK || COLS <= 128 || COLS % 128 == 0)), "groups stay inside a warp");
  static int threads(int cols) {  // of a block
    return BLOCK ? ((cols + E - 1) / E + 31) / 32 * 32 : MAXB;
  }

  int t, index;  // thread of the team, team of the block
  __device__ __forceinline__ Team() {
    t = BLOCK ? threadIdx.x : threadIdx.x % (BLOCK ? 1 : TS);
    index = BLOCK ? 0 : threadIdx.x / (BLOCK ? 1 : TS);
  }
  __device__ __forceinline__ int column(int item) const {
    return BLOCK ? ((t >> 5) * ITEMS * 32 + item * 32 + (t & 31)) * VEC : (item * TS + t) * VEC;
  }
};

template <int N>
__device__ __forceinline__ void warp_sum(float (&v)[N], int lanes = 32) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    if (off < lanes)
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], off);
}
// One value per warp of a block and n, written by a lane of each warp, is read by lane n W + warp of every warp: the W warps'
// values are then added by shuffles, log2 W instructions in the place of W loads for each n.
template <class Tm, int N>
struct CrossWarp {
  static constexpr int W = Tm::MAXB / 32;
  static_assert(N * W <= 32 && (W & (W - 1)) == 0, "");
  static __device__ __forceinline__ float sum(float v) {  // over the W lanes of an n
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
  }
  static __device__ __forceinline__ bool exists() { return ((threadIdx.x & 31) & (W - 1)) < (blockDim.x >> 5); }
};
// Sums of N values at once over a team; every thread gets the same bits.  `red`: 2 x 32 floats for a team of several
// warps, used in turns so that one barrier a sum is enough.
template <class Tm, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* red, int& turn) {
  warp_sum(v, Tm::BLOCK ? 32 : Tm::TS);
  if constexpr (Tm::BLOCK) {
    using X = CrossWarp<Tm, N>;
    float* r = red + turn * 32;
    turn ^= 1;
    const int lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) r[n * X::W + (threadIdx.x >> 5)] = v[n];
    __syncthreads();
    const float s = X::sum(X::exists() && lane < N * X::W ? r[lane] : 0.f);
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, s, n * X::W);
  }
}

// Groups of 128 a thread takes part in: VEC = 8: one a piece (a team narrower than 16 lanes: one of all pieces), VEC = 1: one per
// 128 columns; LANES lanes share one.
template <class Tm>
struct Groups {
  static constexpr int LANES = Tm::VEC == 1 ? (Tm::BLOCK ? 32 : Tm::TS) : Tm::BLOCK || Tm::TS >= 16 ? 16 : Tm::TS;
  static constexpr int N = Tm::VEC == 1 ? (Tm::BLOCK ? Tm::ITEMS / 4 : (Tm::COLS + 127) / 128) : (Tm::ITEMS * LANES + 15) / 16;
};

// A thread's part of a row, as it lies in memory and as pairs of floats (sm_100 works on two at once).  `at`: the columns
// of the items, of one that does not exist column 0 (it is loaded and masked).
template <typename T, class Tm>
struct Frag {
  static constexpr int VEC = Tm::VEC, ITEMS = Tm::ITEMS, E = Tm::E;
  Piece<T, VEC> p[ITEMS];
  __device__ __forceinline__ void load(const T* row, const int (&at)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) p[i].load(row + at[i]);
  }
  __device__ __forceinline__ void mask(const bool (&on)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (!on[i]) p[i].zero();
  }
  __device__ __forceinline__ void get(uint64_t (&x)[E / 2]) const {
    float f[E];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) p[i].get(f + i * VEC);
#pragma unroll
    for (int k = 0; k < E / 2; ++k) x[k] = f2_pack(f[2 * k], f[2 * k + 1]);
  }
  __device__ __forceinline__ void amax(float* m) const {
    constexpr int NG = Groups<Tm>::N, PER = ITEMS / NG;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      m[g] = p[g * PER].amax();
#pragma unroll
      for (int i = 1; i < PER; ++i) m[g] = max_nan(m[g], p[g * PER + i].amax());
#pragma unroll
      for (int off = Groups<Tm>::LANES / 2; off > 0; off >>= 1) m[g] = max_nan(m[g], __shfl_xor_sync(0xffffffffu, m[g], off));
    }
  }
};
template <class Tm>
__device__ __forceinline__ void mask_pairs(uint64_t (&x)[Tm::E / 2], const bool (&on)[Tm::ITEMS]) {
#pragma unroll
  for (int i = 0; i < Tm::ITEMS; ++i) {
    if (on[i]) continue;
    if constexpr (Tm::VEC == 8) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[4 * i + k] = 0;
    } else {
      float lo, hi;
      f2_unpack(x[i / 2], lo, hi);
      x[i / 2] = i % 2 ? f2_pack(lo, 0.f) : f2_pack(0.f, hi);
    }
  }
}
template <typename T, class Tm>
__device__ __forceinline__ void store_row(T* row, const uint64_t (&x)[Tm::E / 2], const int (&at)[Tm::ITEMS],
                                          const bool (&on)[Tm::ITEMS]) {
  float f[Tm::E];
#pragma unroll
  for (int k = 0; k < Tm::E / 2; ++k) f2_unpack(x[k], f[2 * k], f[2 * k + 1]);
#pragma unroll
  for (int i = 0; i < Tm::ITEMS; ++i)
    if (on[i]) store_vec<T, Tm::VEC>(row + at[i], f + i * Tm::VEC);
}
template <class Tm>
struct CodeFrag {
  static constexpr int VEC = Tm::VEC, ITEMS = Tm::ITEMS, E = Tm::E;
  using Raw = std::conditional_t<VEC == 1, int8_t, uint2>;
  Raw p[ITEMS];
  __device__ __forceinline__ void load(const int8_t* row, const int (&at)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) p[i] = *reinterpret_cast<const Raw*>(row + at[i]);
  }
  __device__ __forceinline__ void get(uint64_t (&x)[E / 2]) const {
    if constexpr (VEC == 1) {
#pragma unroll
      for (int k = 0; k < E / 2; ++k) x[k] = f2_pack((float)p[2 * k], (float)p[2 * k + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        unpack_codes(p[i].x, x + 4 * i);
        unpack_codes(p[i].y, x + 4 * i + 2);
      }
    }
  }
};
// Brings what lies in whole 16-byte units of `bytes` bytes at p into L2.
__device__ __forceinline__ void row_prefetch(const void* p, int bytes) {
  const uint64_t first = (reinterpret_cast<uint64_t>(p) + 15) & ~15ull, last = (reinterpret_cast<uint64_t>(p) + bytes) & ~15ull;
  if (last > first) bulk_prefetch(reinterpret_cast<const void*>(first), (uint32_t)(last - first));
}

// Codes of a row; up: the factor of each group.
template <class Tm>
__device__ __forceinline__ void store_codes(int8_t* row, const uint64_t (&x)[Tm::E / 2], const float* up,
                                            const int (&at)[Tm::ITEMS], const bool (&on)[Tm::ITEMS]) {
  if constexpr (Tm::VEC == 1) {
#pragma unroll
    for (int i = 0; i < Tm::ITEMS; ++i) {
      float lo, hi;
      f2_unpack(x[i / 2], lo, hi);
      if (on[i]) row[at[i]] = code_of(i % 2 ? hi : lo, up[i * Groups<Tm>::N / Tm::ITEMS]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < Tm::ITEMS; ++i) {
      const float f = up[i * Groups<Tm>::N / Tm::ITEMS];
      const uint64_t u = f2_dup(f);
      const bool good = f == f;
      if (on[i])
        *reinterpret_cast<uint2*>(row + at[i]) =
            make_uint2(pack_codes(x[4 * i], x[4 * i + 1], u, good), pack_codes(x[4 * i + 2], x[4 * i + 3], u, good));
    }
  }
}

}  // namespace tpf

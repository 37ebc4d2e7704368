// Row-wise pieces shared by the layer norm, the 8-bit checkpoint and the normalised projection: element types, how the
// threads of a team share a row, sums over a team, and the 8-bit format.
//
// 8-bit format.  Groups of 128 consecutive elements of a row (the last one ragged) share a scale.  With a = max |x| of
// the group, f = fl32(127 / a) and s = fl32(a / 127): code = rint(x f), value = code s.  The product x f is exact in the
// FMA that rounds it (ties to even), so the codes do not depend on the order of any operation.  |x f| <= 127 (1 + 2^-24)
// rounds to at most 127.  a < 2^-119 (where f would overflow): the group is kept as zeros.  A group that holds an
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

// VEC consecutive elements, VEC = 8 or 1.  Eight are one 16-byte access, or one of 32 bytes in fp32 (sm_100 has 256-bit
// loads and stores).
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  if constexpr (VEC == 1) {
    x[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(p)
                 : "memory");
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, bf16>::value) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
}
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
__device__ __forceinline__ float param_at(const ParamVec& v, int64_t i, float absent) {
  if (v.p == nullptr) return absent;
  if (v.type == kRowF32) return static_cast<const float*>(v.p)[i];
  if (v.type == kRowBF16) return __bfloat162float(static_cast<const bf16*>(v.p)[i]);
  return __half2float(static_cast<const __half*>(v.p)[i]);
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

// ---- 8-bit format --------------------------------------------------------------------------------
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
struct GroupScale {
  float up, down;  // code = rint(x up), value = code down
};
__device__ __forceinline__ GroupScale group_scale(float amax) {
  if (!(amax <= 3.402823466e38f)) return {0.f, __int_as_float(0x7fc00000)};  // (NaN compares false)
  if (amax < kTiny) return {0.f, 0.f};
  return {__fdiv_rn(127.f, amax), __fdiv_rn(amax, 127.f)};
}
// The code in the low byte.  1.5 * 2^23 + n has n in its low bits, two's complement; the FMA rounds the exact product.
__device__ __forceinline__ uint32_t code_bits(float x, float up) { return __float_as_uint(__fmaf_rn(x, up, 12582912.f)); }
__device__ __forceinline__ int8_t code_of(float x, const GroupScale& s) {
  return s.down == s.down ? (int8_t)(code_bits(x, s.up) & 0xff) : (int8_t)0;
}
__device__ __forceinline__ uint32_t pack_codes(const float* x, const GroupScale& s) {
  const uint32_t lo = __byte_perm(code_bits(x[0], s.up), code_bits(x[1], s.up), 0x0040);
  const uint32_t hi = __byte_perm(code_bits(x[2], s.up), code_bits(x[3], s.up), 0x0040);
  return s.down == s.down ? __byte_perm(lo, hi, 0x5410) : 0u;
}
// Four codes -> their values.  With the sign bit flipped a code is 0 .. 255, and 2^23 + that is put together from bytes:
// conversions from integers run at a quarter of the rate.
__device__ __forceinline__ void unpack_codes(uint32_t w, float down, float* x) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.f) * down;
}
template <int VEC>
__device__ __forceinline__ void load_codes(const int8_t* p, float down, float* x) {
  if constexpr (VEC == 1) {
    x[0] = (float)*p * down;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    unpack_codes(u.x, down, x);
    unpack_codes(u.y, down, x + 4);
  }
}
template <int VEC>
__device__ __forceinline__ void store_codes(int8_t* p, const float* x, const GroupScale& s) {
  if constexpr (VEC == 1) *p = code_of(x[0], s);
  else *reinterpret_cast<uint2*>(p) = make_uint2(pack_codes(x, s), pack_codes(x + 4, s));
}

// ---- a team of TS threads on a row ---------------------------------------------------------------
// A thread owns ITEMS pieces of VEC consecutive elements.  The pieces of one item lie side by side over the lanes of a
// warp (coalesced accesses), the items of a warp follow one another, the warps of a team as well.  So a group of 128
// elements is always inside one warp: 16 lanes of an item (VEC = 8), or 4 items (VEC = 1).
// TS <= 32: several teams in a warp, 256 threads a block.  TS > 32: one team is the block.
template <int VEC_, int TS_, int ITEMS_>
struct Team {
  static constexpr int VEC = VEC_, TS = TS_, ITEMS = ITEMS_, E = VEC * ITEMS;
  static constexpr int BLOCK = TS <= 32 ? 256 : TS, TEAMS = BLOCK / TS, WARPS = BLOCK / 32;
  static constexpr int COLS = TS * E;  // widest row
  static_assert(VEC == 8 || (VEC == 1 && TS >= 32 && ITEMS % 4 == 0), "groups stay inside a warp");
  static_assert(TS >= 32 || ITEMS == 1, "a team of a part of a warp has one item");

  int t, index;  // thread of the team, team of the block
  __device__ __forceinline__ Team() {
    t = TS <= 32 ? threadIdx.x % TS : threadIdx.x;
    index = TS <= 32 ? threadIdx.x / TS : 0;
  }
  __device__ __forceinline__ int column(int item) const {
    return TS <= 32 ? (item * TS + t) * VEC : ((t >> 5) * ITEMS * 32 + item * 32 + (t & 31)) * VEC;
  }
};

// Sums of N values at once over a team; every thread gets the same bits.  `red`: 2 x WARPS x N floats for teams of several
// warps, used in turns so that one barrier a sum is enough.
template <class Tm, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float* red, int& turn) {
  constexpr int W = Tm::TS <= 32 ? Tm::TS : 32;
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], off);
  if constexpr (Tm::TS > 32) {
    float* r = red + turn * Tm::WARPS * N;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) r[(threadIdx.x >> 5) * N + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = r[n];
#pragma unroll
      for (int w = 1; w < Tm::WARPS; ++w) v[n] += r[w * N + n];
    }
  }
}

// Largest |x| of each group a thread takes part in: VEC = 8: one a piece; VEC = 1: one per four items.
template <class Tm>
__device__ __forceinline__ void group_amax(const float* x, float (&amax)[Tm::VEC == 8 ? Tm::ITEMS : (Tm::ITEMS + 3) / 4]) {
  constexpr int NG = Tm::VEC == 8 ? Tm::ITEMS : (Tm::ITEMS + 3) / 4;
  constexpr int PER = Tm::E / NG;
  constexpr int LANES = Tm::VEC == 1 ? 32 : Tm::TS < 16 ? Tm::TS : 16;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) a = max_nan(a, fabsf(x[g * PER + e]));
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, off));
    amax[g] = a;
  }
}

}  // namespace tpf

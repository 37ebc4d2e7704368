// Activations put away in 8 bits and taken out again (the format is described in tpf_rows.cuh).
//
// Both directions are bound by memory: three bytes an element in bf16.  The unit of work is a group of 128 elements.  Where
// eight elements can be accessed at once, LANES = 4, 8 or 16 lanes hold a group (of 32, 64 or more columns); else 8 to 32 lanes
// do, a lane with every LANES-th element, or, to unpack, eight elements of the flat arrays at a time.
#include "tpf_rows.cuh"
#include "tpf_rows.h"

namespace tpf {

namespace {

struct Int8Args {
  const void* x;     // pack: source, unpack: destination
  int64_t x_pitch;
  int8_t* codes;     // contiguous
  float* scales;
  int64_t groups;    // of all rows
  FastDiv per_row;   // groups of a row
  int cols;
};

struct GroupPos {
  int64_t x, code;  // offsets of the group's first element
  int count;        // its columns
};
// FLAT: contiguous rows of a multiple of 128 columns, groups of all rows lie one after the other.
template <bool FLAT>
__device__ __forceinline__ GroupPos locate(const Int8Args& a, int64_t g) {
  if constexpr (FLAT) return {g * kGroup, g * kGroup, kGroup};
  const uint32_t row = a.per_row.div((uint32_t)g);
  const int first = (int)((uint32_t)g - row * a.per_row.d) * kGroup;
  return {row * a.x_pitch + first, (int64_t)row * a.cols + first, min(kGroup, a.cols - first)};
}

constexpr int kUnroll = 4;  // groups a team works on at once, their loads issued before the first use

// VEC = 8: LANES lanes with eight elements each; the last piece of a row whose width is no multiple of eight (only possible
// in a single row) element by element.  VEC = 1: E elements each, LANES apart.
// A lane whose columns do not exist, or not all of them, loads the group's first ones instead and ignores them.
template <typename T, int VEC, int LANES, int E, bool FLAT, bool PACK>
__global__ void __launch_bounds__(256) int8_kernel(const Int8Args a) {
  griddep_wait();
  constexpr int TEAMS = 256 / LANES, STRIDE = VEC == 8 ? 1 : LANES;  // distance of a lane's elements
  constexpr int PIECES = E / VEC;
  const int lane = threadIdx.x % LANES;
  const int64_t g0 = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / LANES) * kUnroll;
  const int c0 = VEC == 8 ? lane * 8 : lane;
  GroupPos pos[kUnroll];
  bool live[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    live[u] = g0 + u < a.groups;
    pos[u] = locate<FLAT>(a, live[u] ? g0 + u : a.groups - 1);
  }
  // the column a lane loads its piece from
  auto column = [&](int u, int e) {
    const int c = c0 + e * STRIDE;
    return FLAT || c + VEC <= pos[u].count ? c : 0;
  };
  auto whole = [&](int u) { return VEC == 8 && (FLAT || c0 + 8 <= pos[u].count); };
  auto loadable = [&](int u) { return FLAT || VEC == 1 || pos[u].count >= 8; };
  if constexpr (PACK) {
    Piece<T, VEC> raw[kUnroll][PIECES];
    float amax[kUnroll], up[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const T* src = static_cast<const T*>(a.x) + pos[u].x;
#pragma unroll
      for (int e = 0; e < PIECES; ++e) {
        if (loadable(u)) raw[u][e].load(src + column(u, e));
        else raw[u][e].zero();
      }
    }
    float tail[kUnroll][FLAT || VEC == 1 ? 1 : 8];  // the ragged end of a single row
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float m = 0.f;
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < PIECES; ++e) {
          if (c0 + e * STRIDE >= pos[u].count) raw[u][e].zero();
          m = max_nan(m, raw[u][e].amax());
        }
      } else if (whole(u)) {
        m = raw[u][0].amax();
      } else if constexpr (!FLAT) {
        const T* src = static_cast<const T*>(a.x) + pos[u].x + c0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          tail[u][e] = c0 + e < pos[u].count ? to_f32(src[e]) : 0.f;
          m = max_nan(m, fabsf(tail[u][e]));
        }
      }
#pragma unroll
      for (int off = LANES / 2; off > 0; off >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
      amax[u] = m;
    }
    const float down = group_scales<kUnroll, LANES>(amax, up);
    if (lane < kUnroll && g0 + lane < a.groups) a.scales[g0 + lane] = down;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!live[u]) continue;
      int8_t* code = a.codes + pos[u].code + c0;
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < PIECES; ++e) {
          float x;
          raw[u][e].get(&x);
          if (c0 + e * STRIDE < pos[u].count) code[e * STRIDE] = code_of(x, up[u]);
        }
      } else if (whole(u)) {
        float x[8];
        raw[u][0].get(x);
        const uint64_t f = f2_dup(up[u]);
        const bool good = up[u] == up[u];
        *reinterpret_cast<uint2*>(code) = make_uint2(pack_codes(f2_pack(x[0], x[1]), f2_pack(x[2], x[3]), f, good),
                                                     pack_codes(f2_pack(x[4], x[5]), f2_pack(x[6], x[7]), f, good));
      } else if constexpr (!FLAT) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e < pos[u].count) code[e] = code_of(tail[u][e], up[u]);
      }
    }
  } else {
    using Raw = std::conditional_t<VEC == 1, int8_t, uint2>;
    Raw raw[kUnroll][PIECES];
    float down[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int8_t* code = a.codes + pos[u].code;
      down[u] = a.scales[live[u] ? g0 + u : a.groups - 1];
#pragma unroll
      for (int e = 0; e < PIECES; ++e)
        raw[u][e] = loadable(u) ? *reinterpret_cast<const Raw*>(code + column(u, e)) : Raw{};
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!live[u]) continue;
      T* dst = static_cast<T*>(const_cast<void*>(a.x)) + pos[u].x + c0;
      if constexpr (VEC == 1) {
#pragma unroll
        for (int e = 0; e < PIECES; ++e)
          if (c0 + e * STRIDE < pos[u].count) dst[e * STRIDE] = from_f32<T>((float)raw[u][e] * down[u]);
      } else if (whole(u)) {
        uint64_t p[4];
        unpack_codes(raw[u][0].x, p);
        unpack_codes(raw[u][0].y, p + 2);
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) f2_unpack(f2_mul(p[k], f2_dup(down[u])), x[2 * k], x[2 * k + 1]);
        store_vec<T, VEC>(dst, x);
      } else if constexpr (!FLAT) {
        const int8_t* code = a.codes + pos[u].code + c0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + e < pos[u].count) dst[e] = from_f32<T>((float)code[e] * down[u]);
      }
    }
  }
}

// Unpacking rows of a width that is no multiple of eight: codes and values lie at the same index of two contiguous arrays, so a
// thread takes eight from a boundary on, whatever row they are of.  The groups of all rows follow one another: eight elements
// are of a group and the next, or (a ragged group of fewer than eight among them) of a few more.
template <typename T>
__global__ void __launch_bounds__(256) int8_unpack_flat_kernel(const Int8Args a, int64_t n, FastDiv by_cols) {
  griddep_wait();
  T* x = static_cast<T*>(const_cast<void*>(a.x));
  const int64_t first = (int64_t)blockIdx.x * (256 * 8 * kUnroll) + threadIdx.x * 8;
  // of element i; how many elements from i on are in it; are eight in it and the next?
  auto group = [&](uint32_t i, int& left, bool& two) {
    const uint32_t row = by_cols.div(i);
    const int col = (int)(i - row * by_cols.d), after = (col / kGroup + 1) * kGroup;  // where the next group of the row begins
    left = min(a.cols - col, after - col);
    two = left + min(after < a.cols ? a.cols - after : a.cols, kGroup) >= 8;
    return (int64_t)row * a.per_row.d + col / kGroup;
  };
  uint2 raw[kUnroll];
  float s0[kUnroll], s1[kUnroll];
  int left[kUnroll];
  bool two[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * (256 * 8);
    if (i >= n) continue;
    const int64_t g = group((uint32_t)i, left[u], two[u]);
    s0[u] = a.scales[g];
    s1[u] = a.scales[g + 1 < a.groups ? g + 1 : g];
    if (i + 8 <= n) raw[u] = *reinterpret_cast<const uint2*>(a.codes + i);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = first + u * (256 * 8);
    if (i >= n) continue;
    if (i + 8 > n || !two[u]) {
      for (int e = 0; e < 8 && i + e < n; ++e) {
        int rest;
        bool unused;
        const int64_t g = group((uint32_t)(i + e), rest, unused);
        x[i + e] = from_f32<T>((float)a.codes[i + e] * a.scales[g]);
      }
      continue;
    }
    uint64_t p[4];
    unpack_codes(raw[u].x, p);
    unpack_codes(raw[u].y, p + 2);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) f2_unpack(p[k], v[2 * k], v[2 * k + 1]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= e < left[u] ? s0[u] : s1[u];
    store_vec<T, 8>(x + i, v);
  }
}

template <typename T, int VEC, int LANES, int E, bool FLAT, bool PACK>
int int8_launch(const Int8Args& a, cudaStream_t stream) {
  constexpr int per_block = 256 / LANES * kUnroll;
  launch_kernel(int8_kernel<T, VEC, LANES, E, FLAT, PACK>, dim3((unsigned)((a.groups + per_block - 1) / per_block)), dim3(256),
                0, stream, a);
  TPF_LAUNCH_OK();
  return TPF_OK;
}
template <typename T, bool PACK>
int int8_by_width(const Int8Args& a, bool vec, bool flat, cudaStream_t stream) {
  const int64_t n = a.groups / a.per_row.d * a.cols;
  if (!PACK && flat && n < (1ll << 31) - 256 * 8 * kUnroll) {
    launch_kernel(int8_unpack_flat_kernel<T>, dim3((unsigned)((n + 256 * 8 * kUnroll - 1) / (256 * 8 * kUnroll))), dim3(256), 0,
                  stream, a, n, FastDiv::make((uint32_t)a.cols));
    TPF_LAUNCH_OK();
    return TPF_OK;
  }
  if (!vec) {
    // Elements 32 apart with a warp a group leave lanes idle in narrow rows, and taking the maximum over fewer lanes is
    // cheaper (us; 600000 x 30 fp32, pack and unpack: 26 + 19, a warp a group 91 + 53; 300000 x 60 bf16 24 + 16, 50 + 29;
    // 300000 x 97 bf16 pack 43, 51).  Unpacking comes here from odd addresses or with 2^31 elements.
    if (a.cols <= 32) return int8_launch<T, 1, 8, 4, false, PACK>(a, stream);
    if (PACK) return a.cols <= 64 ? int8_launch<T, 1, 8, 8, false, true>(a, stream) : int8_launch<T, 1, 16, 8, false, true>(a, stream);
    return a.cols <= 64 ? int8_launch<T, 1, 16, 4, false, false>(a, stream) : int8_launch<T, 1, 32, 4, false, false>(a, stream);
  }
  if (a.cols % kGroup == 0 && a.x_pitch == a.cols) return int8_launch<T, 8, 16, 8, true, PACK>(a, stream);
  if (a.cols <= 32) return int8_launch<T, 8, 4, 8, false, PACK>(a, stream);
  if (a.cols <= 64) return int8_launch<T, 8, 8, 8, false, PACK>(a, stream);
  return int8_launch<T, 8, 16, 8, false, PACK>(a, stream);
}

template <bool PACK>
int int8_run(const char* who, const void* x, int64_t pitch, int type, void* codes, float* scales, int64_t rows, int64_t cols,
             cudaStream_t stream) {
  TPF_REQUIRE(row_type_ok(type), TPF_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", who, type);
  TPF_REQUIRE(rows >= 0 && cols >= 0, TPF_ERR_INVALID_ARGUMENT, "%s: extents must not be negative", who);
  if (rows == 0 || cols == 0) return TPF_OK;
  TPF_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, TPF_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  const int64_t per_row = row_groups(cols);
  TPF_REQUIRE(cols < (1ll << 31) - kGroup && rows < (1ll << 31) && per_row * rows < (1ll << 31) - 1024, TPF_ERR_UNSUPPORTED,
              "%s: at most 2^31 groups and columns", who);
  TPF_REQUIRE(rows == 1 || pitch >= cols || (PACK && pitch == 0), TPF_ERR_INVALID_ARGUMENT, "%s: rows overlap", who);
  const bool vec = vec_ok(x, type) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0 &&
                   (rows == 1 || (cols % 8 == 0 && pitch % 8 == 0));
  const Int8Args a{x, rows == 1 ? cols : pitch, static_cast<int8_t*>(codes), scales, per_row * rows, FastDiv::make((uint32_t)per_row),
                   (int)cols};
  // (300000 x 97 bf16: 20 us, 30 element by element; 600000 x 17 7.2, 16)
  const bool flat = !vec && a.x_pitch == cols && vec_ok(x, type) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  if (type == kRowF32) return int8_by_width<float, PACK>(a, vec, flat, stream);
  if (type == kRowBF16) return int8_by_width<bf16, PACK>(a, vec, flat, stream);
  return int8_by_width<__half, PACK>(a, vec, flat, stream);
}

}  // namespace

int int8_pack(const void* x, int64_t x_pitch, int type, void* codes, float* scales, int64_t rows, int64_t cols,
              cudaStream_t stream) {
  return int8_run<true>("int8_pack", x, x_pitch, type, codes, scales, rows, cols, stream);
}
int int8_unpack(const void* codes, const float* scales, int type, void* x, int64_t rows, int64_t cols,
                cudaStream_t stream) {
  return int8_run<false>("int8_unpack", x, cols, type, const_cast<void*>(codes), const_cast<float*>(scales), rows, cols,
                         stream);
}

}  // namespace tpf

// Activations put away in 8 bits and taken out again (the format is described in tpf_rows.cuh).
//
// Both directions are bound by memory: three bytes an element in bf16.  The unit of work is a group of 128 elements.  Where
// eight elements can be accessed at once, LANES = 4, 8 or 16 lanes hold a group (of 32, 64 or more columns), else a warp
// does, a lane with every 32nd element.
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
  int64_t row;
  int first, count;  // columns
};
__device__ __forceinline__ GroupPos locate(const Int8Args& a, int64_t g) {
  const uint32_t row = a.per_row.div((uint32_t)g);
  const int first = (int)((uint32_t)g - row * a.per_row.d) * kGroup;
  return {row, first, min(kGroup, a.cols - first)};
}

constexpr int kUnroll = 4;  // groups a team works on at once, their loads issued before the first use

// VEC = 8: LANES lanes with eight elements each; the last piece of a row whose width is no multiple of eight (only possible
// in a single row) element by element.  VEC = 1: 32 lanes, four elements each, 32 apart.
template <typename T, int VEC, int LANES, bool PACK>
__global__ void __launch_bounds__(256) int8_kernel(const Int8Args a) {
  griddep_wait();
  constexpr int TEAMS = 256 / LANES, STRIDE = VEC == 8 ? 1 : 32;  // distance of a lane's elements
  static_assert(VEC == 8 || LANES == 32, "");
  constexpr int E = VEC == 8 ? 8 : 4;
  const int lane = threadIdx.x % LANES;
  const int64_t g0 = ((int64_t)blockIdx.x * TEAMS + threadIdx.x / LANES) * kUnroll;
  float x[kUnroll][E], down[kUnroll];
  uint2 w[kUnroll];
  GroupPos pos[kUnroll];
  const int c0 = VEC == 8 ? lane * 8 : lane;
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    pos[u] = g0 + u < a.groups ? locate(a, g0 + u) : GroupPos{0, 0, 0};
    const int left = pos[u].count - c0;  // columns of this lane and those behind it
    const T* src = static_cast<const T*>(a.x) + pos[u].row * a.x_pitch + pos[u].first + c0;
    const int8_t* code = a.codes + pos[u].row * a.cols + pos[u].first + c0;
    if constexpr (PACK) {
      if (VEC == 8 && left >= 8) {
        load_vec<T, 8>(src, x[u]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = e * STRIDE < left ? to_f32(src[e * STRIDE]) : 0.f;
      }
    } else {
      down[u] = pos[u].count > 0 ? a.scales[g0 + u] : 0.f;
      if (VEC == 8 && left >= 8) {
        w[u] = *reinterpret_cast<const uint2*>(code);
      } else {
        w[u] = make_uint2(0u, 0u);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e * STRIDE < left) (e < 4 ? w[u].x : w[u].y) |= (uint32_t)(uint8_t)code[e * STRIDE] << (8 * (e & 3));
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int left = pos[u].count - c0;
    if constexpr (PACK) {
      float m = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) m = max_nan(m, fabsf(x[u][e]));
#pragma unroll
      for (int off = LANES / 2; off > 0; off >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
      const GroupScale s = group_scale(m);
      int8_t* code = a.codes + pos[u].row * a.cols + pos[u].first + c0;
      if (VEC == 8 && left >= 8) {
        store_codes<VEC>(code, x[u], s);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e * STRIDE < left) code[e * STRIDE] = code_of(x[u][e], s);
      }
      if (lane == 0 && pos[u].count > 0) a.scales[g0 + u] = s.down;
    } else {
      unpack_codes(w[u].x, down[u], x[u]);
      if constexpr (E == 8) unpack_codes(w[u].y, down[u], x[u] + 4);
      T* dst = static_cast<T*>(const_cast<void*>(a.x)) + pos[u].row * a.x_pitch + pos[u].first + c0;
      if (VEC == 8 && left >= 8) {
        store_vec<T, VEC>(dst, x[u]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e * STRIDE < left) dst[e * STRIDE] = from_f32<T>(x[u][e]);
      }
    }
  }
}

template <typename T, int VEC, int LANES, bool PACK>
int int8_launch(const Int8Args& a, cudaStream_t stream) {
  constexpr int per_block = 256 / LANES * kUnroll;
  launch_kernel(int8_kernel<T, VEC, LANES, PACK>, dim3((unsigned)((a.groups + per_block - 1) / per_block)), dim3(256), 0,
                stream, a);
  TPF_LAUNCH_OK();
  return TPF_OK;
}
template <typename T, bool PACK>
int int8_by_width(const Int8Args& a, bool vec, cudaStream_t stream) {
  if (!vec) return int8_launch<T, 1, 32, PACK>(a, stream);
  if (a.cols <= 32) return int8_launch<T, 8, 4, PACK>(a, stream);
  if (a.cols <= 64) return int8_launch<T, 8, 8, PACK>(a, stream);
  return int8_launch<T, 8, 16, PACK>(a, stream);
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
  const Int8Args a{x, pitch, static_cast<int8_t*>(codes), scales, per_row * rows, FastDiv::make((uint32_t)per_row),
                   (int)cols};
  if (type == kRowF32) return int8_by_width<float, PACK>(a, vec, stream);
  if (type == kRowBF16) return int8_by_width<bf16, PACK>(a, vec, stream);
  return int8_by_width<__half, PACK>(a, vec, stream);
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

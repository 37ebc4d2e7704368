// What the two passes of the layer norm share: arguments, the choice of a team by width, checks.
#pragma once

#include "tpf_rows.cuh"
#include "tpf_rows.h"

namespace tpf {

struct NormArgs {
  const void* x;
  int64_t x_pitch;
  int8_t* codes;
  float* scales;
  float *mean, *rstd;
  ParamVec w, b;
  int64_t rows;
  int cols, groups, code_pitch;
  float inv_cols;
};

// The rows row0, row0 + 1, .. of a team in one round: what does not exist is loaded from the last row instead.
template <int ROWS>
struct RowSet {
  int64_t first;  // exists
  int count;      // rows that exist, 0 .. ROWS
  int last;       // distance of the last row that exists
  __device__ __forceinline__ RowSet(int64_t row0, int64_t rows) {
    const int64_t left = rows - row0;
    first = left > 0 ? row0 : rows - 1;
    count = left >= ROWS ? ROWS : left > 0 ? (int)left : 0;
    last = count > 0 ? count - 1 : 0;
  }
  __device__ __forceinline__ int at(int r) const { return min(r, last); }
};

// Rows a team has in flight at a time, with as many again on their way in registers.  128 registers a thread (two CTAs of
// 256) and this many rows measured best: the forward of 768 * 768 rows of 128 bf16 channels, eight elements a thread, takes
// 50.6 us with four rows, 53 with two and 62 with one; the backward 82 with two, 89 with four (no room left), 90 with one.
template <typename T, class Tm, bool BWD>
constexpr int rows_in_flight() {
  if (Tm::E >= 32 || (Tm::VEC == 1 && Tm::E >= 8)) return 1;
  if (Tm::E >= 16) return BWD ? 1 : 2;
  if (sizeof(T) == 4) return BWD ? 1 : 2;
  return BWD ? 2 : 4;
}
template <class Tm, bool BWD>
constexpr int min_ctas() {
  return Tm::MAXB >= 512 || (BWD && Tm::E >= 32) ? 1 : 512 / Tm::MAXB;
}

// CTAs of `kern` that an SM holds at this block size, from the kernel's registers (looked up once per device).
template <class Kernel>
inline int resident_ctas(Kernel kern, int threads, PerDeviceInt& cache, int* out) {
  int dev = 0;
  if (int rc = current_device(&dev)) return rc;
  int regs = cache.v[dev].load(std::memory_order_acquire);
  if (regs == 0) {
    cudaFuncAttributes attr;
    TPF_CUDA_OK(cudaFuncGetAttributes(&attr, kern));
    regs = attr.numRegs;
    cache.v[dev].store(regs, std::memory_order_release);
  }
  const int warps = 4 * (16384 / ((regs + 7) / 8 * 8 * 32));  // a scheduler has 16384 registers
  int n = warps / (threads / 32);
  if (n > 2048 / threads) n = 2048 / threads;
  *out = n < 1 ? 1 : n;
  return TPF_OK;
}

template <class Launch>
inline int by_type(const Launch& l, int type, int cols, bool vec) {
  if (type == kRowF32) return l.template by_width<float>(cols, vec);
  if (type == kRowBF16) return l.template by_width<bf16>(cols, vec);
  return l.template by_width<__half>(cols, vec);
}

inline int make_norm_args(NormArgs* a, const NormCall& c, const char* who) {
  TPF_REQUIRE(row_type_ok(c.type), TPF_ERR_INVALID_ARGUMENT, "%s: unknown element type %d", who, c.type);
  TPF_REQUIRE(c.rows >= 0, TPF_ERR_INVALID_ARGUMENT, "%s: rows must not be negative", who);
  TPF_REQUIRE(c.cols >= 1 && c.cols <= kMaxNormCols, TPF_ERR_UNSUPPORTED, "%s: 1 to %lld columns, got %lld", who,
              (long long)kMaxNormCols, (long long)c.cols);
  TPF_REQUIRE((c.codes == nullptr) == (c.scales == nullptr), TPF_ERR_INVALID_ARGUMENT,
              "%s: codes and scales come together", who);
  TPF_REQUIRE((c.mean == nullptr) == (c.rstd == nullptr), TPF_ERR_INVALID_ARGUMENT, "%s: mean and rstd come together", who);
  TPF_REQUIRE((c.weight == nullptr || row_type_ok(c.weight_type)) && (c.bias == nullptr || row_type_ok(c.bias_type)),
              TPF_ERR_INVALID_ARGUMENT, "%s: unknown parameter type", who);
  TPF_REQUIRE(c.x == nullptr || c.rows <= 1 || c.x_pitch >= c.cols || c.x_pitch == 0, TPF_ERR_INVALID_ARGUMENT,
              "%s: rows overlap", who);
  *a = NormArgs{c.x, c.x_pitch, static_cast<int8_t*>(c.codes), c.scales, c.mean, c.rstd, {c.weight, c.weight_type},
                {c.bias, c.bias_type}, c.rows, (int)c.cols, (int)row_groups(c.cols), (int)code_pitch(c.cols), 1.f / (float)c.cols};
  return TPF_OK;
}
// May rows at p with this pitch be accessed eight elements at a time?
inline bool rows_vec_ok(const void* p, int64_t pitch, int type) {
  return p == nullptr || (vec_ok(p, type) && pitch % 8 == 0);
}

}  // namespace tpf

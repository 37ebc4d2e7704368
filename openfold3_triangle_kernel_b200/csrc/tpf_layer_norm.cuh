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
  int cols, groups;
  float inv_cols;
};

template <class Tm>
constexpr int rows_in_flight() {  // 32 elements a thread, four rows at most; one where single elements are loaded
  return Tm::E >= 32 || (Tm::VEC == 1 && Tm::E >= 16) ? 1 : Tm::E >= 16 ? 2 : 4;
}

// The team for rows of `cols` elements: as few threads as hold the row in 32 elements each (fewer for narrow rows, so that
// a team covers little more than the row).  vec: eight elements at a time are possible.
template <typename T, class Launch>
inline int by_width(const Launch& l, int cols, bool vec) {
  if (vec) {
    if (cols <= 32) return l.template run<T, Team<8, 4, 1>>();
    if (cols <= 64) return l.template run<T, Team<8, 8, 1>>();
    if (cols <= 128) return l.template run<T, Team<8, 16, 1>>();
    if (cols <= 256) return l.template run<T, Team<8, 32, 1>>();
    if (cols <= 512) return l.template run<T, Team<8, 32, 2>>();
    if (cols <= 1024) return l.template run<T, Team<8, 32, 4>>();
    if (cols <= 2048) return l.template run<T, Team<8, 64, 4>>();
    if (cols <= 4096) return l.template run<T, Team<8, 128, 4>>();
    return l.template run<T, Team<8, 256, 4>>();
  }
  if (cols <= 128) return l.template run<T, Team<1, 32, 4>>();
  if (cols <= 512) return l.template run<T, Team<1, 32, 16>>();
  if (cols <= 1024) return l.template run<T, Team<1, 64, 16>>();
  if (cols <= 2048) return l.template run<T, Team<1, 128, 16>>();
  if (cols <= 4096) return l.template run<T, Team<1, 256, 16>>();
  return l.template run<T, Team<1, 512, 16>>();
}

template <class Launch>
inline int by_type(const Launch& l, int type, int cols, bool vec) {
  if (type == kRowF32) return by_width<float>(l, cols, vec);
  if (type == kRowBF16) return by_width<bf16>(l, cols, vec);
  return by_width<__half>(l, cols, vec);
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
                {c.bias, c.bias_type}, c.rows, (int)c.cols, (int)row_groups(c.cols), 1.f / (float)c.cols};
  return TPF_OK;
}
// May rows at p with this pitch be accessed eight elements at a time?
inline bool rows_vec_ok(const void* p, int64_t pitch, int type) {
  return p == nullptr || (vec_ok(p, type) && pitch % 8 == 0);
}

}  // namespace tpf

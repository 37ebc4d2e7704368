// Row-wise operators for eager CUDA tensors: layer norm, 8-bit checkpoints, normalised projection.
#include <torch/csrc/Dtype.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>

#include "tpf_rows.h"
#include "tpf_torch.h"
#include "tpf_torch_trimul.h"

namespace tpf_torch {

namespace {

constexpr int64_t kMaxCols = 8192;  // of a layer norm (tpf_layer_norm_fwd)
constexpr int64_t kMaxLinearRows = (1ll << 31) - 256, kMaxOuts = 1ll << 30;  // of a projection (tpf_norm_linear_fwd)

// Straight from the allocator of the current device: a tensor through the dispatcher costs 1.2 us, and a small training
// pass makes six.
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
struct Scratch {  // device memory of a call
  c10::DataPtr p;
  explicit Scratch(int64_t bytes) {
    if (bytes > 0) p = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  }
  void* get() const { return p.get(); }
};

cudaStream_t cu_stream() { return static_cast<cudaStream_t>(stream()); }

int row_type(const Tensor& t) {  // -1: not a type of these operators
  switch (t.scalar_type()) {
    case at::kFloat: return TPF_F32;
    case at::kBFloat16: return TPF_BF16;
    case at::kHalf: return TPF_F16;
    default: return -1;
  }
}

// A tensor [*, C] as rows of one pitch: read in place where its strides allow it, else a contiguous copy.
struct Rows {
  Tensor t;
  int64_t pitch, rows, cols;
};
Rows as_rows(const Tensor& t) {
  const int64_t nd = t.dim(), C = t.size(nd - 1);
  Rows r{t, C, 1, C};
  for (int64_t i = 0; i < nd - 1; ++i) r.rows *= t.size(i);
  if (t.is_contiguous()) return r;
  bool ok = C == 1 || t.stride(nd - 1) == 1, first = true;
  int64_t next = 0;
  for (int64_t i = nd - 2; ok && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (first) r.pitch = t.stride(i);
    else ok = t.stride(i) == next;
    first = false;
    next = t.stride(i) * t.size(i);
  }
  if (!ok || (r.pitch < C && r.pitch != 0)) {
    r.t = t.contiguous();
    r.pitch = C;
  }
  return r;
}
Rows as_vector_rows(const Tensor& t) {  // bf16 rows that start on 16-byte boundaries
  Rows r = as_rows(t);
  if (r.pitch >= r.cols && r.pitch % 8 == 0 && (reinterpret_cast<uintptr_t>(r.t.data_ptr()) & 15) == 0) return r;
  r.t = t.is_contiguous() ? t.clone() : t.contiguous();
  if (reinterpret_cast<uintptr_t>(r.t.data_ptr()) & 15) r.t = r.t.clone();
  r.pitch = r.cols;
  return r;
}

using MaybeTensor = std::optional<Tensor>;
Tensor value_or_none(const MaybeTensor& t) { return t ? t->detach().contiguous() : Tensor(); }
void* ptr_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
int type_of(const Tensor& t) { return t.defined() ? row_type(t) : 0; }

tpf::NormCall norm_call(const Rows& x, const Tensor& w, const Tensor& b) {
  tpf::NormCall c = {};
  c.rows = x.rows;
  c.cols = x.cols;
  c.type = row_type(x.t);
  c.x = x.t.data_ptr();
  c.x_pitch = x.pitch;
  c.weight = ptr_of(w);
  c.bias = ptr_of(b);
  c.weight_type = type_of(w);
  c.bias_type = type_of(b);
  return c;
}

// What a forward keeps beside or in place of x: mean and rstd [2, rows]; codes [rows, code_pitch(cols)] and scales
// [rows, groups].
struct Kept {
  Tensor stats, codes, scales;
};
Kept make_kept(tpf::NormCall& c, const Tensor& like, bool save, bool int8) {
  Kept k;
  if (!save) return k;
  k.stats = make({2, c.rows}, at::kFloat, like);
  c.mean = fptr(k.stats);
  c.rstd = c.mean + c.rows;
  if (int8) {
    k.codes = make({c.rows, tpf::code_pitch(c.cols)}, at::kChar, like);
    k.scales = make({c.rows, (c.cols + 127) / 128}, at::kFloat, like);
    c.codes = k.codes.data_ptr();
    c.scales = fptr(k.scales);
  }
  return k;
}

// The call of a backward pass from what was kept; `x`: the rows as they were, unused where there are codes.
tpf::NormCall kept_call(const Rows& x, const Kept& k, const Tensor& w, const Tensor& b, int type, int64_t cols) {
  tpf::NormCall c = {};
  c.rows = k.stats.size(1);
  c.cols = cols;
  c.type = type;
  if (k.codes.defined()) {
    c.codes = k.codes.data_ptr();
    c.scales = fptr(k.scales);
  } else {
    c.x = x.t.data_ptr();
    c.x_pitch = x.pitch;
  }
  c.mean = fptr(k.stats);
  c.rstd = c.mean + c.rows;
  c.weight = ptr_of(w);
  c.bias = ptr_of(b);
  c.weight_type = type_of(w);
  c.bias_type = type_of(b);
  return c;
}

Tensor param_grad(const Tensor& p) { return make(p.sizes(), p.scalar_type(), p); }

Tensor layer_norm_out(const Rows& x, at::IntArrayRef sizes, const Tensor& w, const Tensor& b, double eps, Kept* kept,
                      bool int8) {
  tpf::NormCall c = norm_call(x, w, b);
  Kept k = make_kept(c, x.t, kept != nullptr, int8);
  Tensor y = make(sizes, x.t.scalar_type(), x.t);
  check(tpf::layer_norm_fwd(c, y.data_ptr(), (float)eps, cu_stream()), "tpf_layer_norm_fwd");
  if (kept != nullptr) *kept = k;
  return y;
}

struct NormGradTensors {
  Tensor dx, dw, db;
};
NormGradTensors layer_norm_grads(const tpf::NormCall& c, const Tensor& dy, at::IntArrayRef sizes, const Tensor& w,
                                 const Tensor& b, bool need_x, bool need_w, bool need_b) {
  NormGradTensors r;
  if (need_x) r.dx = make(sizes, dy.scalar_type(), dy);
  if (need_w) r.dw = param_grad(w);
  if (need_b) r.db = param_grad(b);
  const int64_t n = need_w || need_b ? tpf_layer_norm_bwd_workspace_bytes(c.rows, c.cols) : 0;
  const Scratch ws(n);
  const tpf::NormGrads g{dy.data_ptr(), ptr_of(r.dx), ptr_of(r.dw), ptr_of(r.db), type_of(w), type_of(b)};
  check(tpf::layer_norm_bwd(c, g, ws.get(), n, cu_stream()), "tpf_layer_norm_bwd");
  return r;
}

struct LayerNormFn : public torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const MaybeTensor& w_in, const MaybeTensor& b_in,
                        double eps, bool save, bool int8) {
    const Rows x = as_rows(x_in.detach());
    const Tensor w = value_or_none(w_in), b = value_or_none(b_in);
    Kept k;
    Tensor y = layer_norm_out(x, x_in.sizes(), w, b, eps, save ? &k : nullptr, int8);
    if (save) {
      // x itself where its rows were read in place, so that a change to it before the backward is noticed
      const Tensor kept_x = int8 ? Tensor() : x.t.data_ptr() == x_in.data_ptr() ? x_in : x.t;
      ctx->save_for_backward({kept_x, k.stats, k.codes, k.scales, w_in ? *w_in : Tensor(), b_in ? *b_in : Tensor()});
    }
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return first_order(grads, gradients(ctx, grads));
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list r(6);
    if (!grads[0].defined()) return r;
    const auto saved = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    at::NoGradGuard no_grad;
    const Tensor dy = grads[0].contiguous();  // (the engine has seen to y's type and shape, which are x's)
    const auto sizes = dy.sizes();
    const Tensor w = saved[4].defined() ? saved[4].contiguous() : Tensor(), &b = saved[5];
    const Rows x = saved[0].defined() ? as_rows(saved[0]) : Rows{};
    const tpf::NormCall c = kept_call(x, {saved[1], saved[2], saved[3]}, w, Tensor(), row_type(dy), sizes.back());
    const int iw = 1, ib = w.defined() ? 2 : 1;  // an absent parameter has no edge
    const bool need_w = w.defined() && ctx->needs_input_grad(iw), need_b = b.defined() && ctx->needs_input_grad(ib);
    const NormGradTensors g = layer_norm_grads(c, dy, sizes, w, b, ctx->needs_input_grad(0), need_w, need_b);
    r[0] = g.dx;
    r[1] = g.dw;
    r[2] = g.db;
    return r;
  }
};

Tensor as_bf16_matrix(const Tensor& w) {
  Tensor t = (w.scalar_type() == at::kBFloat16 ? w : w.to(at::kBFloat16)).contiguous();
  return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15 ? t.clone() : t;
}

std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s = sizes.vec();
  s.back() = last;
  return s;
}

Tensor norm_linear_out(const Rows& x, at::IntArrayRef sizes, const Tensor& nw, const Tensor& nb, const Tensor& w, double eps,
                       Kept* kept, bool int8) {
  tpf::NormCall c = norm_call(x, nw, nb);
  Kept k = make_kept(c, x.t, kept != nullptr, int8);
  const int64_t outs = w.size(0);
  Tensor out = make(with_last(sizes, outs), at::kBFloat16, x.t);
  const int64_t n = tpf_norm_linear_fwd_workspace_bytes(c.rows, c.cols, outs);
  const Scratch ws(n);
  check(tpf::norm_linear_fwd(c, w.data_ptr(), outs, out.data_ptr(), (float)eps, ws.get(), n, cu_stream()),
        "tpf_norm_linear_fwd");
  if (kept != nullptr) *kept = k;
  return out;
}

struct LinearGradTensors {
  Tensor dx, dnw, dnb, dw;
};
// nw, nb: the norm's parameters, contiguous or undefined; w: the caller's weight (its type is the gradient's).
LinearGradTensors norm_linear_grads(const tpf::NormCall& c, const Tensor& d_out, at::IntArrayRef sizes, const Tensor& nw,
                                    const Tensor& nb, const Tensor& w, bool need_x, bool need_nw, bool need_nb,
                                    bool need_w) {
  LinearGradTensors r;
  const int64_t outs = w.size(0);
  const Tensor wb = as_bf16_matrix(w);
  if (need_x) r.dx = make(sizes, at::kBFloat16, d_out);
  if (need_nw) r.dnw = param_grad(nw);
  if (need_nb) r.dnb = param_grad(nb);
  if (need_w) r.dw = make({outs, c.cols}, w.scalar_type(), w);
  const int64_t n = tpf_norm_linear_bwd_workspace_bytes(c.rows, c.cols, outs);
  const Scratch ws(n);
  const tpf::NormLinearGrads g{d_out.data_ptr(), ptr_of(r.dx), ptr_of(r.dnw), ptr_of(r.dnb), type_of(nw), type_of(nb),
                               ptr_of(r.dw), row_type(w)};
  check(tpf::norm_linear_bwd(c, wb.data_ptr(), outs, g, ws.get(), n, cu_stream()), "tpf_norm_linear_bwd");
  return r;
}

struct NormLinearFn : public torch::autograd::Function<NormLinearFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_in, const Tensor& w_in, const MaybeTensor& nw_in,
                        const MaybeTensor& nb_in, double eps, bool save, bool int8) {
    const Rows x = as_vector_rows(x_in.detach());
    const Tensor nw = value_or_none(nw_in), nb = value_or_none(nb_in);
    Kept k;
    Tensor out = norm_linear_out(x, x_in.sizes(), nw, nb, as_bf16_matrix(w_in.detach()), eps, save ? &k : nullptr, int8);
    if (save) {
      const Tensor kept_x = int8 ? Tensor() : x.t.data_ptr() == x_in.data_ptr() ? x_in : x.t;
      ctx->save_for_backward(
          {kept_x, k.stats, k.codes, k.scales, nw_in ? *nw_in : Tensor(), nb_in ? *nb_in : Tensor(), w_in});
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return first_order(grads, gradients(ctx, grads));
  }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list r(7);
    if (!grads[0].defined()) return r;
    const auto saved = ctx->get_saved_variables();
    c10::cuda::CUDAGuard guard(grads[0].device());
    at::NoGradGuard no_grad;
    const Tensor d_out = aligned_bf16(grads[0]);
    const std::vector<int64_t> sizes = with_last(d_out.sizes(), saved[6].size(1));
    const Tensor nw = saved[4].defined() ? saved[4].contiguous() : Tensor();
    const Tensor nb = saved[5].defined() ? saved[5].contiguous() : Tensor();
    const Rows x = saved[0].defined() ? as_vector_rows(saved[0]) : Rows{};
    const tpf::NormCall c = kept_call(x, {saved[1], saved[2], saved[3]}, nw, nb, TPF_BF16, sizes.back());
    const int inw = 2, inb = nw.defined() ? 3 : 2;  // an absent parameter has no edge
    const LinearGradTensors g = norm_linear_grads(
        c, d_out, sizes, nw, nb, saved[6], ctx->needs_input_grad(0), nw.defined() && ctx->needs_input_grad(inw),
        nb.defined() && ctx->needs_input_grad(inb), ctx->needs_input_grad(1));
    r[0] = g.dx;
    r[1] = g.dw;
    r[2] = g.dnw;
    r[3] = g.dnb;
    return r;
  }
};

// An optional parameter: false if it needs the Python route.
bool unpack_param(py::handle h, const Tensor& x, int64_t cols, MaybeTensor& out) {
  if (h.is_none()) return true;
  if (!plain_type(h)) return false;
  out = THPVariable_Unpack(h.ptr());
  return plain_cuda(*out) && out->device() == x.device() && row_type(*out) >= 0 && out->dim() == 1 && out->size(0) == cols;
}
bool wants_grad(const MaybeTensor& t) { return t && t->requires_grad(); }

}  // namespace

// The eager calls return None when the arguments need the Python route: an unsupported case (which raises there, with its
// reason), a tensor subclass, an active dispatch mode.
py::object py_layer_norm(py::handle hx, py::handle hw, py::handle hb, double eps, bool int8) {
  if (!plain_type(hx) || !plain_context()) return py::none();
  const Tensor& x = THPVariable_Unpack(hx.ptr());
  if (!plain_cuda(x) || !device_supported(x) || row_type(x) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kMaxCols ||
      !(eps >= 0))
    return py::none();
  MaybeTensor w, b;
  if (!unpack_param(hw, x, x.size(-1), w) || !unpack_param(hb, x, x.size(-1), b)) return py::none();
  const bool save = at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b));
  Tensor y;
  {
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(x.device());
    if (save) {
      y = LayerNormFn::apply(x, w, b, eps, true, int8);
    } else {
      at::NoGradGuard no_grad;
      y = LayerNormFn::forward(nullptr, x, w, b, eps, false, false);
    }
  }
  return py::cast(y);
}

py::object py_norm_linear(py::handle hx, py::handle hnw, py::handle hnb, py::handle hw, double eps, bool int8) {
  if (!plain_type(hx) || !plain_type(hw) || !plain_context()) return py::none();
  const Tensor &x = THPVariable_Unpack(hx.ptr()), &w = THPVariable_Unpack(hw.ptr());
  if (!plain_cuda(x) || !plain_cuda(w) || !device_supported(x) || x.scalar_type() != at::kBFloat16 || x.dim() < 1 ||
      w.device() != x.device() || w.dim() != 2 || row_type(w) < 0 || !(eps >= 0))
    return py::none();
  const int64_t cols = x.size(-1), outs = w.size(0);
  if (cols < 8 || cols % 8 || cols > kMaxCols || w.size(1) != cols || outs < 8 || outs % 8 || outs > kMaxOuts ||
      x.numel() / cols >= kMaxLinearRows)
    return py::none();
  MaybeTensor nw, nb;
  if (!unpack_param(hnw, x, cols, nw) || !unpack_param(hnb, x, cols, nb)) return py::none();
  const bool save =
      at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || wants_grad(nw) || wants_grad(nb));
  Tensor out;
  {
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(x.device());
    if (save) {
      out = NormLinearFn::apply(x, w, nw, nb, eps, true, int8);
    } else {
      at::NoGradGuard no_grad;
      out = NormLinearFn::forward(nullptr, x, w, nw, nb, eps, false, false);
    }
  }
  return py::cast(out);
}

// Launches behind the torch.library operators, which have checked the arguments.  Absent tensors of an output list are empty.
Kept kept_args(const MaybeTensor& x, const Tensor& stats, const Tensor& codes, const Tensor& scales) {
  return {stats.contiguous(), x ? Tensor() : codes.contiguous(), scales.contiguous()};
}
std::vector<Tensor> layer_norm_fwd(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps, bool int8) {
  c10::cuda::CUDAGuard guard(x.device());
  Kept k;
  Tensor y = layer_norm_out(as_rows(x), x.sizes(), value_or_none(w), value_or_none(b), eps, &k, int8);
  if (!int8) {
    k.codes = at::empty({0}, x.options().dtype(at::kChar));
    k.scales = empty_f32({0}, x);
  }
  return {y, k.stats, k.codes, k.scales};
}

std::vector<Tensor> layer_norm_bwd(const Tensor& dy, const MaybeTensor& x, const Tensor& stats, const Tensor& codes,
                                   const Tensor& scales, const MaybeTensor& w, const MaybeTensor& b) {
  c10::cuda::CUDAGuard guard(dy.device());
  const Rows rows = x ? as_rows(*x) : Rows{};
  const Tensor wc = value_or_none(w), bc = value_or_none(b), d = dy.contiguous();
  const Kept k = kept_args(x, stats, codes, scales);
  const tpf::NormCall c = kept_call(rows, k, wc, Tensor(), row_type(dy), dy.size(-1));
  NormGradTensors g = layer_norm_grads(c, d, dy.sizes(), wc, bc, true, wc.defined(), bc.defined());
  const Tensor none = empty_f32({0}, dy);
  return {g.dx, g.dw.defined() ? g.dw : none, g.db.defined() ? g.db : none.clone()};
}

std::vector<Tensor> norm_linear_fwd(const Tensor& x, const MaybeTensor& nw, const MaybeTensor& nb, const Tensor& w,
                                    double eps, bool int8) {
  c10::cuda::CUDAGuard guard(x.device());
  Kept k;
  Tensor out = norm_linear_out(as_vector_rows(x), x.sizes(), value_or_none(nw), value_or_none(nb), as_bf16_matrix(w), eps,
                               &k, int8);
  if (!int8) {
    k.codes = at::empty({0}, x.options().dtype(at::kChar));
    k.scales = empty_f32({0}, x);
  }
  return {out, k.stats, k.codes, k.scales};
}

std::vector<Tensor> norm_linear_bwd(const Tensor& d_out, const MaybeTensor& x, const Tensor& stats, const Tensor& codes,
                                    const Tensor& scales, const MaybeTensor& nw, const MaybeTensor& nb, const Tensor& w) {
  c10::cuda::CUDAGuard guard(d_out.device());
  const Rows rows = x ? as_vector_rows(*x) : Rows{};
  const Tensor nwc = value_or_none(nw), nbc = value_or_none(nb), d = aligned_bf16(d_out);
  const Kept k = kept_args(x, stats, codes, scales);
  const tpf::NormCall c = kept_call(rows, k, nwc, nbc, TPF_BF16, w.size(1));
  LinearGradTensors g = norm_linear_grads(c, d, with_last(d_out.sizes(), w.size(1)), nwc, nbc, w, true, nwc.defined(),
                                          nbc.defined(), true);
  const Tensor none = empty_f32({0}, d_out);
  return {g.dx, g.dw, g.dnw.defined() ? g.dnw : none, g.dnb.defined() ? g.dnb : none.clone()};
}

std::vector<Tensor> int8_pack(const Tensor& t) {
  c10::cuda::CUDAGuard guard(t.device());
  const Rows x = as_rows(t);
  std::vector<int64_t> groups = with_last(t.sizes(), (x.cols + 127) / 128);
  Tensor codes = make(t.sizes(), at::kChar, t), scales = make(groups, at::kFloat, t);
  check(tpf::int8_pack(x.t.data_ptr(), x.pitch, row_type(t), codes.data_ptr(), fptr(scales), x.rows, x.cols, cu_stream()),
        "tpf_int8_pack");
  return {codes, scales};
}

Tensor int8_unpack(const Tensor& codes_in, const Tensor& scales_in, int64_t type) {
  c10::cuda::CUDAGuard guard(codes_in.device());
  const Tensor codes = codes_in.contiguous(), scales = scales_in.contiguous();
  const int64_t cols = codes.size(-1);
  int64_t rows = 1;
  for (int64_t i = 0; i < codes.dim() - 1; ++i) rows *= codes.size(i);
  Tensor x = make(codes.sizes(), (at::ScalarType)type, codes);
  check(tpf::int8_unpack(codes.data_ptr(), fptr(scales), row_type(x), x.data_ptr(), rows, cols, cu_stream()),
        "tpf_int8_unpack");
  return x;
}

// Fewer groups and columns than the kernels can count?
bool few_groups(const Tensor& x) {
  const int64_t cols = x.size(-1);
  return cols == 0 || (cols < (1ll << 31) - 128 && x.numel() / cols * ((cols + 127) / 128) < (1ll << 31) - 1024);
}

// The eager calls of the 8-bit checkpoint: None as above.
py::object py_int8_pack(py::handle hx) {
  if (!plain_type(hx) || !plain_context()) return py::none();
  const Tensor& x = THPVariable_Unpack(hx.ptr());
  if (!plain_cuda(x) || !device_supported(x) || row_type(x) < 0 || x.dim() < 1 || !few_groups(x)) return py::none();
  std::vector<Tensor> r;
  {
    py::gil_scoped_release release;
    at::NoGradGuard no_grad;
    r = int8_pack(x.detach());
  }
  return py::make_tuple(r[0], r[1]);
}

py::object py_int8_unpack(py::handle hc, py::handle hs, py::object dtype) {
  if (!plain_type(hc) || !plain_type(hs) || !plain_context() || !THPDtype_Check(dtype.ptr())) return py::none();
  const Tensor &codes = THPVariable_Unpack(hc.ptr()), &scales = THPVariable_Unpack(hs.ptr());
  const auto type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  if (!plain_cuda(codes) || !plain_cuda(scales) || !device_supported(codes) || scales.device() != codes.device() ||
      codes.scalar_type() != at::kChar || scales.scalar_type() != at::kFloat || codes.dim() < 1 ||
      (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) || !few_groups(codes) ||
      scales.sizes().vec() != with_last(codes.sizes(), (codes.size(-1) + 127) / 128))
    return py::none();
  Tensor x;
  {
    py::gil_scoped_release release;
    at::NoGradGuard no_grad;
    x = int8_unpack(codes, scales, (int64_t)type);
  }
  return py::cast(x);
}

}  // namespace tpf_torch

// Dropout, the position rotation of heads and the window attention for eager CUDA tensors.
#include <cmath>
#include <limits>

#include "tpf_dropout.h"
#include "tpf_rotary.h"
#include "tpf_torch_memory.h"
#include "tpf_window.h"

namespace tpf_torch {

namespace {

bool aligned(const Tensor& t, int64_t bytes) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & (bytes - 1)) == 0; }

// A gradient as the kernels read it: contiguous, on a 16-byte boundary (32 in fp32).
Tensor dense(const Tensor& t) {
  Tensor c = t.contiguous();
  return aligned(c, 32) ? c : c.clone();
}

// A saved tensor that a kernel reads from its first element on.  (A hook of the caller's may have handed back other strides.)
Tensor in_order(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// An optional tensor argument: false if it needs the Python route.
bool unpack_optional(py::handle h, const Tensor& x, Tensor& out) {
  if (h.is_none()) return true;
  if (!plain_type(h)) return false;
  out = THPVariable_Unpack(h.ptr());
  return plain_cuda(out) && out.device() == x.device();
}

// ---- dropout ---------------------------------------------------------------------------------------------
struct DropoutArgs {
  Tensor seed_tensor;  // int64 [2], or undefined: the numbers
  int64_t seed, offset, threshold, shared;  // shared: a dimension, or -1
};

// Fills the sizes and strides of a call from dimensions that lie at one stride in x and the residual; false: a copy is needed.
bool dropout_layout(const Tensor& x, const Tensor& residual, int64_t shared, tpf::DropoutCall& c) {
  struct Dim {
    int64_t size, x, r, o;
    bool shared;
  };
  c10::SmallVector<Dim, 8> dims;
  int64_t out = 1;
  for (int64_t d = x.dim() - 1; d >= 0; --d) {  // from the last one
    const int64_t n = x.size(d);
    const Dim now{n, x.stride(d), residual.defined() ? residual.stride(d) : 0, out, d == shared};
    out *= n;
    if (n == 1) continue;
    if (!dims.empty() && !dims.back().shared && !now.shared && now.x == dims.back().x * dims.back().size &&
        (!residual.defined() || now.r == dims.back().r * dims.back().size))
      dims.back().size *= n;
    else
      dims.push_back(now);
  }
  size_t next = 0;
  int64_t inner = 1;
  if (!dims.empty() && !dims[0].shared && dims[0].x == 1 && (!residual.defined() || dims[0].r == 1)) inner = dims[next++].size;
  // (a shared dimension or a stride in the last place: elements on their own, in the caller's order, only where nothing else is left)
  else if (!dims.empty() && !dims[0].shared) return false;
  const Dim one{1, 0, 0, 0, false};
  Dim s = one, rest[3] = {one, one, one};
  int n = 0;
  for (; next < dims.size(); ++next) {
    if (dims[next].shared) s = dims[next];
    else if (n == 3) return false;
    else rest[n++] = dims[next];
  }
  if (n == 3) {  // no shared dimension: the third place is free
    if (s.size != 1 || rest[0].size > 65535) return false;
    s = rest[0];
    rest[0] = rest[1];
    rest[1] = rest[2];
  }
  constexpr int64_t kMostRows = 1ll << 31;
  if (rest[1].size >= kMostRows || rest[0].size >= kMostRows || rest[1].size * rest[0].size >= kMostRows) return false;
  const Dim order[3] = {rest[1], rest[0], s};  // p, q, s
  for (int i = 0; i < 3; ++i) {
    c.sizes[i] = order[i].size;
    c.x_strides[i] = order[i].x;
    c.residual_strides[i] = order[i].r;
    c.out_strides[i] = order[i].o;
  }
  c.sizes[3] = inner;
  c.shared = s.shared;  // (not where the shared dimension is a single element, whose place another one may have taken)
  return true;
}

Tensor dropout_out(const Tensor& x_in, const Tensor& residual_in, const DropoutArgs& a) {
  Tensor x = x_in, residual = residual_in;
  if (x.numel() == 0) return make(x.sizes(), x.scalar_type(), x);
  tpf::DropoutCall c = {};
  if (!dropout_layout(x, residual, a.shared, c)) {
    x = x.contiguous();
    if (residual.defined()) residual = residual.contiguous();
    TORCH_CHECK(dropout_layout(x, residual, a.shared, c), "turbo_dropout: a layout that a copy does not settle");
  }
  Tensor out = make(x.sizes(), x.scalar_type(), x);
  c.x = x.data_ptr();
  c.residual = ptr_of(residual);
  c.out = out.data_ptr();
  c.type = row_type(x);
  c.threshold = (int)a.threshold;
  c.seed_ptr = a.seed_tensor.defined() ? static_cast<const int64_t*>(a.seed_tensor.data_ptr()) : nullptr;
  c.seed = a.seed;
  c.offset = a.offset;
  check(tpf::dropout(c, cu_stream()), "tpf_dropout");
  return out;
}

struct DropoutFn : public torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& residual, const DropoutArgs& a) {
    ctx->save_for_backward({a.seed_tensor});
    ctx->saved_data["a"] = std::vector<int64_t>{a.seed, a.offset, a.threshold, a.shared, residual ? 1 : 0};
    return dropout_out(x.detach(), residual ? residual->detach() : Tensor(), a);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return first_order(grads, gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list r(3);
    if (!grads[0].defined()) return r;
    c10::cuda::CUDAGuard guard(grads[0].device());
    at::NoGradGuard no_grad;
    const std::vector<int64_t> v = ctx->saved_data["a"].toIntVector();
    const DropoutArgs a{in_order(ctx->get_saved_variables()[0]), v[0], v[1], v[2], v[3]};
    if (ctx->needs_input_grad(0)) r[0] = dropout_out(grads[0].detach(), Tensor(), a);
    // (the very tensor: a view of it would hide from whoever accumulates gradients that others hold it, too)
    if (v[4]) r[1] = grads[0];
    return r;
  }
};

// ---- rotation --------------------------------------------------------------------------------------------
struct RotaryArgs {
  Tensor turns, positions;  // int64; positions contiguous or undefined
  int64_t first;
  double magnitude;
  bool half, norm;
  double eps;
};

// A tensor [*, N, H, D] with its leading dimensions as one batch: read in place where its strides allow it, else a copy.
struct Heads {
  Tensor t;
  int64_t batch, strides[3];
};
Heads as_heads(const Tensor& t, bool tiles) {  // tiles: for TMA
  const int64_t nd = t.dim();
  Heads h{t, 1, {0, t.stride(nd - 3), t.stride(nd - 2)}};
  bool ok = t.stride(nd - 1) == 1 || t.size(nd - 1) == 1, first = true;
  int64_t next = 0;
  for (int64_t d = nd - 4; d >= 0; --d) {
    h.batch *= t.size(d);
    if (t.size(d) == 1) continue;
    if (first) h.strides[0] = t.stride(d);
    else ok = ok && t.stride(d) == next;
    first = false;
    next = t.stride(d) * t.size(d);
  }
  if (tiles && t.numel() > 0) {
    ok = ok && aligned(t, 16);
    const int64_t sizes[3] = {h.batch, t.size(nd - 3), t.size(nd - 2)};
    for (int i = 0; i < 3; ++i) ok = ok && (sizes[i] == 1 || (h.strides[i] > 0 && h.strides[i] % 8 == 0));
  }
  if (!ok) {
    h.t = t.is_contiguous() ? t.clone() : t.contiguous();
    if (tiles && !aligned(h.t, 16)) h.t = h.t.clone();
    h.strides[2] = t.size(nd - 1);
    h.strides[1] = t.size(nd - 2) * h.strides[2];
    h.strides[0] = t.size(nd - 3) * h.strides[1];
  }
  return h;
}

void rotary_common(tpf::RotaryCall& c, const RotaryArgs& a, const Tensor& like, int64_t batch) {
  const int64_t nd = like.dim();
  c.type = row_type(like);
  c.batch = batch;
  c.tokens = like.size(nd - 3);
  c.dim = like.size(nd - 1);
  c.rot = 2 * a.turns.numel();
  c.turns = static_cast<const int64_t*>(a.turns.data_ptr());
  c.magnitude = (float)a.magnitude;
  c.positions = a.positions.defined() ? static_cast<const int64_t*>(a.positions.data_ptr()) : nullptr;
  c.first = a.first;
  c.half = a.half;
  c.norm = a.norm;
  c.eps = (float)a.eps;
}

void set_source(tpf::RotaryTensor& t, const Heads& h) {
  t.x = h.t.data_ptr();
  for (int i = 0; i < 3; ++i) t.strides[i] = h.strides[i];
  t.heads = h.t.size(h.t.dim() - 2);
}

variable_list rotary_out(const Heads& q, const Heads& k, const Tensor& qw, const Tensor& kw, const RotaryArgs& a) {
  tpf::RotaryCall c = {};
  rotary_common(c, a, q.t, q.batch);
  variable_list out(2);
  const Heads* in[2] = {&q, &k};
  const Tensor* w[2] = {&qw, &kw};
  for (int i = 0; i < 2; ++i) {
    if (!in[i]->t.defined()) continue;
    out[i] = make(in[i]->t.sizes(), in[i]->t.scalar_type(), in[i]->t);
    set_source(c.t[i], *in[i]);
    c.t[i].weight = ptr_of(*w[i]);
    c.t[i].weight_type = type_of(*w[i]);
    c.t[i].out = out[i].data_ptr();
  }
  check(tpf::rotary_fwd(c, cu_stream()), "tpf_rotary_fwd");
  return out;
}

// d[i]: the gradient of output i, or undefined (nothing came).  x: the inputs (with a norm).
struct RotaryGrads {
  Tensor dx[2], dw[2];
};
RotaryGrads rotary_grads(const Tensor (&d)[2], const Heads (&x)[2], const Tensor (&w)[2], const bool (&need_w)[2],
                         const RotaryArgs& a) {
  RotaryGrads r;
  const Tensor& like = d[0].defined() ? d[0] : d[1];
  tpf::RotaryCall c = {};
  int64_t batch = 1;
  for (int64_t i = 0; i < like.dim() - 3; ++i) batch *= like.size(i);
  rotary_common(c, a, like, batch);
  bool any_w = false;
  for (int i = 0; i < 2; ++i) {
    if (need_w[i]) r.dw[i] = d[i].defined() ? make(w[i].sizes(), w[i].scalar_type(), w[i]) : at::zeros_like(w[i]);
    if (!d[i].defined()) continue;
    r.dx[i] = make(d[i].sizes(), d[i].scalar_type(), d[i]);
    if (a.norm) set_source(c.t[i], x[i]);
    c.t[i].heads = d[i].size(d[i].dim() - 2);
    c.t[i].weight = ptr_of(w[i]);
    c.t[i].weight_type = type_of(w[i]);
    c.t[i].dy = d[i].data_ptr();
    c.t[i].out = r.dx[i].data_ptr();
    if (need_w[i]) c.t[i].dweight = r.dw[i].data_ptr();
    any_w = any_w || need_w[i];
  }
  const int64_t n = any_w ? tpf_rotary_bwd_workspace_bytes(c.dim) : 0;
  const Scratch ws(n);
  check(tpf::rotary_bwd(c, ws.get(), n, cu_stream()), "tpf_rotary_bwd");
  return r;
}

Tensor param(const Tensor& w) { return w.defined() ? w.detach().contiguous() : Tensor(); }
Tensor kept(const Tensor& in, const Heads& h) { return h.t.data_ptr() == in.data_ptr() ? in : h.t; }

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const MaybeTensor& k, const MaybeTensor& qw,
                               const MaybeTensor& kw, const RotaryArgs& a) {
    const Heads hq = as_heads(q.detach(), false), hk = k ? as_heads(k->detach(), false) : Heads{};
    variable_list out = rotary_out(hq, hk, qw ? param(*qw) : Tensor(), kw ? param(*kw) : Tensor(), a);
    if (!k) out.resize(1);
    // (the inputs themselves where they were read in place, so that a change to them before the backward is noticed)
    ctx->save_for_backward({a.norm ? kept(q, hq) : Tensor(), a.norm && k ? kept(*k, hk) : Tensor(), qw ? *qw : Tensor(),
                            kw ? *kw : Tensor(), a.turns, a.positions});
    // (an entry costs a microsecond)
    ctx->saved_data["a"] = std::vector<double>{(double)(a.first >> 32), (double)(a.first & 0xffffffff), a.magnitude, (double)a.half,
                                               (double)a.norm, a.eps, (double)k.has_value()};
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return first_order(grads, gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list r(5);
    const std::vector<double> v = ctx->saved_data["a"].toDoubleVector();
    const bool has_k = v[6] != 0;
    const Tensor none;
    const Tensor& some = grads[0].defined() ? grads[0] : has_k ? grads[1] : none;
    if (!some.defined()) return r;
    c10::cuda::CUDAGuard guard(some.device());
    at::NoGradGuard no_grad;
    const auto saved = ctx->get_saved_variables();
    const RotaryArgs a{in_order(saved[4]), in_order(saved[5]), ((int64_t)v[0] << 32) + (int64_t)v[1], v[2], v[3] != 0, v[4] != 0,
                       v[5]};
    const Tensor d[2] = {grads[0].defined() ? dense(grads[0]) : none, has_k && grads[1].defined() ? dense(grads[1]) : none};
    const Heads x[2] = {saved[0].defined() ? as_heads(saved[0].detach(), false) : Heads{},
                        saved[1].defined() ? as_heads(saved[1].detach(), false) : Heads{}};
    const Tensor w[2] = {param(saved[2]), param(saved[3])};
    int edge = has_k ? 2 : 1;  // an absent tensor has no edge
    bool need_w[2] = {false, false};
    if (w[0].defined()) need_w[0] = ctx->needs_input_grad(edge++);
    if (w[1].defined()) need_w[1] = ctx->needs_input_grad(edge++);
    const RotaryGrads g = rotary_grads(d, x, w, need_w, a);
    r[0] = g.dx[0];
    r[1] = g.dx[1];
    r[2] = g.dw[0];
    r[3] = g.dw[1];
    return r;
  }
};

// ---- window attention ------------------------------------------------------------------------------------
struct WindowArgs {
  Tensor offsets, lengths;  // int32 [B], contiguous, or undefined
  int64_t offset, left, right, sinks;  // a negative reach: unlimited
  double scale;
};

tpf::WindowCall window_call(const Heads& q, const Heads& k, const Heads& v, const WindowArgs& a) {
  const int64_t nd = q.t.dim();
  tpf::WindowCall c = {};
  c.B = q.batch, c.N = q.t.size(nd - 3), c.H = q.t.size(nd - 2), c.D = q.t.size(nd - 1);
  c.M = k.t.size(nd - 3), c.HK = k.t.size(nd - 2);
  c.type = row_type(q.t);
  c.scale = (float)a.scale;
  c.left = a.left < 0 ? tpf::kWindowUnlimited : (int)a.left;
  c.right = a.right < 0 ? tpf::kWindowUnlimited : (int)a.right;
  c.sinks = (int)a.sinks;
  c.offsets = a.offsets.defined() ? static_cast<const int*>(a.offsets.data_ptr()) : nullptr;
  c.lengths = a.lengths.defined() ? static_cast<const int*>(a.lengths.data_ptr()) : nullptr;
  c.offset = a.offset;
  c.q = q.t.data_ptr(), c.k = k.t.data_ptr(), c.v = v.t.data_ptr();
  for (int i = 0; i < 3; ++i) c.qs[i] = q.strides[i], c.ks[i] = k.strides[i], c.vs[i] = v.strides[i];
  return c;
}

std::vector<int64_t> lse_sizes(const Tensor& q) {  // [*, H, N]
  std::vector<int64_t> s(q.sizes().begin(), q.sizes().end() - 1);
  std::swap(s[s.size() - 1], s[s.size() - 2]);
  return s;
}

std::pair<Tensor, Tensor> window_out(const Heads& q, const Heads& k, const Heads& v, const WindowArgs& a, bool want_lse) {
  tpf::WindowCall c = window_call(q, k, v, a);
  Tensor out = make(q.t.sizes(), q.t.scalar_type(), q.t), lse;
  if (want_lse) lse = make(lse_sizes(q.t), at::kFloat, q.t);
  c.out = out.data_ptr();
  c.lse = fptr(lse);
  check(tpf::window_attn_fwd(c, cu_stream()), "tpf_window_attn_fwd");
  return {out, lse};
}

variable_list window_grads(const Tensor& d_out, const Heads& q, const Heads& k, const Heads& v, const Tensor& out, const Tensor& lse,
                           const WindowArgs& a, bool need_q, bool need_kv) {
  tpf::WindowCall c = window_call(q, k, v, a);
  variable_list r(3);
  if (need_q) r[0] = make(q.t.sizes(), q.t.scalar_type(), q.t);
  if (need_kv) {
    r[1] = make(k.t.sizes(), k.t.scalar_type(), k.t);
    r[2] = make(v.t.sizes(), v.t.scalar_type(), v.t);
  }
  c.d_out = d_out.data_ptr();
  c.out = out.data_ptr();
  c.lse = fptr(lse);
  c.dq = ptr_of(r[0]), c.dk = ptr_of(r[1]), c.dv = ptr_of(r[2]);
  const int64_t n = tpf::window_attn_bwd_workspace_bytes(c);
  const Scratch ws(n);
  check(tpf::window_attn_bwd(c, ws.get(), n, cu_stream()), "tpf_window_attn_bwd");
  return r;
}

struct WindowFn : public torch::autograd::Function<WindowFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const WindowArgs& a) {
    const Heads hq = as_heads(q.detach(), true), hk = as_heads(k.detach(), true), hv = as_heads(v.detach(), true);
    auto [out, lse] = window_out(hq, hk, hv, a, true);
    ctx->save_for_backward({kept(q, hq), kept(k, hk), kept(v, hv), out, lse, a.offsets, a.lengths});
    ctx->saved_data["a"] = std::vector<double>{(double)a.offset, (double)a.left, (double)a.right, (double)a.sinks, a.scale};
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return first_order(grads, gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    variable_list r(4);
    if (!grads[0].defined()) return r;
    c10::cuda::CUDAGuard guard(grads[0].device());
    at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const std::vector<double> v = ctx->saved_data["a"].toDoubleVector();  // (whole numbers below 2^53 are exact)
    const WindowArgs a{in_order(s[5]), in_order(s[6]), (int64_t)v[0], (int64_t)v[1], (int64_t)v[2], (int64_t)v[3], v[4]};
    const bool need_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const variable_list g = window_grads(dense(grads[0]), as_heads(s[0].detach(), true), as_heads(s[1].detach(), true),
                                         as_heads(s[2].detach(), true), dense(s[3]), s[4].contiguous(), a, ctx->needs_input_grad(0),
                                         need_kv);
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) r[i] = g[i];
    return r;
  }
};

bool heads_ok(const Tensor& t, const Tensor& like) {
  return plain_cuda(t) && t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.dim() == like.dim();
}
bool same_but(const Tensor& a, const Tensor& b, int64_t dim) {  // the same sizes but for one dimension, counted from the end
  for (int64_t d = 0; d < a.dim(); ++d)
    if (d != a.dim() - dim && a.size(d) != b.size(d)) return false;
  return true;
}
bool weight_ok(const Tensor& w, const Tensor& x) { return !w.defined() || (row_type(w) >= 0 && w.dim() == 1 && w.size(0) == x.size(-1)); }

}  // namespace

// The eager calls return None when the arguments need the Python route: an unsupported case (which raises there, with its
// reason), a tensor subclass, an active dispatch mode.
py::object py_dropout(py::handle hx, py::handle hr, py::handle hs, int64_t seed, int64_t offset, int64_t threshold, int64_t shared) {
  if (!plain_type(hx) || !plain_context()) return py::none();
  const Tensor& x = THPVariable_Unpack(hx.ptr());
  if (!plain_cuda(x) || !device_supported(x) || row_type(x) < 0 || x.dim() < 1) return py::none();
  Tensor r, s;
  if (!unpack_optional(hr, x, r) || !unpack_optional(hs, x, s)) return py::none();
  if (r.defined() && (r.scalar_type() != x.scalar_type() || r.sizes() != x.sizes())) return py::none();
  if (s.defined() && (s.scalar_type() != at::kLong || s.dim() != 1 || s.size(0) != 2 || !s.is_contiguous())) return py::none();
  if (x.numel() >= 1ll << 36) return py::none();
  if (shared >= 0) {
    constexpr int64_t kMost = 1ll << 31;
    if (shared >= x.dim() - 1 || x.size(shared) >= kMost || c10::multiply_integers(x.sizes().slice(0, shared)) >= kMost) return py::none();
  }
  const DropoutArgs a{s, seed, offset, threshold, shared};
  Tensor out;
  {
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(x.device());
    if (at::GradMode::is_enabled() && (x.requires_grad() || (r.defined() && r.requires_grad()))) {
      out = DropoutFn::apply(x, maybe(r), a);
    } else {
      at::NoGradGuard no_grad;
      out = dropout_out(x, r, a);
    }
  }
  return py::cast(out);
}

py::object py_rotary(py::handle hq, py::handle hk, py::handle hqw, py::handle hkw, py::handle ht, py::handle hp, int64_t first,
                     double magnitude, bool half, bool norm, double eps) {
  if (!plain_type(hq) || !plain_type(ht) || !plain_context()) return py::none();
  const Tensor &q = THPVariable_Unpack(hq.ptr()), &turns = THPVariable_Unpack(ht.ptr());
  if (!plain_cuda(q) || !device_supported(q) || row_type(q) < 0 || q.dim() < 3) return py::none();
  Tensor k, qw, kw, pos;
  if (!unpack_optional(hk, q, k) || !unpack_optional(hqw, q, qw) || !unpack_optional(hkw, q, kw) || !unpack_optional(hp, q, pos))
    return py::none();
  const int64_t D = q.size(-1);
  if (k.defined() && (!heads_ok(k, q) || !same_but(k, q, 2))) return py::none();
  if (!weight_ok(qw, q) || !weight_ok(kw, q) || D < 2 || D > 256 || !(eps >= 0) ||
      !(std::abs(magnitude) <= std::numeric_limits<float>::max()))
    return py::none();
  if (!plain_cuda(turns) || turns.device() != q.device() || turns.scalar_type() != at::kLong || turns.dim() != 1 ||
      !turns.is_contiguous() || turns.size(0) < 1 || 2 * turns.size(0) > D)
    return py::none();
  if (pos.defined() && (pos.scalar_type() != at::kLong || !pos.is_contiguous() || pos.sizes() != q.sizes().slice(0, q.dim() - 2)))
    return py::none();
  constexpr int64_t kMostRows = (1ll << 31) - 256;
  if (q.numel() / D > kMostRows || (k.defined() && k.numel() / D > kMostRows)) return py::none();
  if (q.size(-2) + (k.defined() ? k.size(-2) : 0) >= 1 << 24) return py::none();
  const RotaryArgs a{turns, pos, first, magnitude, half, norm, eps};
  auto wants = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
  variable_list out;
  {
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(q.device());
    if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(qw) || wants(kw))) {
      out = RotaryFn::apply(q, maybe(k), maybe(qw), maybe(kw), a);
    } else {
      at::NoGradGuard no_grad;
      out = rotary_out(as_heads(q, false), k.defined() ? as_heads(k, false) : Heads{}, param(qw), param(kw), a);
    }
  }
  if (!k.defined()) return py::cast(out[0]);
  return py::make_tuple(out[0], out[1]);
}

py::object py_window_attention(py::handle hq, py::handle hk, py::handle hv, py::handle window, py::handle hsinks, py::handle ho,
                               py::handle hl, py::handle hscale, bool return_lse) {
  if (!plain_type(hq) || !plain_type(hk) || !plain_type(hv) || !plain_context()) return py::none();
  auto number = [](py::handle h, int64_t lo, int64_t hi, int64_t* out) {
    if (!PyLong_CheckExact(h.ptr())) return false;
    int overflow = 0;
    *out = PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
    return overflow == 0 && *out >= lo && *out <= hi;
  };
  if (!PyTuple_CheckExact(window.ptr()) || PyTuple_GET_SIZE(window.ptr()) != 2) return py::none();
  int64_t reach[2] = {-1, -1}, sinks = 0, offset = 0;
  for (int i = 0; i < 2; ++i) {
    const py::handle n = PyTuple_GET_ITEM(window.ptr(), i);
    if (!n.is_none() && !number(n, 0, tpf::kWindowMost - 1, &reach[i])) return py::none();
  }
  if (!number(hsinks, 0, tpf::kMostSinks, &sinks)) return py::none();
  const bool offset_is_number = number(ho, -tpf::kWindowMost, tpf::kWindowMost, &offset);
  if (!offset_is_number) offset = 0;
  const Tensor &q = THPVariable_Unpack(hq.ptr()), &k = THPVariable_Unpack(hk.ptr()), &v = THPVariable_Unpack(hv.ptr());
  if (!plain_cuda(q) || !device_supported(q) || (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) || q.dim() < 3)
    return py::none();
  if (!heads_ok(k, q) || !heads_ok(v, q) || k.sizes() != v.sizes()) return py::none();
  const int64_t nd = q.dim(), D = q.size(nd - 1), H = q.size(nd - 2), HK = k.size(nd - 2);
  if (D != k.size(nd - 1) || D < 8 || D > 128 || D % 8 || HK < 1 || H < 1 || H % HK) return py::none();
  int64_t batch = 1;
  for (int64_t d = 0; d < nd - 3; ++d) {
    if (q.size(d) != k.size(d)) return py::none();
    batch *= q.size(d);
  }
  if (batch > 65535 || H > 65535 || q.size(nd - 3) > tpf::kWindowMost || k.size(nd - 3) > tpf::kWindowMost) return py::none();
  double scale = 1.0 / std::sqrt((double)D);
  if (!hscale.is_none()) {
    if (!PyFloat_CheckExact(hscale.ptr())) return py::none();
    scale = PyFloat_AS_DOUBLE(hscale.ptr());
    if (!(scale >= 0x1p-100 && scale <= 0x1p100)) return py::none();
  }
  Tensor offsets, lengths;
  if (!offset_is_number && (ho.is_none() || !THPVariable_Check(ho.ptr()) || !unpack_optional(ho, q, offsets))) return py::none();
  if (!hl.is_none() && (!THPVariable_Check(hl.ptr()) || !unpack_optional(hl, q, lengths))) return py::none();
  for (const Tensor* t : {&offsets, &lengths})
    if (t->defined() && (t->scalar_type() != at::kInt || !t->is_contiguous() || t->sizes() != q.sizes().slice(0, nd - 3)))
      return py::none();
  const WindowArgs a{offsets, lengths, offset, reach[0], reach[1], sinks, scale};
  Tensor out, lse;
  {
    py::gil_scoped_release release;
    c10::cuda::CUDAGuard guard(q.device());
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      const variable_list r = WindowFn::apply(q, k, v, a);
      out = r[0];
      lse = r[1];
    } else {
      at::NoGradGuard no_grad;
      std::tie(out, lse) = window_out(as_heads(q, true), as_heads(k, true), as_heads(v, true), a, return_lse);
    }
  }
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

// Launches behind the torch.library operators, which have checked the arguments.  Absent tensors of an output list are empty.
Tensor dropout_op(const Tensor& x, const MaybeTensor& residual, const MaybeTensor& seed_tensor, int64_t seed, int64_t offset,
                  int64_t threshold, int64_t shared) {
  c10::cuda::CUDAGuard guard(x.device());
  return dropout_out(x, residual ? *residual : Tensor(), {seed_tensor ? seed_tensor->contiguous() : Tensor(), seed, offset, threshold,
                                                          shared});
}

std::vector<Tensor> rotary_fwd_op(const Tensor& q, const MaybeTensor& k, const MaybeTensor& qw, const MaybeTensor& kw,
                                  const Tensor& turns, const MaybeTensor& positions, int64_t first, double magnitude, bool half,
                                  bool norm, double eps) {
  c10::cuda::CUDAGuard guard(q.device());
  const RotaryArgs a{turns.contiguous(), positions ? positions->contiguous() : Tensor(), first, magnitude, half, norm, eps};
  variable_list r = rotary_out(as_heads(q, false), k ? as_heads(*k, false) : Heads{}, qw ? param(*qw) : Tensor(),
                               kw ? param(*kw) : Tensor(), a);
  if (!r[1].defined()) r[1] = at::empty({0}, q.options());
  return r;
}

std::vector<Tensor> rotary_bwd_op(const MaybeTensor& dq, const MaybeTensor& dk, const MaybeTensor& q, const MaybeTensor& k,
                                  const MaybeTensor& qw, const MaybeTensor& kw, const Tensor& turns, const MaybeTensor& positions,
                                  int64_t first, double magnitude, bool half, bool norm, double eps) {
  const Tensor& some = dq ? *dq : *dk;
  c10::cuda::CUDAGuard guard(some.device());
  const RotaryArgs a{turns.contiguous(), positions ? positions->contiguous() : Tensor(), first, magnitude, half, norm, eps};
  const Tensor d[2] = {dq ? dense(*dq) : Tensor(), dk ? dense(*dk) : Tensor()};
  const Heads x[2] = {q && dq ? as_heads(*q, false) : Heads{}, k && dk ? as_heads(*k, false) : Heads{}};
  const Tensor w[2] = {qw ? param(*qw) : Tensor(), kw ? param(*kw) : Tensor()};
  RotaryGrads g = rotary_grads(d, x, w, {w[0].defined(), w[1].defined()}, a);
  auto some_or_empty = [&](const Tensor& t, const Tensor& like) { return t.defined() ? t : at::empty({0}, like.options()); };
  const Tensor f32 = empty_f32({0}, some);
  return {some_or_empty(g.dx[0], some), some_or_empty(g.dx[1], some), some_or_empty(g.dw[0], f32), some_or_empty(g.dw[1], f32)};
}

std::tuple<Tensor, Tensor> window_fwd_op(const Tensor& q, const Tensor& k, const Tensor& v, const MaybeTensor& offsets,
                                         const MaybeTensor& lengths, int64_t offset, int64_t left, int64_t right, int64_t sinks,
                                         double scale) {
  c10::cuda::CUDAGuard guard(q.device());
  const WindowArgs a{offsets ? offsets->contiguous() : Tensor(), lengths ? lengths->contiguous() : Tensor(), offset, left, right, sinks,
                     scale};
  auto [out, lse] = window_out(as_heads(q, true), as_heads(k, true), as_heads(v, true), a, true);
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor> window_bwd_op(const Tensor& d_out, const Tensor& q, const Tensor& k, const Tensor& v,
                                                 const Tensor& out, const Tensor& lse, const MaybeTensor& offsets,
                                                 const MaybeTensor& lengths, int64_t offset, int64_t left, int64_t right,
                                                 int64_t sinks, double scale) {
  c10::cuda::CUDAGuard guard(q.device());
  const WindowArgs a{offsets ? offsets->contiguous() : Tensor(), lengths ? lengths->contiguous() : Tensor(), offset, left, right, sinks,
                     scale};
  const variable_list g = window_grads(dense(d_out), as_heads(q, true), as_heads(k, true), as_heads(v, true), dense(out),
                                       lse.contiguous(), a, true, true);
  return {g[0], g[1], g[2]};
}

}  // namespace tpf_torch

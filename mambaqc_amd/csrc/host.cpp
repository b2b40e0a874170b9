// The host side of the recurrent stack's operators, as a Python module over torch's C++ API: output and
// workspace allocation, the calls into libmambaqc_hip.so, the autograd nodes, and the AdamW step's
// tables. Nothing is computed here. It exists for its host time: what a training step of one small
// layer waits for is the path from the Python call to the launch (forward and backward of a gate with
// norms over 3001 x 515, whose kernels take 25 us: 87 us through Python nodes), and a table of 40
// tensors with 8-bit states took 130 us to check and fill. The decode steps are host time alone: with
// their arguments checked here too, and weights taken without a call into Python where they are what
// the kernels read, 5.0 and 7.2 us a call against 7.0 and 10.2.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/mambaqc_hip_ext.h"

namespace {

using at::Tensor;
using MaybeTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MQC_F32;
    case at::kBFloat16: return MQC_BF16;
    case at::kHalf: return MQC_F16;
    default:
      TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(),
                       "; expected float32, bfloat16 or float16");
  }
}
void check(int64_t status, const char* name) {
  TORCH_CHECK(status == MQC_OK, name, " failed with status ", status, ": ",
              mqc_status_string((int)status));
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const MaybeTensor& t) { return t ? t->data_ptr() : nullptr; }
const float* f32(const MaybeTensor& t) { return t ? (const float*)t->data_ptr() : nullptr; }
Tensor workspace(int64_t bytes, const char* name, const Tensor& like) {
  if (bytes < 0) check(bytes, name);
  return at::empty({bytes}, like.options().dtype(at::kByte));
}
Tensor like_f32(at::IntArrayRef sizes, const Tensor& like) {
  return at::empty(sizes, like.options().dtype(at::kFloat));
}
void on_device(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda(), "mambaqc_amd.", name, ": expected tensors on a ROCm device, got ", t.device(),
              "; this package runs only on the GPU");
  TORCH_CHECK(t.device() == like.device(), "mambaqc_amd.", name, ": tensors on different devices (",
              like.device(), ", ", t.device(), ")");
}
// Forward-mode gradients would be lost without a word: the kernels see values alone.
bool tangent(const Tensor& t) { return t._fw_grad(0).defined(); }
bool tangent(const MaybeTensor& t) { return t && tangent(*t); }
template <typename... Inputs>
void no_tangents(const char* name, const Inputs&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(tangent(inputs) || ...), name,
                              ": forward-mode automatic differentiation is not supported");
}
// Autograd does not see what the operands go through; their gradients' edges are the node's. (Views that
// torch negates as it reads them, such as the imaginary part of a conjugate, are made what they stand for.)
Tensor as_type(const Tensor& t, at::ScalarType type) {
  const at::NoGradGuard none;
  Tensor v = t.requires_grad() ? t.detach() : t;
  if (v.is_neg()) v = v.resolve_neg();
  return v.scalar_type() == type ? v : v.to(type);
}
// A parameter as the kernels read it: itself, or `convert`'s (_native.param_f32) where it is not that;
// without one (in a backward, which runs without Python's lock) a copy.
Tensor weight(const Tensor& t, const py::object* convert) {
  if (t.scalar_type() == at::kFloat && t.is_contiguous() && (uintptr_t)t.data_ptr() % 16 == 0)
    return as_type(t, at::kFloat);
  return convert ? (*convert)(t).cast<Tensor>() : as_type(t, at::kFloat).contiguous();
}
// What a kernel reads beside the operands, dense in `type`, where it has these sizes.
Tensor beside(const char* name, const char* what, const Tensor& t, at::IntArrayRef sizes,
              at::ScalarType type, const Tensor& like) {
  no_tangents(name, t);
  on_device(name, t, like);
  TORCH_CHECK_VALUE(t.sizes() == sizes, name, ": ", what, " must be ", sizes, ", got ", t.sizes());
  return as_type(t, type).contiguous();
}
bool records(std::initializer_list<MaybeTensor> inputs) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : inputs)
    if (t && t->requires_grad()) return true;
  return false;
}
// The kernels write through pointers: tells autograd (and whatever keeps copies of parameters by their
// version) that a tensor changed.
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Variable edge(const MaybeTensor& t) { return t ? *t : Variable(); }
MaybeTensor maybe(const Variable& v) { return v.defined() ? MaybeTensor(v) : std::nullopt; }
// The types that gradients are wanted in, -1 for none.
std::vector<int64_t> grad_types(std::initializer_list<MaybeTensor> inputs) {
  std::vector<int64_t> types;
  for (const auto& t : inputs) types.push_back(t && t->requires_grad() ? (int64_t)t->scalar_type() : -1);
  return types;
}
// The gradients of a node's inputs, of which the first ones are tensors.
variable_list as_grads(const std::vector<MaybeTensor>& grads, const std::vector<int64_t>& types,
                       size_t inputs) {
  variable_list out;
  for (size_t i = 0; i < grads.size(); ++i)
    out.push_back(grads[i] && types[i] >= 0 ? grads[i]->to((at::ScalarType)types[i]) : Variable());
  out.resize(inputs);
  return out;
}
// The kernels' gradients are not differentiable: a second backward through them raises.
variable_list once(const char* name, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  const std::string message = std::string(name) + ": a gradient of the gradient is not supported";
  for (auto& g : grads)
    if (g.defined()) {
      const auto node = std::make_shared<torch::autograd::DelayedError>(message, 1);
      g = (*node)({g.detach().requires_grad_()})[0];
    }
  return grads;
}

// --- gate, norms and residual ---------------------------------------------------------------------
// z in `type` and the elements between its rows, read in place where these are evenly spaced and the
// last axis is dense (the gate half of a projection's output).
std::pair<Tensor, int64_t> spaced_rows(const Tensor& t, at::ScalarType type) {
  const Tensor z = as_type(t, type);
  const int64_t d = z.size(-1);
  int64_t row = -1, want = 0;
  for (int64_t i = z.dim() - 2; i >= 0; --i) {
    const int64_t n = z.size(i), s = z.stride(i);
    if (n == 1) continue;
    if (row < 0) row = s;
    else if (s != want) row = 0;
    if (row == 0) break;
    want = s * n;
  }
  if (row < 0) row = d;
  if ((d > 1 && z.stride(-1) != 1) || row < d) return {z.contiguous(), d};
  return {z, row};
}

// Operands as the kernels read them: in the promoted type, weights in fp32 (kernels/gate_norm.py).
struct GateNorm {
  Tensor x, y;
  MaybeTensor z;
  int64_t z_row;
  MaybeTensor post;
  Tensor scale, pre;
  GateNorm(const Tensor& x_, const Tensor& y_, const MaybeTensor& z_, const MaybeTensor& post_,
           const Tensor& scale_, const Tensor& pre_, const py::object* convert)
      : z_row(0) {
    no_tangents("gate_norm_residual", x_, y_, z_, post_, scale_, pre_);
    for (const Tensor* t : {&x_, &y_, &scale_, &pre_}) on_device("gate_norm_residual", *t, x_);
    if (post_) on_device("gate_norm_residual", *post_, x_), post = weight(*post_, convert);
    scale = weight(scale_, convert), pre = weight(pre_, convert);
    auto type = at::promote_types(x_.scalar_type(), y_.scalar_type());
    if (z_) type = at::promote_types(type, z_->scalar_type());
    x = as_type(x_, type).contiguous();
    y = as_type(y_, type).contiguous();
    if (z_) {
      on_device("gate_norm_residual", *z_, x_);
      std::tie(z, z_row) = spaced_rows(*z_, type);
    }
  }
  int64_t d() const { return x.size(-1); }
  int64_t rows() const { return d() ? x.numel() / d() : 0; }
};

std::tuple<Tensor, Tensor, MaybeTensor> gate_norm_forward(const GateNorm& o, double eps, bool train) {
  const c10::DeviceGuard guard(o.x.device());
  Tensor out = at::empty_like(o.x), n = at::empty_like(o.x);
  MaybeTensor stats;
  if (train) stats = like_f32({o.rows(), 2}, o.x);
  if (o.rows() > 0)
    check(mqc_gate_norm_fwd(o.x.data_ptr(), o.y.data_ptr(), ptr(o.z), o.z_row, f32(o.post), f32(o.scale),
                            f32(o.pre), out.data_ptr(), n.data_ptr(), (float*)ptr(stats), o.rows(),
                            o.d(), (float)eps, dtype_code(o.x), stream_of(o.x)),
          "mqc_gate_norm_fwd");
  return {out, n, stats};
}

// dx, dy, dz, dpost, dscale, dpre.
std::vector<MaybeTensor> gate_norm_backward(const GateNorm& o, Tensor stats, MaybeTensor dout,
                                            MaybeTensor dn) {
  const c10::DeviceGuard guard(o.x.device());
  const auto grad = [&](const char* what, const Tensor& t) {
    return beside("gate_norm_residual", what, t, o.x.sizes(), o.x.scalar_type(), o.x);
  };
  stats = beside("gate_norm_residual", "the rows' inverse norms", stats, {o.rows(), 2}, at::kFloat, o.x);
  if (dout) dout = grad("the gradient of out", *dout);
  if (dn) dn = grad("the gradient of n", *dn);
  Tensor dx = at::empty_like(o.x), dy = at::empty_like(o.x);
  MaybeTensor dz, dpost;
  if (o.z) dz = at::empty_like(o.x);
  if (o.rows() == 0) {
    if (o.post) dpost = at::zeros_like(*o.post);
    return {dx, dy, dz, dpost, at::zeros_like(o.scale), at::zeros_like(o.pre)};
  }
  Tensor dscale = at::empty_like(o.scale), dpre = at::empty_like(o.pre);
  if (o.post) dpost = at::empty_like(*o.post);
  const int64_t bytes = mqc_gate_norm_workspace_bytes(o.rows(), o.d());
  const Tensor ws = workspace(bytes, "mqc_gate_norm_bwd", o.x);
  check(mqc_gate_norm_bwd(o.x.data_ptr(), o.y.data_ptr(), ptr(o.z), o.z_row, f32(o.post), f32(o.scale),
                          f32(o.pre), f32(stats), ptr(dout), ptr(dn), dx.data_ptr(), dy.data_ptr(),
                          ptr(dz), (float*)ptr(dpost), (float*)dscale.data_ptr(),
                          (float*)dpre.data_ptr(), o.rows(), o.d(), dtype_code(o.x), ws.data_ptr(),
                          bytes, stream_of(o.x)),
        "mqc_gate_norm_bwd");
  return {dx, dy, dz, dpost, dscale, dpre};
}

bool gate_norm_shapes(const Tensor& x, const Tensor& y, const MaybeTensor& z, const MaybeTensor& post,
                      const Tensor& scale, const Tensor& pre) {
  if (x.dim() < 1 || y.sizes() != x.sizes() || (z && z->sizes() != x.sizes())) return false;
  const at::IntArrayRef last = x.sizes().slice(x.dim() - 1);
  return scale.sizes() == last && pre.sizes() == last && (!post || post->sizes() == last);
}

struct GateNormNode : torch::autograd::Function<GateNormNode> {
  // The first six are what gradients go to; `o` is read.
  static variable_list forward(AutogradContext* ctx, const Variable& x, const Variable& y,
                               const MaybeTensor& z, const MaybeTensor& post, const Variable& scale,
                               const Variable& pre, const GateNorm& o, double eps) {
    auto [out, n, stats] = gate_norm_forward(o, eps, true);
    ctx->save_for_backward({o.x, o.y, edge(o.z), edge(o.post), o.scale, o.pre, *stats});
    ctx->set_materialize_grads(false);
    ctx->saved_data["types"] = grad_types({x, y, z, post, scale, pre});
    return {out, n};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (what hooks on saved tensors give back may be laid out in other ways than what was saved)
    const auto s = ctx->get_saved_variables();
    TORCH_CHECK_VALUE(gate_norm_shapes(s[0], s[1], maybe(s[2]), maybe(s[3]), s[4], s[5]),
                      "gate_norm_residual: the saved tensors came back in other shapes");
    const GateNorm o(s[0], s[1], maybe(s[2]), maybe(s[3]), s[4], s[5], nullptr);
    const auto got = gate_norm_backward(o, s[6], maybe(grads[0]), maybe(grads[1]));
    return once("gate_norm_residual", as_grads(got, ctx->saved_data["types"].toIntVector(), 8));
  }
};

// gate_norm_residual (out, n), or nothing where the shapes do not match.
std::optional<std::tuple<Tensor, Tensor>> gate_norm(const Tensor& x, const Tensor& y, const MaybeTensor& z,
                                                    const MaybeTensor& post, const Tensor& scale,
                                                    const Tensor& pre, double eps,
                                                    const py::object& convert) {
  if (!gate_norm_shapes(x, y, z, post, scale, pre)) return std::nullopt;
  const GateNorm o(x, y, z, post, scale, pre, &convert);
  if (records({x, y, z, post, scale, pre})) {
    const auto out = GateNormNode::apply(x, y, z, post, scale, pre, o, eps);
    return std::make_tuple(out[0], out[1]);
  }
  auto [out, n, stats] = gate_norm_forward(o, eps, false);
  return std::make_tuple(out, n);
}

// --- layer norm -----------------------------------------------------------------------------------
// Operands as the kernels read them, weights in fp32 (kernels/norm.py).
struct LayerNorm {
  Tensor x;
  int64_t x_row;
  MaybeTensor w, b;
  LayerNorm(const Tensor& x_, const MaybeTensor& w_, const MaybeTensor& b_, const py::object* convert) {
    no_tangents("layer_norm", x_, w_, b_);
    on_device("layer_norm", x_, x_);
    if (w_) on_device("layer_norm", *w_, x_), w = weight(*w_, convert);
    if (b_) on_device("layer_norm", *b_, x_), b = weight(*b_, convert);
    std::tie(x, x_row) = spaced_rows(x_, x_.scalar_type());
    dtype_code(x);
  }
  int64_t d() const { return x.size(-1); }
  int64_t rows() const { return d() ? x.numel() / d() : 0; }
};

std::tuple<Tensor, MaybeTensor> layer_norm_forward(const LayerNorm& o, double eps, bool train) {
  const c10::DeviceGuard guard(o.x.device());
  Tensor y = at::empty(o.x.sizes(), o.x.options());
  MaybeTensor stats;
  if (train) stats = like_f32({o.rows(), 2}, o.x);
  if (o.rows() > 0)
    check(mqc_layer_norm_fwd(o.x.data_ptr(), o.x_row, f32(o.w), f32(o.b), y.data_ptr(),
                             (float*)ptr(stats), o.rows(), o.d(), (float)eps, dtype_code(o.x),
                             stream_of(o.x)),
          "mqc_layer_norm_fwd");
  return {y, stats};
}

// dx, dweight, dbias (without their tensors nothing).
std::vector<MaybeTensor> layer_norm_backward(const LayerNorm& o, Tensor stats, Tensor dy) {
  const c10::DeviceGuard guard(o.x.device());
  stats = beside("layer_norm", "the rows' means and inverse roots", stats, {o.rows(), 2}, at::kFloat, o.x);
  dy = beside("layer_norm", "the gradient of y", dy, o.x.sizes(), o.x.scalar_type(), o.x);
  Tensor dx = at::empty(o.x.sizes(), o.x.options());
  MaybeTensor dw, db;
  if (o.rows() == 0) {
    if (o.w) dw = at::zeros_like(*o.w);
    if (o.b) db = at::zeros_like(*o.b);
    return {dx, dw, db};
  }
  if (o.w) dw = at::empty_like(*o.w);
  if (o.b) db = at::empty_like(*o.b);
  const int64_t bytes = dw || db ? mqc_layer_norm_workspace_bytes(o.rows(), o.d()) : 0;
  const Tensor ws = workspace(bytes, "mqc_layer_norm_bwd", o.x);
  check(mqc_layer_norm_bwd(o.x.data_ptr(), o.x_row, f32(o.w), f32(stats), dy.data_ptr(), dx.data_ptr(),
                           (float*)ptr(dw), (float*)ptr(db), o.rows(), o.d(), dtype_code(o.x),
                           ws.data_ptr(), bytes, stream_of(o.x)),
        "mqc_layer_norm_bwd");
  return {dx, dw, db};
}

bool layer_norm_shapes(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b) {
  if (x.dim() < 1) return false;
  const at::IntArrayRef last = x.sizes().slice(x.dim() - 1);
  return (!w || w->sizes() == last) && (!b || b->sizes() == last);
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static variable_list forward(AutogradContext* ctx, const Variable& x, const MaybeTensor& w,
                               const MaybeTensor& b, const LayerNorm& o, double eps) {
    auto [y, stats] = layer_norm_forward(o, eps, true);
    ctx->save_for_backward({o.x, edge(o.w), edge(o.b), *stats});
    ctx->saved_data["types"] = grad_types({x, w, b});
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (laid out anew, as in GateNormNode)
    const auto s = ctx->get_saved_variables();
    TORCH_CHECK_VALUE(layer_norm_shapes(s[0], maybe(s[1]), maybe(s[2])),
                      "layer_norm: the saved tensors came back in other shapes");
    const LayerNorm o(s[0], maybe(s[1]), maybe(s[2]), nullptr);
    const auto got = layer_norm_backward(o, s[3], grads[0]);
    return once("layer_norm", as_grads(got, ctx->saved_data["types"].toIntVector(), 5));
  }
};

// layer_norm, or nothing where the shapes do not match.
MaybeTensor layer_norm(const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, double eps,
                       const py::object& convert) {
  if (!layer_norm_shapes(x, w, b)) return std::nullopt;
  const LayerNorm o(x, w, b, &convert);
  if (records({x, w, b})) return LayerNormNode::apply(x, w, b, o, eps)[0];
  return std::get<0>(layer_norm_forward(o, eps, false));
}

// --- the gated scan -------------------------------------------------------------------------------
// t [b, n, d] in `type` and the elements between its tokens, read in place where these are evenly
// spaced and the last axis is dense.
std::pair<Tensor, int64_t> token_rows(const Tensor& t, at::ScalarType type) {
  const Tensor v = as_type(t, type);
  const int64_t b = v.size(0), n = v.size(1), d = v.size(2);
  const int64_t row = n > 1 ? v.stride(1) : v.stride(0);
  if ((d > 1 && v.stride(2) != 1) || (b > 1 && n > 1 && v.stride(0) != n * v.stride(1)) ||
      (b * n > 1 && row < d))
    return {v.contiguous(), d};
  return {v, b * n <= 1 ? d : row};
}

// Operands as the kernels read them: tokens in the promoted type, rates in fp32 (kernels/gated.py).
struct Scan {
  Tensor dt;
  int64_t dt_row;
  Tensor g;
  int64_t g_row;
  Tensor x;
  int64_t x_row;
  Tensor rate;
  MaybeTensor reset;
  // (the state h is only looked at)
  Scan(const char* name, const Tensor& dt_, const Tensor& g_, const Tensor& x_, const Tensor& rate_,
       const MaybeTensor& reset_, const MaybeTensor& h, const py::object* convert) {
    no_tangents(name, dt_, g_, x_, rate_, h);
    for (const Tensor* t : {&x_, &dt_, &g_, &rate_}) on_device(name, *t, x_);
    if (h) on_device(name, *h, x_);
    rate = weight(rate_, convert);
    if (reset_) on_device(name, *reset_, x_), reset = reset_->contiguous();
    const auto type =
        at::promote_types(at::promote_types(dt_.scalar_type(), g_.scalar_type()), x_.scalar_type());
    std::tie(dt, dt_row) = token_rows(dt_, type);
    std::tie(g, g_row) = token_rows(g_, type);
    std::tie(x, x_row) = token_rows(x_, type);
  }
  int64_t b() const { return x.size(0); }
  int64_t t() const { return x.size(1); }
  int64_t d() const { return x.size(2); }
};

// States that a training forward stores of t steps.
int64_t chunks(int64_t t) {
  const int64_t every = mqc_gated_scan_chunk();
  return (t + every - 1) / every;
}

std::tuple<Tensor, Tensor, MaybeTensor> scan_forward(const Scan& o, const MaybeTensor& h0, bool train) {
  const c10::DeviceGuard guard(o.x.device());
  const int64_t b = o.b(), t = o.t(), d = o.d();
  Tensor y = at::empty({b, t, d}, o.x.options()), h = like_f32({b, d}, o.x);
  MaybeTensor carries;
  if (train) carries = like_f32({b, chunks(t), d}, o.x);
  const int64_t bytes = mqc_gated_scan_workspace_bytes(b, t, d);
  const Tensor ws = workspace(bytes, "mqc_gated_scan_fwd", o.x);
  check(mqc_gated_scan_fwd(o.dt.data_ptr(), o.dt_row, o.g.data_ptr(), o.g_row, o.x.data_ptr(), o.x_row,
                           f32(o.rate), f32(h0), ptr(o.reset), y.data_ptr(), (float*)h.data_ptr(),
                           (float*)ptr(carries), b, t, d, dtype_code(o.x), ws.data_ptr(), bytes,
                           stream_of(o.x)),
        "mqc_gated_scan_fwd");
  return {y, h, carries};
}

// ddt, dg, dx, dlog_rate, dh0.
std::vector<MaybeTensor> scan_backward(const Scan& o, Tensor carries, MaybeTensor dy, MaybeTensor dh,
                                       bool want_dh0) {
  const c10::DeviceGuard guard(o.x.device());
  const int64_t b = o.b(), t = o.t(), d = o.d();
  carries = beside("gated_scan", "the chunks' states", carries, {b, chunks(t), d}, at::kFloat, o.x);
  if (dy) dy = beside("gated_scan", "the gradient of y", *dy, {b, t, d}, o.x.scalar_type(), o.x);
  if (dh) dh = beside("gated_scan", "the state's gradient", *dh, {b, d}, at::kFloat, o.x);
  const auto grad = [&] { return at::empty({b, t, d}, o.x.options()); };
  Tensor ddt = grad(), dg = grad(), dx = grad();
  MaybeTensor dh0;
  if (o.x.numel() == 0) {
    if (want_dh0) dh0 = dh ? dh->clone() : at::zeros({b, d}, o.rate.options());
    return {ddt, dg, dx, at::zeros_like(o.rate), dh0};
  }
  if (!dy) dy = at::zeros({b, t, d}, o.x.options());
  Tensor drate = at::empty_like(o.rate);
  if (want_dh0) dh0 = like_f32({b, d}, o.x);
  const int64_t bytes = mqc_gated_scan_workspace_bytes(b, t, d);
  const Tensor ws = workspace(bytes, "mqc_gated_scan_bwd", o.x);
  check(mqc_gated_scan_bwd(o.dt.data_ptr(), o.dt_row, o.g.data_ptr(), o.g_row, o.x.data_ptr(), o.x_row,
                           f32(o.rate), ptr(o.reset), f32(carries), ptr(dy), f32(dh), ddt.data_ptr(),
                           dg.data_ptr(), dx.data_ptr(), (float*)drate.data_ptr(), (float*)ptr(dh0), b,
                           t, d, dtype_code(o.x), ws.data_ptr(), bytes, stream_of(o.x)),
        "mqc_gated_scan_bwd");
  return {ddt, dg, dx, drate, dh0};
}

bool scan_shapes(const Tensor& dt, const Tensor& g, const Tensor& x, const Tensor& rate,
                 const MaybeTensor& h, const MaybeTensor& reset) {
  if (x.dim() != 3 || dt.sizes() != x.sizes() || g.sizes() != x.sizes()) return false;
  const int64_t b = x.size(0), t = x.size(1), d = x.size(2);
  return rate.dim() == 1 && rate.size(0) == d && (!h || h->sizes() == at::IntArrayRef{b, d}) &&
         (!reset || (reset->sizes() == at::IntArrayRef{b, t} && reset->scalar_type() == at::kBool));
}

struct ScanNode : torch::autograd::Function<ScanNode> {
  static variable_list forward(AutogradContext* ctx, const Variable& dt, const Variable& g,
                               const Variable& x, const Variable& log_rate, const MaybeTensor& h0,
                               const Scan& o, const MaybeTensor& h0_read) {
    auto [y, h, carries] = scan_forward(o, h0_read, true);
    ctx->save_for_backward({o.dt, o.g, o.x, o.rate, edge(o.reset), *carries});
    ctx->set_materialize_grads(false);
    ctx->saved_data["types"] = grad_types({dt, g, x, log_rate, h0});
    return {y, h};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (laid out anew, as in GateNormNode)
    const auto s = ctx->get_saved_variables();
    const auto types = ctx->saved_data["types"].toIntVector();
    TORCH_CHECK_VALUE(scan_shapes(s[0], s[1], s[2], s[3], std::nullopt, maybe(s[4])),
                      "gated_scan: the saved tensors came back in other shapes");
    const Scan o("gated_scan", s[0], s[1], s[2], s[3], maybe(s[4]), std::nullopt, nullptr);
    const auto got = scan_backward(o, s[5], maybe(grads[0]), maybe(grads[1]), types[4] >= 0);
    return once("gated_scan", as_grads(got, types, 7));
  }
};

// gated_scan (y, last state), or nothing where the arguments do not match.
std::optional<std::tuple<Tensor, Tensor>> gated_scan(const Tensor& dt, const Tensor& g, const Tensor& x,
                                                     const Tensor& log_rate, const MaybeTensor& h0,
                                                     const MaybeTensor& reset, const py::object& convert) {
  if (!scan_shapes(dt, g, x, log_rate, h0, reset)) return std::nullopt;
  const Scan o("gated_scan", dt, g, x, log_rate, reset, h0, &convert);
  MaybeTensor state;
  if (h0) state = as_type(*h0, at::kFloat).contiguous();
  if (records({dt, g, x, log_rate, h0})) {
    const auto out = ScanNode::apply(dt, g, x, log_rate, h0, o, state);
    return std::make_tuple(out[0], out[1]);
  }
  auto [y, h, carries] = scan_forward(o, state, false);
  return std::make_tuple(y, h);
}

// gated_scan_step_, or nothing where the arguments do not match.
MaybeTensor gated_scan_step(const Tensor& dt, const Tensor& g, const Tensor& x, const Tensor& log_rate,
                            const Tensor& h, const py::object& convert) {
  if (!scan_shapes(dt, g, x, log_rate, h, std::nullopt) || x.size(1) != 1 ||
      h.scalar_type() != at::kFloat || !h.is_contiguous() || h.is_neg())
    return std::nullopt;
  const Scan o("gated_scan_step_", dt, g, x, log_rate, std::nullopt, h, &convert);
  const c10::DeviceGuard guard(o.x.device());
  Tensor y = at::empty({o.b(), 1, o.d()}, o.x.options());
  check(mqc_gated_scan_step(o.dt.data_ptr(), o.dt_row, o.g.data_ptr(), o.g_row, o.x.data_ptr(), o.x_row,
                            f32(o.rate), (float*)h.data_ptr(), y.data_ptr(), o.b(), o.d(),
                            dtype_code(o.x), stream_of(o.x)),
        "mqc_gated_scan_step");
  changed(h);
  return y;
}

// --- the gated delta rule -------------------------------------------------------------------------
// t [b, n, h, d] in `type` with a dense last axis; batch rows, tokens and heads are read where they are.
Tensor dense_last(const Tensor& t, at::ScalarType type) {
  const Tensor v = as_type(t, type);
  return v.size(3) > 1 && v.stride(3) != 1 ? v.contiguous() : v;
}

// Operands as the kernels read them: q, k and v in the promoted type, the gates in their own
// (kernels/delta.py).
struct Delta {
  Tensor q, k, v, g, beta;
  MaybeTensor reset;
  float scale;
  int64_t strides[9];
  // (the state h is only looked at)
  Delta(const char* name, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g_,
        const Tensor& beta_, const MaybeTensor& reset_, const MaybeTensor& h,
        const std::optional<double>& scale_) {
    no_tangents(name, q_, k_, v_, g_, beta_, h);
    for (const Tensor* t : {&v_, &q_, &k_, &g_, &beta_}) on_device(name, *t, v_);
    if (h) on_device(name, *h, v_);
    if (reset_) on_device(name, *reset_, v_), reset = reset_->contiguous();
    const auto type =
        at::promote_types(at::promote_types(q_.scalar_type(), k_.scalar_type()), v_.scalar_type());
    q = dense_last(q_, type), k = dense_last(k_, type), v = dense_last(v_, type);
    g = as_type(g_, g_.scalar_type()).contiguous();
    beta = as_type(beta_, beta_.scalar_type()).contiguous();
    dtype_code(v), dtype_code(g), dtype_code(beta);
    scale = (float)(scale_ ? *scale_ : 1 / std::sqrt((double)q.size(3)));
    const Tensor* const rows[3] = {&q, &k, &v};
    for (int i = 0; i < 3; ++i)
      for (int j = 0; j < 3; ++j) strides[3 * i + j] = rows[i]->stride(j);
  }
  int64_t b() const { return v.size(0); }
  int64_t t() const { return v.size(1); }
  int64_t hk() const { return q.size(2); }
  int64_t hv() const { return v.size(2); }
  int64_t dk() const { return q.size(3); }
  int64_t dv() const { return v.size(3); }
  // What a training forward stores: the chunks' states, and residuals.
  std::vector<int64_t> saved(bool states) const {
    const int64_t c = mqc_gated_delta_chunk(), width = mqc_gated_delta_value_width(dv());
    return {b(), hv(), (t() + c - 1) / c, states ? mqc_gated_delta_key_width(dk()) : c, width};
  }
};

std::tuple<Tensor, Tensor, MaybeTensor, MaybeTensor> delta_forward(const Delta& o, const MaybeTensor& h0,
                                                                   bool train) {
  const c10::DeviceGuard guard(o.v.device());
  const int64_t b = o.b(), t = o.t(), hk = o.hk(), hv = o.hv(), dk = o.dk(), dv = o.dv();
  const int64_t bytes = mqc_gated_delta_workspace_bytes(b, t, hk, hv, dk, dv, dtype_code(o.v), 0);
  const Tensor ws = workspace(bytes, "mqc_gated_delta_fwd", o.v);
  Tensor out = at::empty({b, t, hv, dv}, o.v.options()), h = like_f32({b, hv, dk, dv}, o.v);
  MaybeTensor states, resid;
  if (train) states = like_f32(o.saved(true), o.v), resid = like_f32(o.saved(false), o.v);
  check(mqc_gated_delta_fwd(o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.strides, o.g.data_ptr(),
                            dtype_code(o.g), o.beta.data_ptr(), dtype_code(o.beta), ptr(o.reset),
                            f32(h0), out.data_ptr(), (float*)h.data_ptr(), (float*)ptr(states),
                            (float*)ptr(resid), b, t, hk, hv, dk, dv, o.scale, dtype_code(o.v),
                            ws.data_ptr(), bytes, stream_of(o.v)),
        "mqc_gated_delta_fwd");
  return {out, h, states, resid};
}

// dq, dk, dv, dlog_decay, dbeta, dh0.
std::vector<MaybeTensor> delta_backward(const Delta& o, Tensor states, Tensor resid, MaybeTensor d_o,
                                        MaybeTensor dh, bool want_dh0) {
  const c10::DeviceGuard guard(o.v.device());
  const int64_t b = o.b(), t = o.t(), hk = o.hk(), hv = o.hv(), dk = o.dk(), dv = o.dv();
  states = beside("gated_delta", "the chunks' states", states, o.saved(true), at::kFloat, o.v);
  resid = beside("gated_delta", "the chunks' residuals", resid, o.saved(false), at::kFloat, o.v);
  if (d_o) d_o = beside("gated_delta", "the gradient of o", *d_o, {b, t, hv, dv}, o.v.scalar_type(), o.v);
  if (dh) dh = beside("gated_delta", "the state's gradient", *dh, {b, hv, dk, dv}, at::kFloat, o.v);
  const auto like = [](const Tensor& x) { return at::empty(x.sizes(), x.options()); };
  Tensor dq = like(o.q), dkk = like(o.k), dvv = like(o.v), dg = like(o.g), dbeta = like(o.beta);
  MaybeTensor dh0;
  if (o.v.numel() == 0) {
    if (want_dh0) dh0 = dh ? dh->clone() : at::zeros({b, hv, dk, dv}, o.v.options().dtype(at::kFloat));
    return {dq, dkk, dvv, dg, dbeta, dh0};
  }
  if (!d_o) d_o = at::zeros({b, t, hv, dv}, o.v.options());
  if (want_dh0) dh0 = like_f32({b, hv, dk, dv}, o.v);
  const int64_t bytes = mqc_gated_delta_workspace_bytes(b, t, hk, hv, dk, dv, dtype_code(o.v), 1);
  const Tensor ws = workspace(bytes, "mqc_gated_delta_bwd", o.v);
  check(mqc_gated_delta_bwd(o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.strides, o.g.data_ptr(),
                            dtype_code(o.g), o.beta.data_ptr(), dtype_code(o.beta), ptr(o.reset),
                            f32(states), f32(resid), ptr(d_o), f32(dh), dq.data_ptr(), dkk.data_ptr(),
                            dvv.data_ptr(), dg.data_ptr(), dbeta.data_ptr(), (float*)ptr(dh0), b, t, hk,
                            hv, dk, dv, o.scale, dtype_code(o.v), ws.data_ptr(), bytes, stream_of(o.v)),
        "mqc_gated_delta_bwd");
  return {dq, dkk, dvv, dg, dbeta, dh0};
}

bool delta_shapes(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                  const MaybeTensor& h, const MaybeTensor& reset) {
  if (q.dim() != 4 || v.dim() != 4 || k.sizes() != q.sizes()) return false;
  const int64_t b = v.size(0), t = v.size(1), hk = q.size(2), hv = v.size(2), dk = q.size(3),
                dv = v.size(3);
  const at::IntArrayRef gates = v.sizes().slice(0, 3);
  return q.size(0) == b && q.size(1) == t && hk > 0 && hv > 0 && hv % hk == 0 && dk > 0 && dv > 0 &&
         dk <= 128 && g.sizes() == gates && beta.sizes() == gates &&
         (!h || h->sizes() == at::IntArrayRef{b, hv, dk, dv}) &&
         (!reset || (reset->sizes() == at::IntArrayRef{b, t} && reset->scalar_type() == at::kBool));
}

struct DeltaNode : torch::autograd::Function<DeltaNode> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k,
                               const Variable& v, const Variable& g, const Variable& beta,
                               const MaybeTensor& h0, const Delta& o, const MaybeTensor& h0_read) {
    auto [out, h, states, resid] = delta_forward(o, h0_read, true);
    ctx->save_for_backward({o.q, o.k, o.v, o.g, o.beta, edge(o.reset), *states, *resid});
    ctx->set_materialize_grads(false);
    ctx->saved_data["types"] = grad_types({q, k, v, g, beta, h0});
    ctx->saved_data["scale"] = (double)o.scale;
    return {out, h};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    // (laid out anew, as in GateNormNode)
    const auto s = ctx->get_saved_variables();
    const auto types = ctx->saved_data["types"].toIntVector();
    TORCH_CHECK_VALUE(delta_shapes(s[0], s[1], s[2], s[3], s[4], std::nullopt, maybe(s[5])),
                      "gated_delta: the saved tensors came back in other shapes");
    const Delta o("gated_delta", s[0], s[1], s[2], s[3], s[4], maybe(s[5]), std::nullopt,
                  ctx->saved_data["scale"].toDouble());
    const auto got = delta_backward(o, s[6], s[7], maybe(grads[0]), maybe(grads[1]), types[5] >= 0);
    return once("gated_delta", as_grads(got, types, 8));
  }
};

// gated_delta (o, last state), or nothing where the arguments do not match.
std::optional<std::tuple<Tensor, Tensor>> gated_delta(const Tensor& q, const Tensor& k, const Tensor& v,
                                                      const Tensor& g, const Tensor& beta,
                                                      const MaybeTensor& h0, const MaybeTensor& reset,
                                                      const std::optional<double>& scale) {
  if (!delta_shapes(q, k, v, g, beta, h0, reset)) return std::nullopt;
  const Delta o("gated_delta", q, k, v, g, beta, reset, h0, scale);
  MaybeTensor state;
  if (h0) state = as_type(*h0, at::kFloat).contiguous();
  if (records({q, k, v, g, beta, h0})) {
    const auto out = DeltaNode::apply(q, k, v, g, beta, h0, o, state);
    return std::make_tuple(out[0], out[1]);
  }
  auto [out, h, states, resid] = delta_forward(o, state, false);
  return std::make_tuple(out, h);
}

// gated_delta_step_, or nothing where the arguments do not match.
MaybeTensor gated_delta_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                             const Tensor& beta, const Tensor& h, const std::optional<double>& scale) {
  if (!delta_shapes(q, k, v, g, beta, h, std::nullopt) || v.size(1) != 1 ||
      h.scalar_type() != at::kFloat || !h.is_contiguous() || h.is_neg())
    return std::nullopt;
  const Delta o("gated_delta_step_", q, k, v, g, beta, std::nullopt, h, scale);
  const c10::DeviceGuard guard(o.v.device());
  Tensor out = at::empty({o.b(), 1, o.hv(), o.dv()}, o.v.options());
  check(mqc_gated_delta_step(o.q.data_ptr(), o.k.data_ptr(), o.v.data_ptr(), o.strides, o.g.data_ptr(),
                             dtype_code(o.g), o.beta.data_ptr(), dtype_code(o.beta),
                             (float*)h.data_ptr(), out.data_ptr(), o.b(), o.hk(), o.hv(), o.dk(), o.dv(),
                             o.scale, dtype_code(o.v), stream_of(o.v)),
        "mqc_gated_delta_step");
  changed(h);
  return out;
}

// --- the AdamW step's tables ----------------------------------------------------------------------
using Lists = std::vector<std::vector<Tensor>>;

// The rows of mqc_adamw_step (lists: params, grads, m, v) or mqc_adamw8_step (params, grads, m, r,
// m_scale, r_scale; tensor i rounds by seeds[i]) and those of mqc_grad_norm, or nothing where a list
// or tensor is not what they take.
std::optional<std::pair<py::bytes, py::bytes>> adam_rows(const Lists& lists, int64_t block,
                                                          const std::vector<int64_t>& seeds) {
  const bool eight = lists.size() == 6;
  const size_t count = lists[0].size();
  for (const auto& l : lists)
    if (l.size() != count) return std::nullopt;
  if (eight && seeds.size() != count) return std::nullopt;
  std::vector<int64_t> rows, norm;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;  // of parameters, whose elements are written side by side
  rows.reserve(count * 9);
  norm.reserve(count * 3);
  spans.reserve(count);
  const auto dense = [&](const Tensor& t) {
    return t.layout() == at::kStrided && t.is_cuda() && t.device() == lists[0][0].device() &&
           t.is_contiguous() && !t.is_neg();
  };
  const auto state = eight ? at::kFloat8_e4m3fn : at::kFloat;
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = lists[0][i], &g = lists[1][i];
    const int64_t n = p.numel(), blocks = (n + block - 1) / block;
    const auto type = p.scalar_type();
    if (type != at::kFloat && type != at::kBFloat16 && type != at::kHalf) return std::nullopt;
    if (!dense(p) || !dense(g) || g.scalar_type() != type || g.sizes() != p.sizes()) return std::nullopt;
    for (size_t s = 2; s < lists.size(); ++s) {
      const Tensor& t = lists[s][i];
      if (!dense(t) || t.scalar_type() != (s < 4 ? state : at::kFloat) ||
          t.numel() != (s < 4 ? n : blocks))
        return std::nullopt;
    }
    for (const auto& l : lists) rows.push_back((int64_t)l[i].data_ptr());
    rows.push_back(n);
    rows.push_back(dtype_code(p));
    if (eight) rows.push_back(seeds[i]);
    norm.insert(norm.end(), {(int64_t)g.data_ptr(), n, dtype_code(p)});
    const uintptr_t start = (uintptr_t)p.data_ptr();
    if (n > 0) spans.emplace_back(start, start + n * (type == at::kFloat ? 4 : 2));
  }
  if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return std::nullopt;
  const auto bytes = [](const std::vector<int64_t>& v) {
    return py::bytes((const char*)v.data(), v.size() * sizeof(int64_t));
  };
  return std::make_pair(bytes(rows), bytes(norm));
}

void changed(const Lists& lists) {
  for (const auto& l : lists)
    for (const auto& t : l) changed(t);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::class_<GateNorm>(m, "GateNorm")
      .def(py::init([](const Tensor& x, const Tensor& y, const MaybeTensor& z, const MaybeTensor& post,
                       const Tensor& scale, const Tensor& pre, const py::object& convert) {
        return GateNorm(x, y, z, post, scale, pre, &convert);
      }));
  m.def("spaced_rows", [](const Tensor& t, py::object type) {
    return spaced_rows(t, torch::python::detail::py_object_to_dtype(type));
  });
  m.def("gate_norm_forward", &gate_norm_forward);
  m.def("gate_norm_backward", &gate_norm_backward);
  m.def("gate_norm", &gate_norm);
  py::class_<Scan>(m, "Scan")
      .def(py::init([](const std::string& name, const Tensor& dt, const Tensor& g, const Tensor& x,
                       const Tensor& rate, const MaybeTensor& reset, const MaybeTensor& h0,
                       const py::object& convert) {
        return Scan(name.c_str(), dt, g, x, rate, reset, h0, &convert);
      }));
  m.def("token_rows", [](const Tensor& t, py::object type) {
    return token_rows(t, torch::python::detail::py_object_to_dtype(type));
  });
  m.def("scan_forward", &scan_forward);
  m.def("scan_backward", &scan_backward);
  m.def("gated_scan", &gated_scan);
  m.def("gated_scan_step", &gated_scan_step);
  py::class_<Delta>(m, "Delta")
      .def(py::init([](const std::string& name, const Tensor& q, const Tensor& k, const Tensor& v,
                       const Tensor& g, const Tensor& beta, const MaybeTensor& reset,
                       const MaybeTensor& h0, const std::optional<double>& scale) {
        return Delta(name.c_str(), q, k, v, g, beta, reset, h0, scale);
      }));
  m.def("delta_forward", &delta_forward);
  m.def("delta_backward", &delta_backward);
  m.def("gated_delta", &gated_delta);
  m.def("gated_delta_step", &gated_delta_step);
  py::class_<LayerNorm>(m, "LayerNorm")
      .def(py::init([](const Tensor& x, const MaybeTensor& w, const MaybeTensor& b,
                       const py::object& convert) { return LayerNorm(x, w, b, &convert); }));
  m.def("layer_norm_forward", &layer_norm_forward);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("layer_norm", &layer_norm);
  m.def("adam_rows", &adam_rows);
  m.def("changed", [](const Lists& lists) { changed(lists); });
  m.def("abi", [] { return (int64_t)MQC_ABI_VERSION; });  // of the header this was compiled with
}

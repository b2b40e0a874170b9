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
  m.def("adam_rows", &adam_rows);
  m.def("changed", [](const Lists& lists) { changed(lists); });
  m.def("abi", [] { return (int64_t)MQC_ABI_VERSION; });  // of the header this was compiled with
}

// torch binding of the training operators (boltz_mlx_amd/_train.so): argument checks, outputs and workspaces from torch's
// allocator, torch's current stream, and the autograd nodes. Launches go through the C entry points of include/bzpf.h, in
// the library that the rest of the package calls.
//
// Native because a training step is bound by the host where its tensors are small: torch runs backward passes on a
// thread of its own, where the same code in Python takes twice its time (a LayerNorm step at 400 x 384 112 us with
// Python autograd functions; of it the kernels take 12 us, torch's own engine some 45 us).
//
// Arguments are checked before devices, so that what a call would refuse can be seen without a GPU.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <stdexcept>
#include <string>
#include <tuple>

#include "bzpf.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef const std::optional<Tensor>& Opt;  // None: an undefined tensor
Tensor get(Opt o) { return o.value_or(Tensor()); }

int type_code(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "unsupported dtype ", t);
  return t == at::kFloat ? BZPF_F32 : t == at::kHalf ? BZPF_F16 : BZPF_BF16;
}
int type_code(const Tensor& t) { return type_code(t.scalar_type()); }

// The calling thread's device is t's for the scope, and so the current stream one of t's device.
struct OnDevice {
  c10::OptionalDeviceGuard guard;
  void* stream;
  explicit OnDevice(const Tensor& t) : guard(t.device()) {
    stream = c10::hip::getCurrentHIPStream(t.device().index()).stream();
  }
};

// The entry points, in the library that boltz_mlx_amd._lib has loaded: this module links none, so that a process holds one
// copy, whichever it is. Set when the module is imported, before any call.
#define BZPF_ENTRIES(X)                                                                                       \
  X(last_error) X(layernorm) X(layernorm_bwd_ws) X(layernorm_bwd) X(dropout) X(dropout_add_ln) X(dropout_add_ln_bwd)
struct {
#define X(f) decltype(&::bzpf_##f) f;
  BZPF_ENTRIES(X)
#undef X
} lib;

// An entry point's refusal or failure: boltz_mlx_amd._lib.BzpfError in Python, as from every other call of the package.
struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int rc, const char* name) {
  if (rc != BZPF_OK) throw Failure(c10::str(name, " failed (", rc, "): ", lib.last_error()));
}

template <typename... Ts>
void on_gpu(const char* name, const Ts&... ts) {
  TORCH_CHECK_VALUE((... && (!ts.defined() || ts.is_cuda())), name, ": need ROCm device tensors");
}

struct Rows {
  int64_t rows, D;
};
Rows rows_of(const char* name, const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, name, ": need rows of channels, got ", x.sizes());
  Rows r{1, x.size(-1)};
  for (int64_t i = 0; i + 1 < x.dim(); i++) r.rows *= x.size(i);
  return r;
}
// The row width of the LayerNorm operators.
int width(const char* name, const Rows& r) {
  TORCH_CHECK_VALUE(r.D >= 8 && r.D <= 8192, name, ": rows of 8 to 8192 channels, got ", r.D);
  return (int)r.D;
}

void alike(const char* name, const Tensor& x, const Tensor& t) {
  TORCH_CHECK_VALUE(t.sizes() == x.sizes() && t.device() == x.device(), name,
                    ": need tensors of one shape on one device, got ", x.sizes(), " on ", x.device(), " and ", t.sizes(),
                    " on ", t.device());
}
void fp32(const char* name, const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat, name, ": ", what, " must be fp32");
}

// A LayerNorm's weight or bias, checked against x, in fp32 and contiguous (itself where it is both; undefined stays).
// The caller holds it until its launch is made.
Tensor param(const char* name, const Tensor& x, const Tensor& p) {
  if (!p.defined()) return p;
  TORCH_CHECK_VALUE(p.numel() == x.size(-1) && p.device() == x.device(), name, ": weight and bias must be [", x.size(-1),
                    "] tensors on ", x.device());
  return p.scalar_type() == at::kFloat && p.is_contiguous() ? p : p.detach().to(at::kFloat).contiguous();
}
const float* f32(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
float* f32_out(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
const void* in(const Tensor& t) { return t.const_data_ptr(); }
void* out(const Tensor& t) { return t.data_ptr(); }

struct Drop {
  double p;
  int64_t site, shared;  // 0: a draw for each element, 1: for each row, 2: for each column of [.., I, J, D]
};
struct DropArgs {
  const int64_t* rng;
  int64_t I = 1, J = 1;
};
DropArgs drop_args(const char* name, const Tensor& x, const Drop& d, const Tensor& rng) {
  TORCH_CHECK_VALUE(d.p >= 0.0 && d.p <= 1.0, name, ": p must lie in [0, 1], got ", d.p);
  TORCH_CHECK_VALUE(d.site >= 0 && d.site < 65536, name, ": site must lie in [0, 65535], got ", d.site);
  TORCH_CHECK_VALUE(d.p == 0.0 || (rng.defined() && rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 &&
                                   rng.is_contiguous() && rng.device() == x.device()),
                    name, ": rng must be an int64 tensor (seed, offset) on ", x.device(), " (dropout_rng)");
  DropArgs a{d.p > 0.0 ? rng.const_data_ptr<int64_t>() : nullptr};
  if (d.shared) {
    TORCH_CHECK_VALUE(x.dim() >= 3, name, ": draws are shared over the rows or columns of a [.., I, J, D] tensor, got ",
                      x.sizes());
    a.I = x.size(-3), a.J = x.size(-2);
  }
  return a;
}

// dweight, dbias and the workspace of a backward pass over x's rows (zeros where there are no rows).
struct ParamGrads {
  Tensor dw, db, ws;
  int64_t ws_bytes = 0;
  ParamGrads(const Tensor& x, Rows r, bool need_w, bool need_b) {
    const auto opt = x.options().dtype(at::kFloat);
    const auto make = [&] { return r.rows ? at::empty({r.D}, opt) : at::zeros({r.D}, opt); };
    if (need_w) dw = make();
    if (need_b) db = make();
    if (!need_w && !need_b) return;
    ws_bytes = lib.layernorm_bwd_ws(r.rows, (int)r.D);
    if (ws_bytes > 0) ws = at::empty({ws_bytes / 4}, opt);
  }
};

Tensor layer_norm(const Tensor& x_, const Tensor& weight, const Tensor& bias, double eps, at::ScalarType to) {
  const char* name = "layer_norm";
  const Rows r = rows_of(name, x_);
  const int D = width(name, r), xt = type_code(x_), yt = type_code(to);
  const Tensor w = param(name, x_, weight), b = param(name, x_, bias);
  on_gpu(name, x_);
  const OnDevice dev(x_);
  const Tensor x = x_.contiguous(), y = at::empty(x.sizes(), x.options().dtype(to));
  check(lib.layernorm(in(x), xt, f32(w), f32(b), (float)eps, out(y), yt, r.rows, D, dev.stream), "bzpf_layernorm");
  return y;
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& dy_, const Tensor& x_, const Tensor& weight, double eps,
                                                  bool need_weight, bool need_bias) {
  const char* name = "layer_norm_bwd";
  alike(name, x_, dy_);
  const Rows r = rows_of(name, x_);
  const int D = width(name, r), gt = type_code(dy_), xt = type_code(x_);
  const Tensor w = param(name, x_, weight);
  on_gpu(name, x_);
  const OnDevice dev(x_);
  const Tensor dy = dy_.contiguous(), x = x_.contiguous(), dx = at::empty(x.sizes(), x.options());
  const ParamGrads g(x, r, need_weight, need_bias);
  if (r.rows)
    check(lib.layernorm_bwd(in(dy), gt, in(x), xt, f32(w), (float)eps, out(dx), f32_out(g.dw), f32_out(g.db),
                             f32_out(g.ws), g.ws_bytes, r.rows, D, dev.stream),
          "bzpf_layernorm_bwd");
  return {dx, g.dw, g.db};
}

Tensor dropout(const Tensor& x_, const Drop& d, const Tensor& rng, at::ScalarType to) {
  const char* name = "dropout";
  const DropArgs a = drop_args(name, x_, d, rng);
  const int xt = type_code(x_), yt = type_code(to);
  on_gpu(name, x_);
  const OnDevice dev(x_);
  const Tensor x = x_.contiguous(), y = at::empty(x.sizes(), x.options().dtype(to));
  const int64_t n = x.numel(), D = x.dim() ? x.size(-1) : 1;
  if (n)
    check(lib.dropout(in(x), xt, d.p, a.rng, (int)d.site, (int)d.shared, a.I, a.J, out(y), yt, n / D, D, dev.stream),
          "bzpf_dropout");
  return y;
}

std::tuple<Tensor, Tensor> dropout_add_ln(const Tensor& z_, const Tensor& y_, const Tensor& weight, const Tensor& bias,
                                          double eps, const Drop& d, const Tensor& rng, at::ScalarType to) {
  const char* name = "dropout_add_ln";
  alike(name, z_, y_);
  fp32(name, z_, "z");
  const DropArgs a = drop_args(name, z_, d, rng);
  const Rows r = rows_of(name, z_);
  const int D = width(name, r), yt = type_code(y_), lt = type_code(to);
  const Tensor w = param(name, z_, weight), b = param(name, z_, bias);
  on_gpu(name, z_);
  const OnDevice dev(z_);
  const Tensor z = z_.contiguous(), y = y_.contiguous(), z_new = at::empty(z.sizes(), z.options());
  const Tensor ln = at::empty(z.sizes(), z.options().dtype(to));
  check(lib.dropout_add_ln(f32(z), in(y), yt, d.p, a.rng, (int)d.site, (int)d.shared, a.I, a.J, f32(w), f32(b),
                            (float)eps, f32_out(z_new), out(ln), lt, r.rows, D, dev.stream),
        "bzpf_dropout_add_ln");
  return {z_new, ln};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> dropout_add_ln_bwd(const Tensor& dz_new_, const Tensor& dln_,
                                                              const Tensor& z_new_, const Tensor& weight, double eps,
                                                              const Drop& d, const Tensor& rng, at::ScalarType y_type,
                                                              bool need_weight, bool need_bias) {
  const char* name = "dropout_add_ln_bwd";
  alike(name, z_new_, dln_);
  fp32(name, z_new_, "z_new");
  if (dz_new_.defined()) {
    alike(name, z_new_, dz_new_);
    fp32(name, dz_new_, "dz_new");
  }
  const DropArgs a = drop_args(name, z_new_, d, rng);
  const Rows r = rows_of(name, z_new_);
  const int D = width(name, r), lt = type_code(dln_), yt = type_code(y_type);
  const Tensor w = param(name, z_new_, weight);
  on_gpu(name, z_new_);
  const OnDevice dev(z_new_);
  const Tensor dln = dln_.contiguous(), z_new = z_new_.contiguous();
  const Tensor dz_new = dz_new_.defined() ? dz_new_.contiguous() : dz_new_;
  const Tensor dz = at::empty(z_new.sizes(), z_new.options());
  const Tensor dy = at::empty(z_new.sizes(), z_new.options().dtype(y_type));
  const ParamGrads g(z_new, r, need_weight, need_bias);
  if (r.rows)
    check(lib.dropout_add_ln_bwd(f32(dz_new), in(dln), lt, f32(z_new), f32(w), (float)eps, d.p, a.rng, (int)d.site,
                                  (int)d.shared, a.I, a.J, f32_out(dz), out(dy), yt, f32_out(g.dw), f32_out(g.db),
                                  f32_out(g.ws), g.ws_bytes, r.rows, D, dev.stream),
          "bzpf_dropout_add_ln_bwd");
  return {dz, dy, g.dw, g.db};
}

// ------------------------------------------------------------------------------------------------ autograd

// Backward passes are not differentiable: a call that asks for their graph is refused rather than given none.
void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": gradients of gradients are not provided (create_graph)");
}
int64_t type_of(const Tensor& t) { return static_cast<int64_t>(t.defined() ? t.scalar_type() : at::kFloat); }
// A parameter's gradient in its type.
Tensor as(const Tensor& g, int64_t type) { return g.defined() ? g.to(static_cast<at::ScalarType>(type)) : g; }

// The weight and bias of a node: which of them are there (a node's inputs are counted over those that are), and the bias's
// type. `before`: the node's inputs before them.
void save_params(AutogradContext* ctx, const Tensor& w, const Tensor& b) {
  TORCH_CHECK_VALUE((!w.defined() || w.dim() == 1) && (!b.defined() || b.dim() == 1),
                    "weight and bias must be one-dimensional (their gradients are)");
  ctx->saved_data["has"] = (int64_t)w.defined() + 2 * (int64_t)b.defined();
  ctx->saved_data["b"] = type_of(b);
}
struct Needs {
  bool weight, bias;
  Needs(AutogradContext* ctx, int before) {
    const int64_t has = ctx->saved_data["has"].toInt();
    weight = (has & 1) && ctx->needs_input_grad(before);
    bias = (has & 2) && ctx->needs_input_grad(before + (has & 1));
  }
};

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, Opt w_, Opt b_, double eps, at::ScalarType to) {
    const Tensor x = x_.contiguous(), w = get(w_), b = get(b_);
    ctx->save_for_backward({x, w});
    ctx->saved_data["eps"] = eps;
    save_params(ctx, w, b);
    return layer_norm(x, w, b, eps, to);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("layer_norm");
    const variable_list s = ctx->get_saved_variables();
    const Needs need(ctx, 1);
    auto [dx, dw, db] =
        layer_norm_bwd(g[0], s[0], s[1], ctx->saved_data["eps"].toDouble(), need.weight, need.bias);
    return {dx, as(dw, type_of(s[1])), as(db, ctx->saved_data["b"].toInt()), Tensor(), Tensor()};
  }
};

void save(AutogradContext* ctx, const Drop& d) {
  ctx->saved_data["p"] = d.p;
  ctx->saved_data["site"] = d.site;
  ctx->saved_data["shared"] = d.shared;
}
Drop saved(AutogradContext* ctx) {
  return Drop{ctx->saved_data["p"].toDouble(), ctx->saved_data["site"].toInt(), ctx->saved_data["shared"].toInt()};
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, Opt rng_, int64_t site, int64_t shared) {
    const Drop d{p, site, shared};
    const Tensor rng = get(rng_);
    save(ctx, d);
    ctx->save_for_backward({rng});
    return dropout(x, d, rng, x.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("dropout");
    const Tensor rng = ctx->get_saved_variables()[0];
    return {dropout(g[0], saved(ctx), rng, g[0].scalar_type()), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct DropoutAddLNNode : torch::autograd::Function<DropoutAddLNNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& y, Opt w_, Opt b_, double eps,
                               double p, Opt rng_, int64_t site, int64_t shared, at::ScalarType to) {
    const Drop d{p, site, shared};
    const Tensor w = get(w_), b = get(b_), rng = get(rng_);
    auto [z_new, ln] = dropout_add_ln(z, y, w, b, eps, d, rng, to);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({z_new, w, rng});
    save(ctx, d);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["y"] = type_of(y);
    save_params(ctx, w, b);
    return {z_new, ln};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& g) {
    once("dropout_add_ln");
    const variable_list s = ctx->get_saved_variables();
    const Drop d = saved(ctx);
    const auto y_type = static_cast<at::ScalarType>(ctx->saved_data["y"].toInt());
    Tensor dz, dy, dw, db;
    if (g[1].defined()) {
      const Needs need(ctx, 2);
      std::tie(dz, dy, dw, db) = dropout_add_ln_bwd(g[0], g[1], s[0], s[1], ctx->saved_data["eps"].toDouble(), d, s[2],
                                                    y_type, need.weight, need.bias);
    } else if (g[0].defined()) {  // the LayerNorm's output was not used
      dz = g[0];
      dy = dropout(dz, d, s[2], y_type);
    }
    return {dz, dy, as(dw, type_of(s[1])), as(db, ctx->saved_data["b"].toInt()), Tensor(), Tensor(), Tensor(), Tensor(),
            Tensor(), Tensor()};
  }
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  typedef py::call_guard<py::gil_scoped_release> NoGil;
  typedef std::optional<at::ScalarType> Type;

  const std::string torch_here = py::str(py::module_::import("torch").attr("__version__"));
  if (torch_here != BZPF_TORCH) throw py::import_error("built with torch " BZPF_TORCH ", this is " + torch_here);
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& e) {
      PyErr_SetString(py::module_::import("boltz_mlx_amd._lib").attr("BzpfError").ptr(), e.what());
    }
  });
  const py::object address = py::module_::import("boltz_mlx_amd._lib").attr("address");
#define X(f) lib.f = reinterpret_cast<decltype(lib.f)>(address("bzpf_" #f).cast<uintptr_t>());
  BZPF_ENTRIES(X)
#undef X

  m.def("layer_norm", [](const Tensor& x, Opt w, Opt b, double eps, at::ScalarType to) {
    return layer_norm(x, get(w), get(b), eps, to);
  }, NoGil());
  m.def("layer_norm_bwd", [](const Tensor& dy, const Tensor& x, Opt w, double eps, bool need_weight, bool need_bias) {
    return layer_norm_bwd(dy, x, get(w), eps, need_weight, need_bias);
  }, NoGil());
  m.def("dropout", [](const Tensor& x, double p, Opt rng, int64_t site, int64_t shared, Type to) {
    return dropout(x, Drop{p, site, shared}, get(rng), to.value_or(x.scalar_type()));
  }, NoGil());
  m.def("dropout_add_ln", [](const Tensor& z, const Tensor& y, Opt w, Opt b, double eps, double p, Opt rng, int64_t site,
                              int64_t shared, Type to) {
    return dropout_add_ln(z, y, get(w), get(b), eps, Drop{p, site, shared}, get(rng), to.value_or(y.scalar_type()));
  }, NoGil());
  m.def("dropout_add_ln_bwd", [](Opt dz_new, const Tensor& dln, const Tensor& z_new, Opt w, double eps, double p, Opt rng,
                                  int64_t site, int64_t shared, Type y_type, bool need_weight, bool need_bias) {
    return dropout_add_ln_bwd(get(dz_new), dln, z_new, get(w), eps, Drop{p, site, shared}, get(rng),
                              y_type.value_or(dln.scalar_type()), need_weight, need_bias);
  }, NoGil());
  m.def("grad_layer_norm", [](const Tensor& x, Opt w, Opt b, double eps, at::ScalarType to) {
    return LayerNormNode::apply(x, w, b, eps, to);
  }, NoGil());
  m.def("grad_dropout", [](const Tensor& x, double p, Opt rng, int64_t site, int64_t shared) {
    return DropoutNode::apply(x, p, rng, site, shared);
  }, NoGil());
  m.def("grad_dropout_add_ln", [](const Tensor& z, const Tensor& y, Opt w, Opt b, double eps, double p, Opt rng,
                                   int64_t site, int64_t shared, Type to) {
    const variable_list o =
        DropoutAddLNNode::apply(z, y, w, b, eps, p, rng, site, shared, to.value_or(y.scalar_type()));
    return std::make_tuple(o[0], o[1]);
  }, NoGil());
}

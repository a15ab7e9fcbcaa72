// Host glue of the model-side operators (tgengine_amd.ops), part of the torch
// extension module `tgengine_amd._tgx_host`: argument checks, outputs and
// workspaces from the caching allocator, autograd, and the launches through
// libtgx on the caller's current stream.
//
// Without a gradient to keep (no input asks for one, or grad mode is off) a call
// goes straight to the launch.  The backward passes are kernels themselves and
// leave no graph: asking for one (create_graph) raises.  So do the ways to follow a call
// that see none of its launches, forward-mode derivatives and tracing.
#include <torch/extension.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "tgx.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

[[noreturn]] void bad(const std::string& msg) { throw std::invalid_argument(msg); }

void check(int rc, const char* what) {
  if (rc != TGX_OK) throw std::runtime_error(std::string(what) + " failed: " + tgx_last_error());
}

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

int32_t dtype_of(const Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return TGX_F32;
  if (t.scalar_type() == at::kBFloat16) return TGX_BF16;
  bad(std::string(what) + " must be float32 or bfloat16");
}

void on_gpu(const Tensor& t, const char* what) {
  if (!t.is_cuda()) throw std::runtime_error(std::string(what) + " must be on the GPU (libtgx has no CPU path)");
}

void same_device(const Tensor& t, const Tensor& like, const char* what) {
  if (t.device() != like.device()) bad(std::string(what) + " must be on the device of the first argument");
}

bool keeps_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// forward-mode derivatives would be taken for zeros, and a trace would record the outputs' bare
// memory
void reverse_mode_only(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined())
      throw std::runtime_error(std::string(what) + " has no forward-mode derivative");
  if (torch::jit::tracer::isTracing()) throw std::runtime_error(std::string(what) + " cannot be traced");
}

// a backward pass that is asked for a graph of its own
void only_once(const char* what) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(std::string(what) + " can be differentiated once only (create_graph is not supported)");
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes == 0 ? Tensor() : at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// rows of the last dimension as (rows, row stride), or a contiguous copy where the
// tensor's rows are not one even step apart
Tensor as_rows(const Tensor& t, int64_t& rows, int64_t& stride) {
  const int64_t dim = t.size(-1);
  rows = dim > 0 ? t.numel() / dim : 0;
  stride = dim;
  if (t.is_contiguous()) return t;
  if (t.dim() == 2 && (t.stride(1) == 1 || dim == 1)) {
    stride = t.stride(0);
    return t;
  }
  return t.contiguous();
}

// ------------------------------------------------------------------ embed
void check_embed(const Tensor& table, const Tensor& ids) {
  on_gpu(table, "embed: table");
  if (table.dim() != 2 || table.size(1) < 1) bad("embed: table must be (rows, dim)");
  dtype_of(table, "embed: table");
  if (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong) bad("embed: ids must be int32 or int64");
  same_device(ids, table, "embed: ids");
}

Tensor embed_out(const Tensor& table_in, const Tensor& ids, double scale) {
  const c10::OptionalDeviceGuard guard(table_in.device());
  // rows in place where they are dense and apart, or one row for all
  const int64_t dim = table_in.size(1), step = table_in.size(0) > 1 ? table_in.stride(0) : dim;
  const bool in_place = (dim == 1 || table_in.stride(1) == 1) && (step >= dim || step == 0);
  const Tensor table = in_place ? table_in : table_in.contiguous();
  std::vector<int64_t> shape = ids.sizes().vec();
  shape.push_back(dim);
  Tensor out = at::empty(shape, table.options());
  check(tgx_embed(table.data_ptr(), table.size(0), dim, in_place ? step : dim, dtype_of(table, "embed: table"),
                  ids.data_ptr(), ids.scalar_type() == at::kInt, ids.numel(), static_cast<float>(scale),
                  out.data_ptr(), stream_of(table)),
        "tgx_embed");
  return out;
}

class Embed : public torch::autograd::Function<Embed> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    return embed_out(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("embed");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const Tensor ids = ctx->get_saved_variables()[0];
    const Tensor g = grads[0].contiguous();
    const c10::OptionalDeviceGuard guard(g.device());
    const int64_t rows = ctx->saved_data["rows"].toInt(), dim = g.size(-1), n = ids.numel();
    Tensor out = at::empty({rows, dim}, g.options());
    const Tensor ws = workspace(tgx_embed_grad_workspace_size(n, dim), g);
    check(tgx_embed_grad(g.data_ptr(), ids.data_ptr(), ids.scalar_type() == at::kInt, n, rows, dim,
                         dtype_of(g, "embed"), static_cast<float>(ctx->saved_data["scale"].toDouble()),
                         out.data_ptr(), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(g)),
          "tgx_embed_grad");
    return {out, Tensor(), Tensor()};
  }
};

Tensor embed(const Tensor& table, const Tensor& ids, double scale) {
  check_embed(table, ids);
  reverse_mode_only("embed", {&table});
  const Tensor flat = ids.contiguous();
  return keeps_grad({&table}) ? Embed::apply(table, flat, scale) : embed_out(table, flat, scale);
}

// ------------------------------------------------------------------ layer norm
struct NormIn {
  Tensor x, w, b;
  int64_t rows = 0, dim = 0, stride = 0;
  int32_t dt = 0, wdt = 0;
  NormIn(const Tensor& x_in, const Tensor& weight, const Tensor& bias) {
    dim = x_in.size(-1);
    x = as_rows(x_in, rows, stride);
    dt = dtype_of(x, "layer_norm: x");
    w = weight.defined() ? weight.contiguous() : weight;
    b = bias.defined() ? bias.contiguous() : bias;
    const Tensor& any = w.defined() ? w : b;
    wdt = any.defined() ? dtype_of(any, "layer_norm: weight") : dt;
  }
};

void check_norm(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  on_gpu(x, "layer_norm: x");
  if (x.dim() < 1 || x.size(-1) < 1) bad("layer_norm: x must have a last dimension of 1 or more");
  dtype_of(x, "layer_norm: x");
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    if (t->dim() != 1 || t->size(0) != x.size(-1)) bad("layer_norm: weight and bias must be (dim,)");
    dtype_of(*t, "layer_norm: weight and bias");
    same_device(*t, x, "layer_norm: weight and bias");
  }
  if (weight.defined() && bias.defined() && weight.scalar_type() != bias.scalar_type())
    bad("layer_norm: weight and bias must have the same dtype");
}

Tensor norm_out(const NormIn& in, at::IntArrayRef shape, double eps, Tensor* stats) {
  Tensor out = at::empty(shape, in.x.options());
  float* mean = nullptr;
  if (stats != nullptr) {
    *stats = at::empty({2, in.rows}, in.x.options().dtype(at::kFloat));
    mean = stats->data_ptr<float>();
  }
  check(tgx_layer_norm(in.x.data_ptr(), in.rows, in.dim, in.stride, in.dt, ptr(in.w), ptr(in.b), in.wdt,
                       static_cast<float>(eps), out.data_ptr(), mean, mean ? mean + in.rows : nullptr,
                       stream_of(in.x)),
        "tgx_layer_norm");
  return out;
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor weight = w.value_or(Tensor()), bias = b.value_or(Tensor());
    const NormIn in(x, weight, bias);
    Tensor stats;
    Tensor out = norm_out(in, x.sizes(), eps, &stats);
    ctx->save_for_backward({x, weight, bias, stats});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("layer_norm");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const c10::OptionalDeviceGuard guard(saved[0].device());
    const NormIn in(saved[0], saved[1], saved[2]);
    const Tensor g = grads[0].contiguous();
    Tensor dx, dw, db;
    if (ctx->needs_input_grad(0)) dx = at::empty(saved[0].sizes(), in.x.options());
    // inputs are counted without those left out
    const size_t iw = 1, ib = saved[1].defined() ? 2 : 1;
    if (saved[1].defined() && ctx->needs_input_grad(iw)) dw = at::empty({in.dim}, in.w.options());
    if (saved[2].defined() && ctx->needs_input_grad(ib)) db = at::empty({in.dim}, in.b.options());
    Tensor ws;
    if (dw.defined() || db.defined()) ws = workspace(tgx_layer_norm_grad_workspace_size(in.rows, in.dim), g);
    const float* mean = saved[3].data_ptr<float>();
    check(tgx_layer_norm_grad(in.x.data_ptr(), g.data_ptr(), in.rows, in.dim, in.stride, in.dt, ptr(in.w), in.wdt,
                              mean, mean + in.rows, ptr(dx), ptr(dw), ptr(db), ptr(ws),
                              ws.defined() ? ws.numel() : 0, stream_of(g)),
          "tgx_layer_norm_grad");
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  check_norm(x, w, b);
  reverse_mode_only("layer_norm", {&x, &w, &b});
  if (keeps_grad({&x, &w, &b})) return LayerNorm::apply(x, weight, bias, eps);
  const c10::OptionalDeviceGuard guard(x.device());
  return norm_out(NormIn(x, w, b), x.sizes(), eps, nullptr);
}

// ------------------------------------------------------------------ attention
// the tensor itself where its last dimension is one value after the other
Tensor dense_last(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

void strides(const Tensor& t, int64_t s[3]) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask) {
  on_gpu(q, "cross_attention: q");
  dtype_of(q, "cross_attention: q");
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4)
    bad("cross_attention: q, k and v must be (batch, tokens, heads, dim)");
  if (k.sizes() != v.sizes()) bad("cross_attention: k and v must have the same shape");
  if (k.size(0) != q.size(0) || k.size(3) != q.size(3)) bad("cross_attention: q and k differ in batch or dim");
  if (q.size(3) < 1 || q.size(3) > TGX_MAX_HEAD_DIM)
    bad("cross_attention: dim must be 1 to " + std::to_string(TGX_MAX_HEAD_DIM));
  if (q.size(2) < 1 || k.size(2) < 1 || q.size(2) % k.size(2) != 0)
    bad("cross_attention: the heads of q must be a multiple of those of k and v");
  for (const Tensor* t : {&k, &v}) {
    if (t->scalar_type() != q.scalar_type()) bad("cross_attention: q, k and v must have the same dtype");
    same_device(*t, q, "cross_attention: k and v");
  }
  if (!mask.defined()) return;
  if (mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte)
    bad("cross_attention: mask must be bool (True = the key takes part)");
  if (mask.dim() != 2 || mask.size(0) != k.size(0) || mask.size(1) != k.size(1))
    bad("cross_attention: mask must be (batch, tokens of k)");
  same_device(mask, q, "cross_attention: mask");
}

tgx_attention_args attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, double scale) {
  tgx_attention_args a{};
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.mask = mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr()) : nullptr;
  a.batch = q.size(0);
  a.lq = q.size(1);
  a.lk = k.size(1);
  a.heads = static_cast<int32_t>(q.size(2));
  a.kv_heads = static_cast<int32_t>(k.size(2));
  a.dim = static_cast<int32_t>(q.size(3));
  a.dtype = dtype_of(q, "cross_attention: q");
  strides(q, a.q_stride);
  strides(k, a.k_stride);
  strides(v, a.v_stride);
  a.mask_stride = mask.defined() ? mask.stride(0) : 0;
  a.scale = static_cast<float>(scale);
  return a;
}

Tensor attention_out(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& mask, double scale, Tensor* lse,
                     Tensor* rest) {
  Tensor out = at::empty(q.sizes(), q.options());
  tgx_attention_args a = attention_args(q, k, v, mask, scale);
  if (lse != nullptr) *lse = at::empty({a.batch, a.lq, a.heads}, q.options().dtype(at::kFloat));
  a.out = out.data_ptr();
  a.lse = lse != nullptr ? lse->data_ptr<float>() : nullptr;
  a.out_rest = rest != nullptr ? ptr(*rest) : nullptr;
  const Tensor ws = workspace(tgx_attention_workspace_size(&a), q);
  a.workspace = ptr(ws);
  a.workspace_bytes = ws.defined() ? ws.numel() : 0;
  check(tgx_attention(&a, stream_of(q)), "tgx_attention");
  return out;
}

class Attention : public torch::autograd::Function<Attention> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const OptTensor& mask_in, double scale) {
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor mask = mask_in.value_or(Tensor());
    Tensor lse, rest;
    if (q.scalar_type() == at::kBFloat16) rest = at::empty(q.sizes(), q.options());
    Tensor out = attention_out(q, k, v, mask, scale, &lse, &rest);
    ctx->save_for_backward({q, k, v, mask, out, lse, rest});
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("cross_attention");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2];
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor g = grads[0].contiguous();
    tgx_attention_args a = attention_args(q, k, v, saved[3], ctx->saved_data["scale"].toDouble());
    a.out = saved[4].data_ptr();
    a.lse = saved[5].data_ptr<float>();
    a.out_rest = ptr(saved[6]);
    a.grad_out = g.data_ptr();
    Tensor d[3];
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) d[i] = at::empty(saved[i].sizes(), q.options());
    a.grad_q = ptr(d[0]);
    a.grad_k = ptr(d[1]);
    a.grad_v = ptr(d[2]);
    const Tensor ws = workspace(tgx_attention_grad_workspace_size(&a), q);
    a.workspace = ptr(ws);
    a.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(tgx_attention_grad(&a, stream_of(q)), "tgx_attention_grad");
    return {d[0], d[1], d[2], Tensor(), Tensor()};
  }
};

Tensor cross_attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const OptTensor& mask_in,
                       const c10::optional<double>& scale_in) {
  Tensor mask = mask_in.value_or(Tensor());
  check_attention(q_in, k_in, v_in, mask);
  reverse_mode_only("cross_attention", {&q_in, &k_in, &v_in});
  const Tensor q = dense_last(q_in), k = dense_last(k_in), v = dense_last(v_in);
  if (mask.defined() && mask.size(1) > 1 && mask.stride(1) != 1) mask = mask.contiguous();
  const double scale = scale_in.has_value() ? *scale_in : 1.0 / std::sqrt(static_cast<double>(q.size(3)));
  if (keeps_grad({&q, &k, &v})) return Attention::apply(q, k, v, mask.defined() ? OptTensor(mask) : c10::nullopt, scale);
  const c10::OptionalDeviceGuard guard(q.device());
  return attention_out(q, k, v, mask, scale, nullptr, nullptr);
}

// ------------------------------------------------------------------ clipping
Tensor clip_grad_norm(std::vector<Tensor> grads, double max_norm, const std::vector<Tensor>& outs) {
  // a leaf that requires a gradient stands for it, as a parameter does
  size_t n = 0;
  for (Tensor& g : grads) {
    Tensor t = g.requires_grad() && g.is_leaf() ? g.grad() : g;
    if (t.defined()) grads[n++] = std::move(t);
    else if (!outs.empty()) bad("clip_grad_norm_: out needs a gradient for each of its tensors");
  }
  grads.resize(n);
  if (n == 0) bad("clip_grad_norm_: no gradients");
  if (!outs.empty() && outs.size() != n) bad("clip_grad_norm_: out must have one tensor per gradient");
  std::vector<const void*> in(n);
  std::vector<void*> out(n);
  std::vector<int32_t> dt(n), odt(n);
  std::vector<int64_t> size(n);
  for (size_t i = 0; i < n; ++i) {
    const Tensor& g = grads[i];
    const Tensor& o = outs.empty() ? g : outs[i];
    reverse_mode_only("clip_grad_norm_", {&g, &o});
    on_gpu(g, "clip_grad_norm_: gradients");
    for (const Tensor* t : {&g, &o}) {
      same_device(*t, grads[0], "clip_grad_norm_: every tensor");
      if (!t->is_contiguous()) bad("clip_grad_norm_: gradients and out must be contiguous");
    }
    if (o.sizes() != g.sizes()) bad("clip_grad_norm_: out must have the gradients' shapes");
    if (!outs.empty() && o.requires_grad() && at::GradMode::is_enabled())
      bad("clip_grad_norm_: out must not require a gradient");
    dt[i] = dtype_of(g, "clip_grad_norm_: gradients");
    odt[i] = dtype_of(o, "clip_grad_norm_: out");
    in[i] = g.data_ptr();
    out[i] = o.data_ptr();
    size[i] = g.numel();
  }
  const c10::OptionalDeviceGuard guard(grads[0].device());
  Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  const Tensor ws = workspace(tgx_clip_grad_norm_workspace_size(size.data(), static_cast<int64_t>(n)), grads[0]);
  const int rc = tgx_clip_grad_norm(in.data(), dt.data(), out.data(), odt.data(), size.data(), static_cast<int64_t>(n),
                                    static_cast<float>(max_norm), norm.data_ptr<float>(), ptr(ws),
                                    ws.defined() ? ws.numel() : 0, stream_of(grads[0]));
  if (rc == TGX_ERR_ARG) bad(tgx_last_error());  // tensors that overlap
  check(rc, "tgx_clip_grad_norm");
  // written behind torch's back: what autograd saved of them is stale
  for (const Tensor& t : outs.empty() ? grads : outs)
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

void bind_ops(py::module_& m) {
  m.def("embed", &embed, py::arg("table"), py::arg("ids"), py::arg("scale") = 1.0);
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5);
  m.def("cross_attention", &cross_attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("mask") = py::none(),
        py::arg("scale") = py::none());
  m.def("clip_grad_norm", &clip_grad_norm, py::arg("grads"), py::arg("max_norm"), py::arg("outs"));
}

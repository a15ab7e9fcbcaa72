// Host glue of the operators around attention (tgengine_amd.ops): the gated recurrence,
// the residual sum with its norms, and the AdamW step.  Same rules as tgx_ops.cpp.
#include "tgx_ops_host.h"

#include <torch/csrc/autograd/python_variable.h>

namespace {

// ------------------------------------------------------------------ gated scan
void check_scan(const Tensor& x, const Tensor& gate, const Tensor& mask, const Tensor& state) {
  on_gpu(x, "gated_scan: x");
  dtype_of(x, "gated_scan: x");
  if (x.dim() != 3 || x.size(2) < 1) bad("gated_scan: x must be (batch, tokens, dim)");
  if (gate.sizes() != x.sizes()) bad("gated_scan: gate must have the shape of x");
  if (gate.scalar_type() != x.scalar_type()) bad("gated_scan: x and gate must have the same dtype");
  same_device(gate, x, "gated_scan: gate");
  if (mask.defined()) {
    if (mask.scalar_type() != at::kBool && mask.scalar_type() != at::kByte)
      bad("gated_scan: mask must be bool (True = the token takes part)");
    if (mask.dim() != 2 || mask.size(0) != x.size(0) || mask.size(1) != x.size(1))
      bad("gated_scan: mask must be (batch, tokens)");
    same_device(mask, x, "gated_scan: mask");
  }
  if (state.defined()) {
    if (state.scalar_type() != at::kFloat) bad("gated_scan: state must be float32");
    if (state.dim() != 2 || state.size(0) != x.size(0) || state.size(1) != x.size(2))
      bad("gated_scan: state must be (batch, dim)");
    same_device(state, x, "gated_scan: state");
  }
}

tgx_scan_args scan_args(const Tensor& x, const Tensor& gate, const Tensor& mask, const Tensor& state) {
  tgx_scan_args a{};
  a.x = x.data_ptr();
  a.gate = gate.data_ptr();
  a.mask = mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr()) : nullptr;
  a.state = static_cast<const float*>(ptr(state));
  a.batch = x.size(0);
  a.length = x.size(1);
  a.dim = x.size(2);
  for (int i = 0; i < 2; ++i) {
    a.x_stride[i] = x.stride(i);
    a.gate_stride[i] = gate.stride(i);
  }
  a.mask_stride = mask.defined() ? mask.stride(0) : 0;
  a.dtype = dtype_of(x, "gated_scan: x");
  return a;
}

// {out, last}; starts: what a gradient needs
variable_list scan_out(const Tensor& x, const Tensor& gate, const Tensor& mask, const Tensor& state, Tensor* starts) {
  tgx_scan_args a = scan_args(x, gate, mask, state);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor out = at::empty(x.sizes(), x.options()), last = at::empty({a.batch, a.dim}, f32);
  if (starts != nullptr) *starts = at::empty({a.batch, tgx_scan_starts(a.length), a.dim}, f32);
  a.out = out.data_ptr();
  a.last = last.data_ptr<float>();
  a.starts = starts != nullptr ? starts->data_ptr<float>() : nullptr;
  const Tensor ws = workspace(tgx_scan_workspace_size(&a), x);
  a.workspace = ptr(ws);
  a.workspace_bytes = ws.defined() ? ws.numel() : 0;
  check(tgx_scan(&a, stream_of(x)), "tgx_scan");
  return {out, last};
}

class Scan : public torch::autograd::Function<Scan> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const OptTensor& state_in,
                               const OptTensor& mask_in) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Tensor state = state_in.value_or(Tensor()), mask = mask_in.value_or(Tensor());
    Tensor starts;
    variable_list out = scan_out(x, gate, mask, state, &starts);
    ctx->save_for_backward({x, gate, state, mask, starts});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("gated_scan");
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gate = saved[1], &state = saved[2];
    const c10::OptionalDeviceGuard guard(x.device());
    tgx_scan_args a = scan_args(x, gate, saved[3], state);
    const Tensor g = grads[0].defined() ? dense(grads[0]) : Tensor();
    const Tensor gl = grads[1].defined() ? dense(grads[1]) : Tensor();
    a.starts = saved[4].data_ptr<float>();
    a.grad_out = ptr(g);
    a.grad_last = static_cast<const float*>(ptr(gl));
    Tensor d[3];  // the first two come together
    for (int i = 0; i < 2; ++i) d[i] = at::empty(x.sizes(), x.options());
    if (state.defined() && ctx->needs_input_grad(2)) d[2] = at::empty(state.sizes(), state.options());
    a.grad_x = ptr(d[0]);
    a.grad_gate = ptr(d[1]);
    a.grad_state = static_cast<float*>(ptr(d[2]));
    const Tensor ws = workspace(tgx_scan_workspace_size(&a), x);
    a.workspace = ptr(ws);
    a.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(tgx_scan_grad(&a, stream_of(x)), "tgx_scan_grad");
    for (int i = 0; i < 2; ++i)
      if (!ctx->needs_input_grad(i)) d[i] = Tensor();
    return {d[0], d[1], d[2], Tensor()};
  }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& x_in, const Tensor& gate_in, const OptTensor& mask_in,
                                      const OptTensor& state_in) {
  Tensor mask = mask_in.value_or(Tensor()), state = state_in.value_or(Tensor());
  check_scan(x_in, gate_in, mask, state);
  reverse_mode_only("gated_scan", {&x_in, &gate_in, &state});
  const Tensor x = dense_last(x_in), gate = dense_last(gate_in);
  if (mask.defined() && mask.size(1) > 1 && mask.stride(1) != 1) mask = mask.contiguous();
  if (state.defined()) state = dense(state);
  variable_list out;
  if (keeps_grad({&x, &gate, &state})) {
    out = Scan::apply(x, gate, state.defined() ? OptTensor(state) : c10::nullopt,
                      mask.defined() ? OptTensor(mask) : c10::nullopt);
  } else {
    const c10::OptionalDeviceGuard guard(x.device());
    out = scan_out(x, gate, mask, state, nullptr);
  }
  return {out[0], out[1]};
}

// ------------------------------------------------------------------ residual norm
// the operator's tensors; those left out are undefined
struct Res {
  Tensor x, residual, gate, weight, bias, scale, post;
  bool parts() const { return gate.defined() || scale.defined() || post.defined(); }
};

void check_residual_norm(const Res& t) {
  on_gpu(t.x, "residual_norm: x");
  if (t.x.dim() < 1 || t.x.size(-1) < 1) bad("residual_norm: x must have a last dimension of 1 or more");
  dtype_of(t.x, "residual_norm: x");
  for (const Tensor* r : {&t.residual, &t.gate}) {
    if (!r->defined()) continue;
    if (r->sizes() != t.x.sizes()) bad("residual_norm: residual and gate must have the shape of x");
    if (r->scalar_type() != t.x.scalar_type()) bad("residual_norm: x, residual and gate must have the same dtype");
    same_device(*r, t.x, "residual_norm: residual and gate");
  }
  const Tensor* first = nullptr;
  for (const Tensor* w : {&t.weight, &t.bias, &t.scale, &t.post}) {
    if (!w->defined()) continue;
    if (w->dim() != 1 || w->size(0) != t.x.size(-1))
      bad("residual_norm: weight, bias, scale and post_weight must be (dim,)");
    dtype_of(*w, "residual_norm: weight, bias, scale and post_weight");
    same_device(*w, t.x, "residual_norm: weight, bias, scale and post_weight");
    if (first != nullptr && first->scalar_type() != w->scalar_type())
      bad("residual_norm: weight, bias, scale and post_weight must have the same dtype");
    first = w;
  }
}

// the arguments, and the contiguous copies that they point to
struct ResCall {
  Res t;
  tgx_residual_norm_args a{};
  ResCall(const Res& in, bool center, double eps) {
    int64_t rows = 0;
    a.dim = in.x.size(-1);
    t.x = as_rows(in.x, a.rows, a.x_stride);
    if (in.residual.defined()) t.residual = as_rows(in.residual, rows, a.residual_stride);
    if (in.gate.defined()) t.gate = as_rows(in.gate, rows, a.gate_stride);
    a.dtype = a.wdtype = dtype_of(in.x, "residual_norm: x");
    const Tensor* from[] = {&in.weight, &in.bias, &in.scale, &in.post};
    Tensor* to[] = {&t.weight, &t.bias, &t.scale, &t.post};
    for (int i = 0; i < 4; ++i) {
      if (!from[i]->defined()) continue;
      *to[i] = dense(*from[i]);
      a.wdtype = dtype_of(*to[i], "residual_norm: weight");
    }
    a.x = t.x.data_ptr();
    a.residual = ptr(t.residual);
    a.gate = ptr(t.gate);
    a.weight = ptr(t.weight);
    a.bias = ptr(t.bias);
    a.scale = ptr(t.scale);
    a.post_weight = ptr(t.post);
    a.center = center;
    a.eps = static_cast<float>(eps);
  }
};

// {y, sum}; stats: what a gradient needs
variable_list residual_norm_out(const Res& t, bool center, double eps, Tensor* stats) {
  ResCall c(t, center, eps);
  Tensor out = at::empty(t.x.sizes(), t.x.options()), sum = at::empty(t.x.sizes(), t.x.options());
  if (stats != nullptr) *stats = at::empty({t.post.defined() ? 4 : 2, c.a.rows}, t.x.options().dtype(at::kFloat));
  c.a.out = out.data_ptr();
  c.a.sum = sum.data_ptr();
  c.a.stats = stats != nullptr ? stats->data_ptr<float>() : nullptr;
  check(tgx_residual_norm(&c.a, stream_of(t.x)), "tgx_residual_norm");
  return {out, sum};
}

class ResidualNorm : public torch::autograd::Function<ResidualNorm> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const OptTensor& weight,
                               const OptTensor& bias, const OptTensor& gate, const OptTensor& scale,
                               const OptTensor& post, bool center, double eps) {
    const c10::OptionalDeviceGuard guard(x.device());
    const Res t{x, residual, gate.value_or(Tensor()), weight.value_or(Tensor()), bias.value_or(Tensor()),
                scale.value_or(Tensor()), post.value_or(Tensor())};
    Tensor stats;
    variable_list out = residual_norm_out(t, center, eps, &stats);
    // an f32 sum is not rounded: alone it gives all that x and residual would
    const bool whole = !t.parts() && x.scalar_type() == at::kFloat;
    ctx->save_for_backward({whole ? out[1] : x, whole ? Tensor() : residual, t.weight, t.bias, t.gate, t.scale, t.post, stats});
    ctx->saved_data["center"] = center;
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    only_once("residual_norm");
    variable_list d(9);
    if (!grads[0].defined() && !grads[1].defined()) return d;
    const variable_list saved = ctx->get_saved_variables();
    const Res t{saved[0], saved[1], saved[4], saved[2], saved[3], saved[5], saved[6]};
    const c10::OptionalDeviceGuard guard(t.x.device());
    ResCall c(t, ctx->saved_data["center"].toBool(), ctx->saved_data["eps"].toDouble());
    const Tensor g = grads[0].defined() ? dense(grads[0]) : Tensor();
    const Tensor gs = grads[1].defined() ? dense(grads[1]) : Tensor();
    c.a.grad_out = ptr(g);
    c.a.grad_sum = ptr(gs);
    c.a.stats = saved[7].data_ptr<float>();
    // inputs are counted without those left out
    const Tensor* in[] = {&t.weight, &t.bias, &t.gate, &t.scale, &t.post};
    void** to[] = {&c.a.grad_weight, &c.a.grad_bias, &c.a.grad_gate, &c.a.grad_scale, &c.a.grad_post_weight};
    const bool wx = ctx->needs_input_grad(0), wr = ctx->needs_input_grad(1);
    bool sums = false;
    for (size_t i = 0, at = 2; i < 5; ++i) {
      if (!in[i]->defined()) continue;
      if (ctx->needs_input_grad(at++)) {
        d[2 + i] = at::empty(in[i]->sizes(), in[i]->options());
        *to[i] = d[2 + i].data_ptr();
        sums |= i != 2;
      }
    }
    if (wr || (wx && !t.parts())) d[1] = at::empty(t.x.sizes(), t.x.options());
    if (wx && t.parts()) d[0] = at::empty(t.x.sizes(), t.x.options());
    c.a.grad_residual = ptr(d[1]);
    c.a.grad_x = ptr(d[0]);
    Tensor ws;
    if (sums) ws = workspace(tgx_residual_norm_grad_workspace_size(&c.a), t.x);
    c.a.workspace = ptr(ws);
    c.a.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(tgx_residual_norm_grad(&c.a, stream_of(t.x)), "tgx_residual_norm_grad");
    if (wx && !t.parts()) d[0] = d[1];
    if (!wr) d[1] = Tensor();
    return d;
  }
};

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                         const OptTensor& bias, const OptTensor& gate, const OptTensor& scale,
                                         const OptTensor& post, bool center, double eps) {
  const Res t{x, residual, gate.value_or(Tensor()), weight.value_or(Tensor()), bias.value_or(Tensor()),
              scale.value_or(Tensor()), post.value_or(Tensor())};
  check_residual_norm(t);
  const std::initializer_list<const Tensor*> all = {&t.x, &t.residual, &t.weight, &t.bias, &t.gate, &t.scale, &t.post};
  reverse_mode_only("residual_norm", all);
  variable_list out;
  if (keeps_grad(all)) {
    out = ResidualNorm::apply(x, residual, weight, bias, gate, scale, post, center, eps);
  } else {
    const c10::OptionalDeviceGuard guard(x.device());
    out = residual_norm_out(t, center, eps, nullptr);
  }
  return {out[0], out[1]};
}

// ------------------------------------------------------------------ AdamW
// the tensors of a list, not counted again: the caller holds the list
class Tensors {
 public:
  Tensors(const py::list& l, size_t n, const char* what) : list_(l.ptr()) {
    if (l.size() != n) bad("adamw_: every list must have one tensor per parameter");
    for (size_t i = 0; i < n; ++i)
      if (!THPVariable_Check(PyList_GET_ITEM(list_, i))) throw py::type_error(std::string("adamw_: ") + what + " must be tensors");
  }
  const Tensor& operator[](size_t i) const { return THPVariable_Unpack(PyList_GET_ITEM(list_, i)); }

 private:
  PyObject* list_;
};

void adamw(const py::list& params_in, const py::list& grads_in, const py::list& exp_avg_in, const py::list& exp_avg_sq_in,
           const py::list& steps_in, const py::list& scales, double lr, const OptTensor& lr_in, double beta1, double beta2,
           double eps, double weight_decay, const OptTensor& norm_in, double max_norm) {
  const size_t n = params_in.size();
  if (n == 0) bad("adamw_: no parameters");
  const Tensors params(params_in, n, "parameters"), grads(grads_in, n, "gradients"), exp_avg(exp_avg_in, n, "averages"),
      exp_avg_sq(exp_avg_sq_in, n, "averages"), steps(steps_in, n, "steps");
  if (scales.size() != 0 && scales.size() != n) bad("adamw_: every list must have one tensor per parameter");
  auto scale_of = [&](size_t i) {
    PyObject* o = scales.size() == 0 ? Py_None : PyList_GET_ITEM(scales.ptr(), i);
    if (o != Py_None && !THPVariable_Check(o)) throw py::type_error("adamw_: scales must be tensors or None");
    return o == Py_None ? Tensor() : THPVariable_Unpack(o);
  };
  std::vector<tgx_adamw_tensor> table(n);
  std::vector<Tensor> copies;
  for (size_t i = 0; i < n; ++i) {
    const Tensor &p = params[i], &g = grads[i], &m = exp_avg[i], &v = exp_avg_sq[i], &t = steps[i];
    reverse_mode_only("adamw_", {&p, &g});
    on_gpu(p, "adamw_: parameters");
    if (p.requires_grad() && !p.is_leaf() && at::GradMode::is_enabled())
      bad("adamw_: parameters must be leaves, or gradients switched off");
    for (const Tensor* x : {&p, &g, &m, &v, &t}) {
      same_device(*x, params[0], "adamw_: every tensor");
      if (!x->is_contiguous()) bad("adamw_: every tensor must be contiguous");
    }
    for (const Tensor* x : {&g, &m, &v})
      if (x->sizes() != p.sizes()) bad("adamw_: gradients and averages must have their parameters' shapes");
    if (t.scalar_type() != at::kLong || t.numel() != 1) bad("adamw_: steps must be int64 of one value");
    if (m.scalar_type() != v.scalar_type() || (m.scalar_type() != at::kFloat && m.scalar_type() != at::kFloat8_e4m3fn))
      bad("adamw_: the averages must be both float32 or both float8_e4m3fn");
    const bool held = m.scalar_type() != at::kFloat;
    tgx_adamw_tensor& a = table[i];
    if (held) {
      const Tensor s = scale_of(i);
      const int64_t blocks = (p.numel() + TGX_ADAMW_BLOCK - 1) / TGX_ADAMW_BLOCK;
      if (!s.defined() || s.scalar_type() != at::kFloat || s.dim() != 2 || s.size(0) != 2 || s.size(1) != blocks ||
          !s.is_contiguous())
        bad("adamw_: 8-bit averages need scales, float32 (2, " + std::to_string(blocks) + ")");
      same_device(s, params[0], "adamw_: every tensor");
      a.scales = s.data_ptr<float>();
    }
    for (const Tensor* x : {&p, &m, &v})
      if (x->is_neg()) bad("adamw_: parameters and averages must not be views of turned signs");
    if (g.is_neg()) copies.push_back(stored(g));
    a.param = p.data_ptr();
    a.grad = (g.is_neg() ? copies.back() : g).data_ptr();
    a.exp_avg = m.data_ptr();
    a.exp_avg_sq = v.data_ptr();
    a.step = t.data_ptr<int64_t>();
    a.size = p.numel();
    a.dtype = dtype_of(p, "adamw_: parameters");
    a.grad_dtype = dtype_of(g, "adamw_: gradients");
    a.bits = held ? 8 : 32;
  }
  tgx_adamw_args a{};
  a.tensors = table.data();
  a.count = static_cast<int64_t>(n);
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.max_norm = max_norm;
  Tensor rate = lr_in.value_or(Tensor()), norm = norm_in.value_or(Tensor());
  for (Tensor* x : {&rate, &norm}) {
    if (!x->defined()) continue;
    *x = stored(*x);
    if (x->scalar_type() != at::kFloat || x->numel() != 1) bad("adamw_: lr and grad_norm must be float32 of one value");
    same_device(*x, params[0], "adamw_: every tensor");
  }
  a.lr_device = static_cast<const float*>(ptr(rate));
  a.grad_norm = static_cast<const float*>(ptr(norm));
  const c10::OptionalDeviceGuard guard(params[0].device());
  const Tensor ws = workspace(tgx_adamw_workspace_size(a.count), params[0]);
  a.workspace = ptr(ws);
  a.workspace_bytes = ws.numel();
  const int rc = tgx_adamw(&a, stream_of(params[0]));
  if (rc == TGX_ERR_ARG) bad(tgx_last_error());  // constants out of range, tensors that overlap
  check(rc, "tgx_adamw");
  // written behind torch's back: what autograd saved of them is stale
  auto written = [](const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  };
  for (size_t i = 0; i < n; ++i) {
    for (const Tensors* l : {&params, &exp_avg, &exp_avg_sq, &steps}) written((*l)[i]);
    if (table[i].bits == 8) written(scale_of(i));
  }
}

}  // namespace

void bind_block_ops(py::module_& m) {
  m.def("adamw", &adamw);
  m.def("gated_scan", &gated_scan, py::arg("x"), py::arg("gate"), py::arg("mask") = py::none(),
        py::arg("state") = py::none());
  m.def("residual_norm", &residual_norm, py::arg("x"), py::arg("residual"), py::arg("weight") = py::none(),
        py::arg("bias") = py::none(), py::arg("gate") = py::none(), py::arg("scale") = py::none(),
        py::arg("post_weight") = py::none(), py::arg("center") = true, py::arg("eps") = 1e-5);
}

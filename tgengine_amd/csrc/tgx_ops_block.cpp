// Host glue of the operators around attention (tgengine_amd.ops): the gated recurrence,
// the residual sum with its norms, and the AdamW step.  Same rules as tgx_ops.cpp.
#include "tgx_ops_host.h"

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
    const Tensor g = grads[0].defined() ? grads[0].contiguous() : Tensor();
    const Tensor gl = grads[1].defined() ? grads[1].contiguous() : Tensor();
    a.starts = saved[4].data_ptr<float>();
    a.grad_out = ptr(g);
    a.grad_last = static_cast<const float*>(ptr(gl));
    Tensor d[3];
    for (int i = 0; i < 2; ++i)
      if (ctx->needs_input_grad(i)) d[i] = at::empty(x.sizes(), x.options());
    if (state.defined() && ctx->needs_input_grad(2)) d[2] = at::empty(state.sizes(), state.options());
    a.grad_x = ptr(d[0]);
    a.grad_gate = ptr(d[1]);
    a.grad_state = static_cast<float*>(ptr(d[2]));
    const Tensor ws = workspace(tgx_scan_workspace_size(&a), x);
    a.workspace = ptr(ws);
    a.workspace_bytes = ws.defined() ? ws.numel() : 0;
    check(tgx_scan_grad(&a, stream_of(x)), "tgx_scan_grad");
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
  if (state.defined()) state = state.contiguous();
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

}  // namespace

void bind_block_ops(py::module_& m) {
  m.def("gated_scan", &gated_scan, py::arg("x"), py::arg("gate"), py::arg("mask") = py::none(),
        py::arg("state") = py::none());
}

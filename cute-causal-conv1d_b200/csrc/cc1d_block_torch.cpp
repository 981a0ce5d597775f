// PyTorch binding of the recurrent-block operators: argument checks, allocation of results,
// autograd nodes, and the calls of the C ABI.  Built as the extension module causal_conv1d._block.
//
// In C++ because these calls are short: through Python and ctypes a decode step took 12 us of
// the host's time (7 here) and a small training pass of the recurrence 127 us (69 here).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "causal_conv1d_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Opt = std::optional<Tensor>;

Tensor or_none(const Opt& t) { return t.has_value() ? *t : Tensor(); }
Opt optional_of(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }

std::string shape_text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

void expect(const char* name, const Tensor& t, at::IntArrayRef shape) {
  if (t.defined() && t.sizes() != shape)
    throw py::value_error(std::string(name) + " must have shape " + shape_text(shape) + ", got " +
                          shape_text(t.sizes()));
}
void expect_dims(const char* name, const Tensor& t, int64_t n) {
  if (t.dim() != n)
    throw py::value_error(std::string(name) + " must have " + std::to_string(n) + " dimensions, got shape " +
                          shape_text(t.sizes()));
}

void one_device(std::initializer_list<const Tensor*> all) {
  const Tensor* first = nullptr;
  for (const Tensor* t : all) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) throw py::value_error("causal_conv1d needs CUDA tensors (there is no CPU implementation)");
    if (!first) first = t;
    else if (t->device() != first->device())
      throw py::value_error("all tensors must be on one device (" + first->device().str() + " vs " +
                            t->device().str() + ")");
  }
}

int32_t dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return CC1D_FLOAT32;
    case at::kHalf: return CC1D_FLOAT16;
    case at::kBFloat16: return CC1D_BFLOAT16;
    case at::kInt: return CC1D_INT32;
    case at::kLong: return CC1D_INT64;
    default: throw py::type_error(std::string("unsupported dtype ") + c10::toString(t));
  }
}

cc1d_tensor describe(const Tensor& t) {
  cc1d_tensor r = {};
  if (!t.defined()) return r;
  r.data = t.data_ptr();
  r.dtype = dtype_code(t.scalar_type());
  for (int64_t i = 0; i < t.dim() && i < 3; ++i) r.stride[i] = t.stride(i);
  return r;
}

void check(int status) {
  if (status == CC1D_OK) return;
  const std::string text = cc1d_last_error();
  switch (status) {
    case CC1D_ERR_VALUE: throw py::value_error(text);
    case CC1D_ERR_TYPE: throw py::type_error(text);
    default: throw std::runtime_error(text.empty() ? "causal_conv1d error" : text);
  }
}

// The current stream of x's device, which is current while this lives.
struct Launch {
  explicit Launch(const Tensor& x)
      : guard(x.device()), stream(c10::cuda::getCurrentCUDAStream(x.get_device()).stream()) {}
  c10::cuda::CUDAGuard guard;
  void* stream;
};

Tensor scratch(int64_t bytes, const Tensor& like) { return at::empty({bytes}, like.options().dtype(at::kByte)); }
Tensor fp32(at::IntArrayRef shape, const Tensor& like) {
  return at::empty(shape, like.options().dtype(at::kFloat));
}

// Refuses forward-mode tangents: a call that dropped one would pass for a function that does not
// depend on that input.
void no_tangents(const char* what, std::initializer_list<const Tensor*> all) {
  for (const Tensor* t : all) {
    if (!t->defined() || !t->_fw_grad(0).defined()) continue;
    py::gil_scoped_acquire gil;
    PyErr_SetString(PyExc_NotImplementedError, (std::string(what) + " has no forward-mode derivative").c_str());
    throw py::error_already_set();
  }
}

// Makes results lead to `inputs` through a node that raises `why` when a derivative is asked for.
void no_derivative(variable_list& results, const variable_list& inputs, const char* why) {
  auto node = std::make_shared<torch::autograd::Error>(why, torch::autograd::collect_next_edges(inputs));
  for (Tensor& r : results)
    if (r.defined()) {
      r = r.detach();
      torch::autograd::set_history(r, node);
    }
}
// The gradients of a node whose backward has no derivative of its own.
variable_list once(variable_list grads, const variable_list& inputs) {
  if (at::GradMode::is_enabled())
    no_derivative(grads, inputs, "trying to differentiate twice a function that was marked with once_differentiable");
  return grads;
}

// ------------------------------------------------------------------------- recurrence
// t in the layout of ref: a unit stride along the channels or along the sequence.
Tensor like_layout(const Tensor& t, const Tensor& ref) {
  if (!t.defined() || t.dim() != 3 || t.strides() == ref.strides()) return t;
  if (ref.stride(1) == 1 && t.stride(1) != 1) return t.transpose(1, 2).contiguous().transpose(1, 2);
  if (ref.stride(1) != 1 && ref.stride(2) == 1 && t.stride(2) != 1) return t.contiguous();
  return t;
}
Tensor laid_out(const Tensor& x) { return x.stride(1) != 1 && x.stride(2) != 1 ? x.contiguous() : x; }

int64_t state_rows(int64_t batch, const Tensor& seq_idx, std::initializer_list<const Tensor*> states) {
  if (!seq_idx.defined()) return batch;
  for (const Tensor* t : states)
    if (t->defined() && t->dim() > 0) return t->size(0);
  return 0;
}
int64_t chunks(int64_t seqlen) { return (seqlen + CC1D_RECURRENCE_CHUNK - 1) / CC1D_RECURRENCE_CHUNK; }

std::tuple<Tensor, Tensor, Tensor> recurrence_forward(Tensor x, Tensor gate, Tensor z, const Tensor& bias,
                                                      const Tensor& seq_idx, const Tensor& init, bool return_final,
                                                      int64_t num_sequences, bool save) {
  expect_dims("x", x, 3);
  x = laid_out(x);
  gate = like_layout(gate, x);
  z = like_layout(z, x);
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2);
  Tensor final, kept;
  if (return_final) {
    int64_t n = B;
    if (seq_idx.defined()) {
      n = init.defined() ? init.size(0) : num_sequences;
      if (n < 0)
        throw py::value_error("num_sequences is needed to return the final states of packed sequences "
                              "that have no initial states");
    }
    if (!seq_idx.defined() && L > 0) final = fp32({n, D}, x);
    else if (init.defined())  // a sequence without positions keeps its state
      final = init.detach().clone(at::MemoryFormat::Contiguous);
    else final = fp32({n, D}, x).zero_();
  }
  const int64_t n = state_rows(B, seq_idx, {&init, &final});
  expect("gate", gate, x.sizes());
  expect("z", z, x.sizes());
  expect("gate_bias", bias, {D});
  expect("seq_idx", seq_idx, {B, L});
  expect("initial_states", init, {n, D});
  expect("final_states", final, {n, D});
  one_device({&x, &gate, &z, &bias, &seq_idx, &init, &final});
  if (save) kept = fp32({B, chunks(L), D}, x);
  Tensor out = at::empty_like(x);
  cc1d_recurrence_params p = {};
  p.batch = B, p.dim = D, p.seqlen = L, p.nstates = n;
  p.x = describe(x), p.gate = describe(gate), p.z = describe(z), p.bias = describe(bias);
  p.seq_idx = describe(seq_idx), p.initial_states = describe(init), p.final_states = describe(final);
  p.out = describe(out);
  p.checkpoints = kept.defined() ? kept.data_ptr<float>() : nullptr;
  Launch launch(x);
  check(cc1d_recurrence_fwd_launch(&p, launch.stream));
  return {out, final, kept};
}

using FiveTensors = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

FiveTensors recurrence_backward(Tensor x, Tensor gate, Tensor z, const Tensor& bias, const Tensor& seq_idx,
                                const Tensor& init, const Tensor& kept, Tensor dout, const Tensor& dfinal,
                                bool want_dbias, bool want_dinit) {
  expect_dims("x", x, 3);
  x = laid_out(x);
  gate = like_layout(gate, x);
  z = like_layout(z, x);
  dout = like_layout(dout, x);
  const int64_t B = x.size(0), D = x.size(1), L = x.size(2);
  const int64_t n = state_rows(B, seq_idx, {&init, &dfinal});
  expect("gate", gate, x.sizes());
  expect("z", z, x.sizes());
  expect("gate_bias", bias, {D});
  expect("seq_idx", seq_idx, {B, L});
  expect("initial_states", init, {n, D});
  expect("dout", dout, x.sizes());
  expect("dfinal_states", dfinal, {n, D});
  expect("checkpoints", kept, {B, chunks(L), D});
  one_device({&x, &gate, &z, &bias, &seq_idx, &init, &kept, &dout, &dfinal});
  Tensor dx = at::empty_like(x), dgate = at::empty_like(x), dz, dbias, dinit;
  if (z.defined()) dz = at::empty_like(x);
  if (want_dbias) dbias = fp32({D}, x);
  if (want_dinit) {
    if (!seq_idx.defined() && L > 0) dinit = fp32({n, D}, x);
    else if (dfinal.defined())  // a sequence without positions hands its gradient through
      dinit = dfinal.clone(at::MemoryFormat::Contiguous);
    else dinit = fp32({n, D}, x).zero_();
  }
  cc1d_recurrence_params p = {};
  p.batch = B, p.dim = D, p.seqlen = L, p.nstates = n;
  p.x = describe(x), p.gate = describe(gate), p.z = describe(z), p.bias = describe(bias);
  p.seq_idx = describe(seq_idx), p.initial_states = describe(init);
  p.dout = describe(dout), p.dfinal_states = describe(dfinal);
  p.dx = describe(dx), p.dgate = describe(dgate), p.dz = describe(dz), p.dinitial_states = describe(dinit);
  p.dbias = dbias.defined() ? dbias.data_ptr<float>() : nullptr;
  p.checkpoints = kept.data_ptr<float>();
  Launch launch(x);
  const int64_t need = cc1d_recurrence_bwd_workspace_bytes(&p);
  Tensor workspace;
  if (need > 0) {
    workspace = scratch(need, x);
    p.workspace = workspace.data_ptr();
    p.workspace_bytes = need;
  }
  check(cc1d_recurrence_bwd_launch(&p, launch.stream));
  if (dbias.defined() && bias.scalar_type() != at::kFloat) dbias = dbias.to(bias.scalar_type());
  return {dx, dgate, dz, dbias, dinit};
}

struct RecurrenceNode : torch::autograd::Function<RecurrenceNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Opt& z,
                               const Opt& bias, const Opt& seq_idx, const Opt& init, bool return_final,
                               int64_t num_sequences) {
    ctx->set_materialize_grads(false);
    auto [out, final, kept] = recurrence_forward(x, gate, or_none(z), or_none(bias), or_none(seq_idx),
                                                 or_none(init), return_final, num_sequences, true);
    ctx->saved_data["dbias"] = bias.has_value() && bias->requires_grad();
    ctx->saved_data["dinit"] = init.has_value() && init->requires_grad();
    ctx->save_for_backward({x, gate, or_none(z), or_none(bias), or_none(seq_idx), or_none(init), kept});
    if (return_final) return {out, final};
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor dfinal = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dfinal.defined()) return variable_list(8);
    const auto s = ctx->get_saved_variables();
    FiveTensors g;
    {
      at::NoGradGuard no_grad;
      const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
      g = recurrence_backward(s[0], s[1], s[2], s[3], s[4], s[5], s[6], dout, dfinal,
                              ctx->saved_data["dbias"].toBool(), ctx->saved_data["dinit"].toBool());
    }
    auto& [dx, dgate, dz, dbias, dinit] = g;
    variable_list inputs(s.begin(), s.end());
    inputs.insert(inputs.end(), grads.begin(), grads.end());
    return once({dx, dgate, dz, dbias, Tensor(), dinit, Tensor(), Tensor()}, inputs);
  }
};

bool tracked(std::initializer_list<const Tensor*> all) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : all)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

std::tuple<Tensor, Tensor> recurrence(const Tensor& x, const Tensor& gate, const Opt& z, const Opt& bias,
                                      const Opt& seq_idx, const Opt& init, bool return_final,
                                      int64_t num_sequences) {
  const Tensor tz = or_none(z), tb = or_none(bias), ti = or_none(init);
  no_tangents("gated_recurrence_fn", {&x, &gate, &tz, &tb, &ti});
  if (tracked({&x, &gate, &tz, &tb, &ti})) {
    const auto r = RecurrenceNode::apply(x, gate, z, bias, seq_idx, init, return_final, num_sequences);
    return {r[0], return_final ? r[1] : Tensor()};
  }
  at::NoGradGuard no_grad;
  auto [out, final, kept] =
      recurrence_forward(x, gate, tz, tb, or_none(seq_idx), ti, return_final, num_sequences, false);
  return {out, final};
}

// State indices as the C ABI takes them.  What 32 bits do not hold is outside any pool, and has
// to stay so.
Tensor indices32(const Tensor& t) {
  if (!t.defined() || t.scalar_type() == at::kInt) return t;
  switch (t.scalar_type()) {
    case at::kLong: return t.clamp(-1, std::numeric_limits<int32_t>::max()).to(at::kInt);
    case at::kShort:
    case at::kChar:
    case at::kByte: return t.to(at::kInt);
    default: throw py::type_error(std::string("state_indices must be an integer tensor, got ") + c10::toString(t.scalar_type()));
  }
}

Tensor update_tokens(const Tensor& x, const Tensor& state, const Tensor& gate, const Tensor& z, const Tensor& bias,
                     const Tensor& wide_index) {
  at::NoGradGuard no_grad;
  const Tensor index = indices32(wide_index);
  if (x.dim() != 2) expect_dims("x", x, 3);
  expect_dims("state", state, 2);
  cc1d_recurrence_update_params p = {};
  p.batch = x.size(0), p.dim = x.size(1), p.seqlen = x.dim() == 2 ? 1 : x.size(2);
  p.nstates = index.defined() ? state.size(0) : p.batch;
  expect("gate", gate, x.sizes());
  expect("z", z, x.sizes());
  expect("gate_bias", bias, {p.dim});
  expect("state", state, {p.nstates, p.dim});
  expect("state_indices", index, {p.batch});
  one_device({&x, &gate, &z, &bias, &state, &index});
  Tensor out = at::empty_like(x);
  p.x = describe(x), p.gate = describe(gate), p.z = describe(z), p.bias = describe(bias);
  p.state = describe(state), p.state_indices = describe(index), p.out = describe(out);
  Launch launch(x);
  check(cc1d_recurrence_update_launch(&p, launch.stream));
  // a graph that saved this state notices; states made in inference mode have no version
  if (x.numel() > 0 && !state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}

Tensor recurrence_update(const Tensor& x, const Tensor& state, const Tensor& gate, const Opt& z, const Opt& bias,
                         const Opt& index) {
  const Tensor tz = or_none(z), tb = or_none(bias);
  no_tangents("gated_recurrence_update", {&x, &state, &gate, &tz, &tb});
  if (tracked({&state}))
    throw std::runtime_error("gated_recurrence_update overwrites state and has no derivative: a state that requires "
                             "grad needs torch.no_grad()");
  variable_list out = {update_tokens(x, state, gate, tz, tb, or_none(index))};
  if (tracked({&x, &gate, &tz, &tb}))
    no_derivative(out, {x, gate, tz, tb}, "gated_recurrence_update has no derivative: use gated_recurrence_fn to train");
  return out[0];
}

// --------------------------------------------------------------------------- add_norm
// t as a (rows, dim) matrix with channel stride 1.
Tensor rows_of(const Tensor& t, int64_t dim) {
  if (!t.defined()) return t;
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, dim});
  return r.stride(1) == 1 ? r : r.contiguous();
}

std::tuple<Tensor, Tensor> add_norm_forward(const Tensor& x, const Tensor& weight, const Tensor& residual,
                                            double eps, double dropout_p, const Tensor& rng,
                                            bool residual_in_fp32) {
  if (x.dim() == 0 || weight.dim() != 1 || weight.size(0) != x.size(-1))
    throw py::value_error("x and weight must have shapes (..., dim) and (dim,)");
  expect("residual", residual, x.sizes());
  if (residual.defined() && residual_in_fp32 && residual.scalar_type() != at::kFloat)
    throw py::value_error("residual must be float32 with residual_in_fp32");
  expect("rng_state", rng, {2});
  const int64_t dim = x.size(-1);
  Tensor out = at::empty_like(x, x.options(), at::MemoryFormat::Contiguous);
  const auto type = residual.defined() ? residual.scalar_type()
                    : residual_in_fp32 ? at::kFloat
                                       : x.scalar_type();
  Tensor stream = at::empty_like(out, out.options().dtype(type));
  one_device({&x, &weight, &residual, &rng});
  if (dim == 0) return {out, stream};
  const Tensor rx = rows_of(x, dim), rr = rows_of(residual, dim), ro = rows_of(out, dim), rs = rows_of(stream, dim);
  cc1d_add_norm_params p = {};
  p.rows = rx.size(0), p.dim = dim, p.eps = eps, p.dropout_p = dropout_p;
  p.x = describe(rx), p.residual = describe(rr), p.weight = describe(weight);
  p.rng_state = describe(rng), p.out = describe(ro), p.residual_out = describe(rs);
  Launch launch(x);
  check(cc1d_add_norm_fwd_launch(&p, launch.stream));
  return {out, stream};
}

using ThreeTensors = std::tuple<Tensor, Tensor, Tensor>;

// (dx, dresidual, dweight)
ThreeTensors add_norm_backward(at::ScalarType x_type, const Tensor& stream, const Tensor& weight,
                               const Tensor& dout, const Tensor& dstream, double eps, double dropout_p,
                               const Tensor& rng, bool want_dx, bool want_dres, bool want_dw) {
  const int64_t dim = stream.size(-1);
  // without dropout dx and dresidual are equal, and one tensor if their types are
  const bool shared = want_dx && want_dres && dropout_p == 0.0 && x_type == stream.scalar_type();
  Tensor dx, dres, dw;
  if (want_dx) dx = at::empty(stream.sizes(), stream.options().dtype(x_type));
  if (want_dres && !shared) dres = at::empty(stream.sizes(), stream.options());
  if (want_dw) dw = fp32({dim}, stream);
  expect("weight", weight, {dim});
  expect("dout", dout, stream.sizes());
  expect("dresidual_out", dstream, stream.sizes());
  one_device({&stream, &weight, &dout, &dstream, &rng});
  if (dim > 0) {
    const Tensor rs = rows_of(stream, dim), ry = rows_of(dout, dim), rd = rows_of(dstream, dim);
    const Tensor rx = rows_of(dx, dim), rr = rows_of(dres, dim);
    cc1d_add_norm_params p = {};
    p.rows = rs.size(0), p.dim = dim, p.eps = eps, p.dropout_p = dropout_p;
    p.x.dtype = dtype_code(x_type);
    p.weight = describe(weight), p.rng_state = describe(rng), p.residual_out = describe(rs);
    p.dout = describe(ry), p.dresidual_out = describe(rd), p.dx = describe(rx), p.dresidual = describe(rr);
    p.dweight = dw.defined() ? dw.data_ptr<float>() : nullptr;
    Launch launch(stream);
    const int64_t need = cc1d_add_norm_bwd_workspace_bytes(&p);
    Tensor workspace;
    if (need > 0) {
      workspace = scratch(need, stream);
      p.workspace = workspace.data_ptr();
      p.workspace_bytes = need;
    }
    check(cc1d_add_norm_bwd_launch(&p, launch.stream));
  }
  if (shared) dres = dx;
  if (dw.defined() && weight.scalar_type() != at::kFloat) dw = dw.to(weight.scalar_type());
  return {dx, dres, dw};
}

struct AddNormNode : torch::autograd::Function<AddNormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Opt& residual,
                               double eps, double dropout_p, const Opt& rng, bool residual_in_fp32) {
    ctx->set_materialize_grads(false);
    auto [out, stream] =
        add_norm_forward(x, weight, or_none(residual), eps, dropout_p, or_none(rng), residual_in_fp32);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["p"] = dropout_p;
    ctx->saved_data["type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["dx"] = x.requires_grad();
    ctx->saved_data["dres"] = residual.has_value() && residual->requires_grad();
    ctx->saved_data["dw"] = weight.requires_grad();
    ctx->save_for_backward({stream, weight, or_none(rng)});
    return {out, stream};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(7);
    const auto s = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    ThreeTensors g;
    {
      at::NoGradGuard no_grad;
      g = add_norm_backward(static_cast<at::ScalarType>(d["type"].toInt()), s[0], s[1], grads[0], grads[1],
                            d["eps"].toDouble(), d["p"].toDouble(), s[2], d["dx"].toBool(), d["dres"].toBool(),
                            d["dw"].toBool());
    }
    auto& [dx, dres, dw] = g;
    return once({dx, dw, dres, Tensor(), Tensor(), Tensor(), Tensor()}, {s[0], s[1], grads[0], grads[1]});
  }
};

std::tuple<Tensor, Tensor> add_norm(const Tensor& x, const Tensor& weight, const Opt& residual, double eps,
                                    double dropout_p, const Opt& rng, bool residual_in_fp32) {
  if (!(dropout_p >= 0.0 && dropout_p < 1.0)) throw py::value_error("dropout_p must be in [0, 1)");
  const Tensor tr = or_none(residual);
  no_tangents("dropout_add_rms_norm_fn", {&x, &weight, &tr});
  Tensor state = dropout_p > 0.0 ? or_none(rng) : Tensor();
  if (dropout_p > 0.0 && !state.defined())
    state = at::randint(int64_t{1} << 62, {2}, x.options().dtype(at::kLong));
  if (tracked({&x, &weight, &tr})) {
    const auto r = AddNormNode::apply(x, weight, residual, eps, dropout_p, optional_of(state), residual_in_fp32);
    return {r[0], r[1]};
  }
  at::NoGradGuard no_grad;
  return add_norm_forward(x, weight, tr, eps, dropout_p, state, residual_in_fp32);
}

}  // namespace

// Absent tensors are None on both sides.  The interpreter's lock is given up during the calls.
PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const py::call_guard<py::gil_scoped_release> unlocked;
  m.def("recurrence", &recurrence, unlocked);
  m.def(
      "recurrence_fwd",
      [](const Tensor& x, const Tensor& gate, const Opt& z, const Opt& bias, const Opt& seq_idx, const Opt& init,
         bool return_final, int64_t num_sequences, bool save) {
        at::NoGradGuard no_grad;
        return recurrence_forward(x, gate, or_none(z), or_none(bias), or_none(seq_idx), or_none(init), return_final,
                                  num_sequences, save);
      },
      unlocked);
  m.def(
      "recurrence_bwd",
      [](const Tensor& x, const Tensor& gate, const Opt& z, const Opt& bias, const Opt& seq_idx, const Opt& init,
         const Tensor& kept, const Tensor& dout, const Opt& dfinal, bool want_dbias, bool want_dinit) {
        at::NoGradGuard no_grad;
        return recurrence_backward(x, gate, or_none(z), or_none(bias), or_none(seq_idx), or_none(init), kept, dout,
                                   or_none(dfinal), want_dbias, want_dinit);
      },
      unlocked);
  m.def("recurrence_update", &recurrence_update, unlocked);
  m.def("add_norm", &add_norm, unlocked);
  m.def(
      "add_norm_fwd",
      [](const Tensor& x, const Tensor& weight, const Opt& residual, double eps, double dropout_p, const Opt& rng,
         bool residual_in_fp32) {
        at::NoGradGuard no_grad;
        return add_norm_forward(x, weight, or_none(residual), eps, dropout_p, or_none(rng), residual_in_fp32);
      },
      unlocked);
  m.def(
      "add_norm_bwd",
      [](at::ScalarType x_type, const Tensor& stream, const Tensor& weight, const Opt& dout, const Opt& dstream,
         double eps, double dropout_p, const Opt& rng, bool want_dx, bool want_dres, bool want_dw) {
        at::NoGradGuard no_grad;
        return add_norm_backward(x_type, stream, weight, or_none(dout), or_none(dstream), eps, dropout_p,
                                 or_none(rng), want_dx, want_dres, want_dw);
      },
      unlocked);
}

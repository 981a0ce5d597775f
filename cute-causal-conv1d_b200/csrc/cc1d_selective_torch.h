// PyTorch binding of the selective recurrence and its token update.
#pragma once

#include "cc1d_torch.h"

namespace {

// B or C as (batch, groups, dstate, seqlen); the user's may lack the groups.
Tensor with_groups(const char* name, const Tensor& t, int64_t dims) {
  if (t.dim() == dims) return t.unsqueeze(1);
  if (t.dim() != dims + 1)
    throw py::value_error(std::string(name) + " must have " + std::to_string(dims) + " dimensions, or " +
                          std::to_string(dims + 1) + " with groups, got shape " + shape_text(t.sizes()));
  return t;
}
// (batch, groups, dstate, seqlen) without its stride between groups, which goes beside it.
cc1d_tensor describe_grouped(const Tensor& t, int64_t* group_stride) {
  cc1d_tensor r = {};
  if (!t.defined()) return r;
  r.data = t.data_ptr();
  r.dtype = dtype_code(t.scalar_type());
  r.stride[0] = t.stride(0), r.stride[1] = t.stride(2), r.stride[2] = t.stride(3);
  *group_stride = t.stride(1);
  return r;
}
void check_rates(const Tensor& A, const Tensor& B, int64_t dim) {
  expect_dims("A", A, 2);
  if (A.size(0) != dim) expect("A", A, {dim, A.size(1)});
  if (B.size(1) < 1 || dim % B.size(1))
    throw py::value_error("dim must be a multiple of B's groups: " + std::to_string(dim) + " and " + std::to_string(B.size(1)));
}

struct SelInputs {
  Tensor x, delta, A, B, C, D, z, bias, seq_idx, init;
  bool softplus;
};

// Lays the inputs out for the kernels and checks their shapes; n: rows of the states.
void sel_prepare(SelInputs& v, int64_t n) {
  const int64_t batch = v.x.size(0), dim = v.x.size(1), L = v.x.size(2);
  v.delta = like_layout(v.delta, v.x);
  v.z = like_layout(v.z, v.x);
  expect("delta", v.delta, v.x.sizes());
  v.B = with_groups("B", v.B, 3);
  v.C = with_groups("C", v.C, 3);
  check_rates(v.A, v.B, dim);
  const int64_t N = v.A.size(1), G = v.B.size(1);
  expect("B", v.B, {batch, G, N, L});
  expect("C", v.C, {batch, G, N, L});
  expect("D", v.D, {dim});
  expect("z", v.z, v.x.sizes());
  expect("delta_bias", v.bias, {dim});
  expect("seq_idx", v.seq_idx, {batch, L});
  expect("initial_states", v.init, {n, dim, N});
}

void sel_describe(const SelInputs& v, int64_t n, cc1d_selective_params& p) {
  p.batch = v.x.size(0), p.dim = v.x.size(1), p.seqlen = v.x.size(2);
  p.dstate = v.A.size(1), p.groups = v.B.size(1), p.nstates = n, p.softplus = v.softplus;
  p.x = describe(v.x), p.delta = describe(v.delta), p.A = describe(v.A), p.D = describe(v.D);
  p.B = describe_grouped(v.B, &p.B_group_stride), p.C = describe_grouped(v.C, &p.C_group_stride);
  p.z = describe(v.z), p.bias = describe(v.bias), p.seq_idx = describe(v.seq_idx);
  p.initial_states = describe(v.init);
}

std::vector<int64_t> kept_shape(int64_t batch, int64_t L, int64_t dim, int64_t N) {
  const int64_t chunk = CC1D_SELECTIVE_CHUNK(N);
  return {batch, (L + chunk - 1) / chunk, dim, (N + 3) / 4 * 4};
}

Tensor sel_workspace(int64_t need, const Tensor& like, cc1d_selective_params& p) {
  if (need < 0) check(CC1D_ERR_VALUE);
  if (need == 0) return Tensor();
  Tensor w = scratch(need, like);
  p.workspace = w.data_ptr();
  p.workspace_bytes = need;
  return w;
}

std::tuple<Tensor, Tensor, Tensor> sel_forward(SelInputs v, bool return_final, int64_t num_sequences, bool save) {
  expect_dims("x", v.x, 3);
  expect_dims("A", v.A, 2);
  v.x = laid_out(v.x);
  const int64_t batch = v.x.size(0), dim = v.x.size(1), L = v.x.size(2), N = v.A.size(1);
  int64_t n = batch;
  if (v.seq_idx.defined()) {
    n = v.init.defined() && v.init.dim() > 0 ? v.init.size(0) : num_sequences;
    if (n < 0 && return_final)
      throw py::value_error("num_sequences is needed to return the final states of packed sequences "
                            "that have no initial states");
    n = std::max<int64_t>(n, 0);
  }
  sel_prepare(v, n);
  one_device({&v.x, &v.delta, &v.A, &v.B, &v.C, &v.D, &v.z, &v.bias, &v.seq_idx, &v.init});
  Tensor final, kept;
  if (return_final) {
    if (!v.seq_idx.defined() && L > 0) final = fp32({n, dim, N}, v.x);
    else if (v.init.defined())  // a sequence without positions keeps its state
      final = v.init.detach().clone(at::MemoryFormat::Contiguous);
    else final = fp32({n, dim, N}, v.x).zero_();
  }
  if (save)
    kept = fp32(kept_shape(batch, L, dim, N), v.x);
  Tensor out = at::empty_like(v.x);
  cc1d_selective_params p = {};
  sel_describe(v, n, p);
  p.final_states = describe(final);
  p.out = describe(out);
  p.checkpoints = kept.defined() ? kept.data_ptr<float>() : nullptr;
  Launch launch(v.x);
  const Tensor workspace = sel_workspace(cc1d_selective_fwd_workspace_bytes(&p), v.x, p);
  check(cc1d_selective_fwd_launch(&p, launch.stream));
  return {out, final, kept};
}

// dx, ddelta, dA, dB, dC, dD, dz, dbias, dinitial_states
using SelGrads = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

SelGrads sel_backward(SelInputs v, const Tensor& kept, Tensor dout, const Tensor& dfinal, bool want_dbias, bool want_dinit) {
  expect_dims("x", v.x, 3);
  expect_dims("A", v.A, 2);
  v.x = laid_out(v.x);
  dout = like_layout(dout, v.x);
  const bool grouped = v.B.dim() == 4, grouped_c = v.C.dim() == 4;
  const int64_t batch = v.x.size(0), dim = v.x.size(1), L = v.x.size(2), N = v.A.size(1);
  const int64_t n = state_rows(batch, v.seq_idx, {&v.init, &dfinal});
  sel_prepare(v, n);
  const int64_t G = v.B.size(1);
  expect("dout", dout, v.x.sizes());
  expect("dfinal_states", dfinal, {n, dim, N});
  expect("checkpoints", kept, kept_shape(batch, L, dim, N));
  one_device({&v.x, &v.delta, &v.A, &v.B, &v.C, &v.D, &v.z, &v.bias, &v.seq_idx, &v.init, &kept, &dout, &dfinal});
  Tensor dx = at::empty_like(v.x), ddelta = at::empty_like(v.x), dz, dD, dbias, dinit;
  Tensor dA = fp32({dim, N}, v.x);
  // along the states, as the sums over channels are stored, unless B lies along the sequence
  const bool along = v.B.stride(2) == 1 || v.B.stride(3) != 1;
  auto grad_of = [&]() {
    return along ? at::empty({batch, L, G, N}, v.x.options()).permute({0, 2, 3, 1})
                 : at::empty({batch, G, N, L}, v.x.options());
  };
  Tensor dB = grad_of(), dC = grad_of();
  if (v.z.defined()) dz = at::empty_like(v.x);
  if (v.D.defined()) dD = fp32({dim}, v.x);
  if (want_dbias) dbias = fp32({dim}, v.x);
  if (want_dinit) {
    if (!v.seq_idx.defined() && L > 0) dinit = fp32({n, dim, N}, v.x);
    else if (dfinal.defined())  // a sequence without positions hands its gradient through
      dinit = dfinal.clone(at::MemoryFormat::Contiguous);
    else dinit = fp32({n, dim, N}, v.x).zero_();
  }
  cc1d_selective_params p = {};
  sel_describe(v, n, p);
  p.dout = describe(dout), p.dfinal_states = describe(dfinal);
  p.dx = describe(dx), p.ddelta = describe(ddelta), p.dz = describe(dz), p.dinitial_states = describe(dinit);
  p.dB = describe_grouped(dB, &p.dB_group_stride), p.dC = describe_grouped(dC, &p.dC_group_stride);
  p.dA = dA.data_ptr<float>();
  p.dD = dD.defined() ? dD.data_ptr<float>() : nullptr;
  p.dbias = dbias.defined() ? dbias.data_ptr<float>() : nullptr;
  p.checkpoints = kept.data_ptr<float>();
  Launch launch(v.x);
  const Tensor workspace = sel_workspace(cc1d_selective_bwd_workspace_bytes(&p), v.x, p);
  check(cc1d_selective_bwd_launch(&p, launch.stream));
  auto as = [](Tensor& g, const Tensor& of) {
    if (g.defined() && of.scalar_type() != at::kFloat) g = g.to(of.scalar_type());
  };
  as(dA, v.A);
  if (dD.defined()) as(dD, v.D);
  if (dbias.defined() && v.bias.defined()) as(dbias, v.bias);
  if (!grouped) dB = dB.squeeze(1);
  if (!grouped_c) dC = dC.squeeze(1);
  return {dx, ddelta, dA, dB, dC, dD, dz, dbias, dinit};
}

struct SelectiveNode : torch::autograd::Function<SelectiveNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Tensor& A,
                               const Tensor& B, const Tensor& C, const Opt& D, const Opt& z, const Opt& bias,
                               bool softplus, const Opt& seq_idx, const Opt& init, bool return_final,
                               int64_t num_sequences) {
    ctx->set_materialize_grads(false);
    const SelInputs v = {x, delta, A, B, C, or_none(D), or_none(z), or_none(bias), or_none(seq_idx), or_none(init), softplus};
    auto [out, final, kept] = sel_forward(v, return_final, num_sequences, true);
    ctx->saved_data["softplus"] = softplus;
    ctx->saved_data["dbias"] = bias.has_value() && bias->requires_grad();
    ctx->saved_data["dinit"] = init.has_value() && init->requires_grad();
    ctx->save_for_backward({x, delta, A, B, C, v.D, v.z, v.bias, v.seq_idx, v.init, kept});
    if (return_final) return {out, final};
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor dfinal = grads.size() > 1 ? grads[1] : Tensor();
    if (!grads[0].defined() && !dfinal.defined()) return variable_list(13);
    const auto s = ctx->get_saved_variables();
    SelGrads g;
    {
      at::NoGradGuard no_grad;
      const Tensor dout = grads[0].defined() ? grads[0] : at::zeros_like(s[0]);
      g = sel_backward({s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], ctx->saved_data["softplus"].toBool()},
                       s[10], dout, dfinal, ctx->saved_data["dbias"].toBool(), ctx->saved_data["dinit"].toBool());
    }
    auto& [dx, ddelta, dA, dB, dC, dD, dz, dbias, dinit] = g;
    variable_list inputs(s.begin(), s.end());
    inputs.insert(inputs.end(), grads.begin(), grads.end());
    return once({dx, ddelta, dA, dB, dC, dD, dz, dbias, Tensor(), Tensor(), dinit, Tensor(), Tensor()}, inputs);
  }
};

std::tuple<Tensor, Tensor> selective(const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B,
                                     const Tensor& C, const Opt& D, const Opt& z, const Opt& bias, bool softplus,
                                     const Opt& seq_idx, const Opt& init, bool return_final, int64_t num_sequences) {
  const Tensor tD = or_none(D), tz = or_none(z), tb = or_none(bias), ti = or_none(init);
  no_tangents("selective_recurrence_fn", {&x, &delta, &A, &B, &C, &tD, &tz, &tb, &ti});
  if (tracked({&x, &delta, &A, &B, &C, &tD, &tz, &tb, &ti})) {
    const auto r = SelectiveNode::apply(x, delta, A, B, C, D, z, bias, softplus, seq_idx, init, return_final, num_sequences);
    return {r[0], return_final ? r[1] : Tensor()};
  }
  at::NoGradGuard no_grad;
  auto [out, final, kept] = sel_forward({x, delta, A, B, C, tD, tz, tb, or_none(seq_idx), ti, softplus}, return_final,
                                        num_sequences, false);
  return {out, final};
}

Tensor sel_update_tokens(const Tensor& x, const Tensor& state, const Tensor& delta, const Tensor& A, const Tensor& tB,
                         const Tensor& tC, const Tensor& D, const Tensor& z, const Tensor& bias, bool softplus,
                         const Tensor& wide_index) {
  at::NoGradGuard no_grad;
  const Tensor index = indices32(wide_index);
  if (x.dim() != 2) expect_dims("x", x, 3);
  expect_dims("state", state, 3);
  expect_dims("A", A, 2);
  const bool one = x.dim() == 2;
  Tensor B = with_groups("B", tB, x.dim()), C = with_groups("C", tC, x.dim());
  if (one) B = B.unsqueeze(3), C = C.unsqueeze(3);
  cc1d_selective_update_params p = {};
  p.batch = x.size(0), p.dim = x.size(1), p.seqlen = one ? 1 : x.size(2);
  p.dstate = A.size(1), p.groups = B.size(1), p.softplus = softplus;
  p.nstates = index.defined() ? state.size(0) : p.batch;
  check_rates(A, B, p.dim);
  expect("delta", delta, x.sizes());
  expect("B", B, {p.batch, p.groups, p.dstate, p.seqlen});
  expect("C", C, {p.batch, p.groups, p.dstate, p.seqlen});
  expect("D", D, {p.dim});
  expect("z", z, x.sizes());
  expect("delta_bias", bias, {p.dim});
  expect("state", state, {p.nstates, p.dim, p.dstate});
  expect("state_indices", index, {p.batch});
  one_device({&x, &delta, &A, &B, &C, &D, &z, &bias, &state, &index});
  Tensor out = at::empty_like(x);
  p.x = describe(x), p.delta = describe(delta), p.A = describe(A), p.D = describe(D), p.z = describe(z);
  p.B = describe_grouped(B, &p.B_group_stride), p.C = describe_grouped(C, &p.C_group_stride);
  p.bias = describe(bias), p.state = describe(state), p.state_indices = describe(index), p.out = describe(out);
  Launch launch(x);
  check(cc1d_selective_update_launch(&p, launch.stream));
  // a graph that saved this state notices; states made in inference mode have no version
  if (x.numel() > 0 && !state.is_inference()) torch::autograd::impl::bump_version(state);
  return out;
}

Tensor selective_update(const Tensor& x, const Tensor& state, const Tensor& delta, const Tensor& A, const Tensor& B,
                        const Tensor& C, const Opt& D, const Opt& z, const Opt& bias, bool softplus, const Opt& index) {
  const Tensor tD = or_none(D), tz = or_none(z), tb = or_none(bias);
  no_tangents("selective_recurrence_update", {&x, &state, &delta, &A, &B, &C, &tD, &tz, &tb});
  if (tracked({&state}))
    throw std::runtime_error("selective_recurrence_update overwrites state and has no derivative: a state that requires "
                             "grad needs torch.no_grad()");
  variable_list out = {sel_update_tokens(x, state, delta, A, B, C, tD, tz, tb, softplus, or_none(index))};
  if (tracked({&x, &delta, &A, &B, &C, &tD, &tz, &tb}))
    no_derivative(out, {x, delta, A, B, C, tD, tz, tb},
                  "selective_recurrence_update has no derivative: use selective_recurrence_fn to train");
  return out[0];
}

void bind_selective(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> unlocked;
  m.def("selective", &selective, unlocked);
  m.def(
      "selective_fwd",
      [](const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
         const Opt& z, const Opt& bias, bool softplus, const Opt& seq_idx, const Opt& init, bool return_final,
         int64_t num_sequences, bool save) {
        at::NoGradGuard no_grad;
        return sel_forward({x, delta, A, B, C, or_none(D), or_none(z), or_none(bias), or_none(seq_idx), or_none(init), softplus},
                           return_final, num_sequences, save);
      },
      unlocked);
  m.def(
      "selective_bwd",
      [](const Tensor& x, const Tensor& delta, const Tensor& A, const Tensor& B, const Tensor& C, const Opt& D,
         const Opt& z, const Opt& bias, bool softplus, const Opt& seq_idx, const Opt& init, const Tensor& kept,
         const Tensor& dout, const Opt& dfinal, bool want_dbias, bool want_dinit) {
        at::NoGradGuard no_grad;
        return sel_backward({x, delta, A, B, C, or_none(D), or_none(z), or_none(bias), or_none(seq_idx), or_none(init), softplus},
                            kept, dout, or_none(dfinal), want_dbias, want_dinit);
      },
      unlocked);
  m.def("selective_update", &selective_update, unlocked);
}

}  // namespace

// PyTorch binding of beam search.
#pragma once

#include "cc1d_torch.h"

namespace {

std::tuple<Tensor, Tensor, Tensor> beam_search_select(const Tensor& logits_in, const Tensor& scores, const Opt& finished_in,
                                                      std::optional<int64_t> end_token, std::optional<int64_t> num_candidates) {
  Tensor logits = logits_in, finished = or_none(finished_in);
  no_tangents("beam_search_select", {&logits, &scores});
  const bool follow = tracked({&logits, &scores});
  variable_list out;
  {
    at::NoGradGuard no_grad;
    expect_dims("logits", logits, 3);
    cc1d_beam_select_params p = {};
    p.batch = logits.size(0), p.beams = logits.size(1), p.vocab = logits.size(2);
    p.candidates = num_candidates.value_or(p.beams);
    expect("scores", scores, {p.batch, p.beams});
    expect("finished", finished, {p.batch, p.beams});
    if (finished.defined() && finished.scalar_type() != at::kBool) throw py::type_error("finished must be a bool tensor");
    if (finished.defined() && !end_token.has_value()) throw py::value_error("finished needs end_token");
    one_device({&logits, &scores, &finished});
    if (p.candidates < 1 || p.candidates > CC1D_BEAM_MAX)
      throw py::value_error("num_candidates must be in [1, min(beams * vocab, " + std::to_string(CC1D_BEAM_MAX) + ")]");
    if (logits.stride(2) != 1) logits = logits.contiguous();
    p.end_token = end_token.value_or(0);
    p.logits = describe(logits), p.scores = describe(scores);
    if (finished.defined()) {
      p.finished = static_cast<const uint8_t*>(finished.data_ptr());
      p.finished_stride[0] = finished.stride(0), p.finished_stride[1] = finished.stride(1);
    }
    const Tensor best = fp32({p.batch, p.candidates}, logits);
    const Tensor parents = at::empty({p.batch, p.candidates}, logits.options().dtype(at::kLong));
    const Tensor tokens = at::empty_like(parents);
    p.out_scores = best.data_ptr<float>();
    p.parents = parents.data_ptr<int64_t>(), p.tokens = tokens.data_ptr<int64_t>();
    Launch launch(logits);
    const int64_t need = cc1d_beam_select_workspace_bytes(&p);
    if (need < 0) check(CC1D_ERR_VALUE);
    const Tensor workspace = scratch(need, logits);
    p.workspace = workspace.data_ptr();
    p.workspace_bytes = need;
    check(cc1d_beam_select_launch(&p, launch.stream));
    out = {best, parents, tokens};
  }
  if (follow) {
    variable_list lead = {out[0]};
    no_derivative(lead, {logits_in, scores}, "beam_search_select has no derivative");
    out[0] = lead[0];
  }
  return {out[0], out[1], out[2]};
}

void beam_search_reorder(const std::vector<Tensor>& states, const Tensor& parents, const Opt& index_in) {
  at::NoGradGuard no_grad;
  const Tensor index = indices32(or_none(index_in));
  expect_dims("parents", parents, 2);
  cc1d_beam_reorder_params p = {};
  p.batch = parents.size(0), p.beams = parents.size(1), p.count = static_cast<int64_t>(states.size());
  const int64_t rows = p.batch * p.beams;
  expect("state_indices", index, {rows});
  for (const Tensor& t : states) {
    if (t.dim() < 1 || t.dim() > 4) throw py::value_error("states must have 1 to 4 dimensions, got shape " + shape_text(t.sizes()));
    if (!index.defined() && t.size(0) != rows)
      throw py::value_error("states must have " + std::to_string(rows) + " rows, one for each beam, got shape " + shape_text(t.sizes()));
  }
  one_device({&parents, &index});
  std::vector<cc1d_beam_rows> all(states.size());
  for (size_t i = 0; i < states.size(); ++i) {
    const Tensor& t = states[i];
    one_device({&parents, &t});
    cc1d_beam_rows& r = all[i];
    r.data = t.data_ptr();
    r.rows = t.size(0), r.row_stride = t.stride(0), r.element_bytes = t.element_size();
    for (int64_t k = 0; k < 3; ++k) {
      r.size[k] = k + 1 < t.dim() ? t.size(k + 1) : 1;
      r.stride[k] = k + 1 < t.dim() ? t.stride(k + 1) : 0;
    }
  }
  p.parents = describe(parents), p.state_indices = describe(index);
  p.tensors = all.data();
  Launch launch(parents);
  check(cc1d_beam_reorder_launch(&p, launch.stream));
  // graphs that saved a state notice; states made in inference mode have no version
  for (const Tensor& t : states)
    if (rows > 0 && t.numel() > 0 && !t.is_inference()) torch::autograd::impl::bump_version(t);
}

void reorder_checked(const std::vector<Tensor>& states, const Tensor& parents, const Opt& index) {
  for (const Tensor& t : states)
    if (tracked({&t}))
      throw std::runtime_error("beam_search_reorder overwrites the states and has no derivative: a state that requires grad "
                               "needs torch.no_grad()");
  beam_search_reorder(states, parents, index);
}

void bind_beam_search(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> unlocked;
  m.def("beam_select", &beam_search_select, unlocked);
  m.def("beam_reorder", &reorder_checked, unlocked);
}

}  // namespace

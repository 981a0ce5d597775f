// extern "C" launchers of beam search.  Argument checks happen here, before any launch;
// include/causal_conv1d_b200.h states the contract.
#include <algorithm>

#include "cc1d_beam_launch.h"
#include "cc1d_check.h"

namespace cc1d {
namespace {

cc1d_status check_select(const cc1d_beam_select_params* p, BeamSelectArgs* a) {
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  if (!sizes_ok(p->batch, p->beams, p->vocab)) return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (p->beams < 1 || p->beams > CC1D_BEAM_MAX) return fail(CC1D_ERR_VALUE, "beams must be in [1, %d]", CC1D_BEAM_MAX);
  if (p->vocab < 1) return fail(CC1D_ERR_VALUE, "vocab must be >= 1");
  if (p->candidates < 1 || p->candidates > CC1D_BEAM_MAX || p->candidates > p->beams * p->vocab)
    return fail(CC1D_ERR_VALUE, "candidates must be in [1, min(beams * vocab, %d)]", CC1D_BEAM_MAX);
  if (!is_float(p->logits.dtype)) return fail(CC1D_ERR_TYPE, "logits must be float32, float16 or bfloat16");
  CC1D_FP32(p->scores, "scores");
  if (p->finished && (p->end_token < 0 || p->end_token >= p->vocab))
    return fail(CC1D_ERR_VALUE, "end_token must be in [0, vocab)");
  if (p->vocab > 1 && p->logits.stride[2] != 1) return fail(CC1D_ERR_VALUE, "logits must have unit stride along the vocabulary");
  if (p->batch > 0) {
    CC1D_REQUIRE(p->logits, "logits");
    CC1D_REQUIRE(p->scores, "scores");
    if (!p->out_scores || !p->parents || !p->tokens) return fail(CC1D_ERR_VALUE, "out_scores, parents and tokens are required");
  }
  *a = BeamSelectArgs{};
  a->batch = p->batch;
  a->beams = p->beams;
  a->vocab = p->vocab;
  a->candidates = p->candidates;
  a->logits = p->logits.data;
  a->logits_s0 = p->logits.stride[0];
  a->logits_s1 = p->logits.stride[1];
  a->scores = static_cast<const float*>(p->scores.data);
  a->scores_s0 = p->scores.stride[0];
  a->scores_s1 = p->scores.stride[1];
  a->finished = p->finished;
  a->finished_s0 = p->finished_stride[0];
  a->finished_s1 = p->finished_stride[1];
  a->end_token = p->end_token;
  a->out_scores = p->out_scores;
  a->parents = p->parents;
  a->tokens = p->tokens;
  // As many CTAs as run at a time, but no part so short that joining the parts' lists takes longer
  // than it saves: 1024 elements for each candidate.  512 rows of 128000 take 53 us in one part and
  // 61 in two.  Parts of 2048, 1024 n and 2048 n elements: 4 rows of 32000, n = 4: 12.3, 11.8, 11.9 us;
  // 16 rows of 128000, n = 32: 44.3, 23.9, 25.3; 8 rows of one request, n = 16: 38.7, 21.8, 21.6.
  const int64_t rows = p->batch * p->beams, want = rows > 0 ? kBeamCtas * sm_count() / rows : 1;
  const int64_t least = std::max<int64_t>(2048, 1024 * p->candidates);
  a->parts = std::max<int64_t>(1, std::min(want, (p->vocab + least - 1) / least));
  a->part = (p->vocab + a->parts - 1) / a->parts;
  a->part = (a->part + 7) / 8 * 8;
  a->parts = (p->vocab + a->part - 1) / a->part;
  if (rows * a->parts > kMax31) return fail(CC1D_ERR_VALUE, "batch * beams is too large");
  return CC1D_OK;
}

int64_t select_bytes(const BeamSelectArgs& a) { return a.batch * a.beams * a.parts * 8 * (a.candidates + 1); }

// A tensor's rows in the fewest dimensions and the widest units that its layout allows.
cc1d_status describe_rows(const cc1d_beam_rows& r, int64_t most_unit, BeamRows* t) {
  const int64_t e = r.element_bytes;
  if (e != 1 && e != 2 && e != 4 && e != 8 && e != 16) return fail(CC1D_ERR_VALUE, "element_bytes must be 1, 2, 4, 8 or 16");
  if (!sizes_ok(r.rows, 1, 1) || !sizes_ok(r.size[0], r.size[1], r.size[2]))
    return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  *t = BeamRows{};
  const int64_t total = r.size[0] * r.size[1] * r.size[2];
  if (total == 0 || r.rows == 0) return CC1D_OK;
  if (!r.data) return fail(CC1D_ERR_VALUE, "data is required");
  struct Dim { int64_t size, step; } d[4];
  int n = 0;
  for (int i = 0; i < 3; ++i)
    if (r.size[i] > 1) d[n++] = {r.size[i], r.stride[i] * e};
  const auto by_step = [](const Dim& x, const Dim& y) { return x.step < y.step; };
  // Rows and elements are apart: threads write them side by side.
  Dim all[4];
  std::copy(d, d + n, all);
  int m = n;
  if (r.rows > 1) all[m++] = {r.rows, r.row_stride * e};
  std::sort(all, all + m, by_step);
  for (int64_t i = 0, reach = e; i < m; reach += all[i].step * (all[i].size - 1), ++i)  // up to the last element
    if (all[i].step < reach) return fail(CC1D_ERR_VALUE, "the states' elements must not overlap");
  std::sort(d, d + n, by_step);
  // an element is a run of bytes; runs that follow one another are one
  int64_t run = e;
  int first = 0;
  while (first < n && d[first].step == run) run *= d[first++].size;
  int64_t unit = most_unit;
  const auto fits = [&](uint64_t bytes) { while (bytes % static_cast<uint64_t>(unit)) unit /= 2; };
  fits(run);
  fits(reinterpret_cast<uintptr_t>(r.data));
  if (r.rows > 1) fits(r.row_stride * e);
  for (int i = first; i < n; ++i) fits(d[i].step);
  // the run in its units, then what is left: four dimensions where three are of elements wider than a unit
  Dim out[4] = {{1, 0}, {1, 0}, {1, 0}, {1, 0}};
  const int outer = n - first == 3 && run == unit ? 0 : 1;
  if (outer) out[0] = {run / unit, unit};
  std::copy(d + first, d + n, out + outer);
  t->data = static_cast<char*>(r.data);
  t->rows = r.rows;
  t->row_bytes = r.row_stride * e;
  t->columns = total * e / unit;
  t->size0 = out[0].size, t->step0 = out[0].step;
  t->size1 = out[1].size, t->step1 = out[1].step;
  t->size2 = out[2].size, t->step2 = out[2].step;
  t->step3 = out[3].step;
  t->unit = static_cast<int32_t>(unit);
  const int64_t blocks = (t->columns + kThreads - 1) / kThreads;
  if (blocks > kMax31) return fail(CC1D_ERR_VALUE, "a row is too large");
  t->blocks = static_cast<int32_t>(blocks);
  return CC1D_OK;
}

}  // namespace
}  // namespace cc1d

using namespace cc1d;

extern "C" {

int64_t cc1d_beam_select_workspace_bytes(const cc1d_beam_select_params* p) {
  set_last_error("");
  BeamSelectArgs a;
  return check_select(p, &a) == CC1D_OK ? select_bytes(a) : -1;
}

cc1d_status cc1d_beam_select_launch(const cc1d_beam_select_params* p, void* stream) {
  set_last_error("");
  BeamSelectArgs a;
  cc1d_status st = check_select(p, &a);
  if (st != CC1D_OK || a.batch == 0) return st;
  if ((st = workspace_ok(p->workspace, p->workspace_bytes, select_bytes(a))) != CC1D_OK) return st;
  a.best = static_cast<int2*>(p->workspace);
  a.sums = reinterpret_cast<float2*>(a.best + a.batch * a.beams * a.parts * a.candidates);
  return launched(beam_select(a, p->logits.dtype, static_cast<cudaStream_t>(stream)), "beam selection launch", 2);
}

cc1d_status cc1d_beam_reorder_launch(const cc1d_beam_reorder_params* p, void* stream) {
  set_last_error("");
  if (!p) return fail(CC1D_ERR_VALUE, "params is NULL");
  if (!sizes_ok(p->batch, p->beams, 1) || p->count < 0) return fail(CC1D_ERR_VALUE, "sizes must be >= 0 and below 2^31");
  if (p->beams < 1 || p->beams > CC1D_BEAM_MAX) return fail(CC1D_ERR_VALUE, "beams must be in [1, %d]", CC1D_BEAM_MAX);
  if (p->parents.dtype != CC1D_INT32 && p->parents.dtype != CC1D_INT64) return fail(CC1D_ERR_TYPE, "parents must be int32 or int64");
  if (p->state_indices.data && p->state_indices.dtype != CC1D_INT32) return fail(CC1D_ERR_TYPE, "state_indices must be int32");
  if (p->batch * p->beams > kMax31) return fail(CC1D_ERR_VALUE, "batch * beams is too large");
  if (p->batch == 0 || p->count == 0) return CC1D_OK;
  CC1D_REQUIRE(p->parents, "parents");
  if (!p->tensors) return fail(CC1D_ERR_VALUE, "tensors is required");
  BeamReorderArgs a = {};
  a.batch = p->batch;
  a.beams = p->beams;
  a.parents = p->parents.data;
  a.parents_s0 = p->parents.stride[0];
  a.parents_s1 = p->parents.stride[1];
  a.wide_parents = p->parents.dtype == CC1D_INT64;
  a.indices = static_cast<const int32_t*>(p->state_indices.data);
  a.indices_stride = p->state_indices.stride[0];
  const auto full = [](const cc1d_beam_rows& r) { return r.rows && r.size[0] && r.size[1] && r.size[2]; };
  for (int64_t i = 0; i < p->count; ++i)
    for (int64_t j = 0; j < i; ++j)
      if (p->tensors[i].data == p->tensors[j].data && full(p->tensors[i]) && full(p->tensors[j]))
        return fail(CC1D_ERR_VALUE, "two of the states start at one place");
  // every tensor is checked before the first one changes
  for (int pass = 0; pass < 2; ++pass) {
    a.count = 0;
    int64_t ctas = 0;
    for (int64_t i = 0; i < p->count; ++i) {
      BeamRows& t = a.t[a.count];
      const cc1d_beam_rows& r = p->tensors[i];
      const cc1d_status st = describe_rows(r, beam_most_unit(p->beams), &t);
      if (st != CC1D_OK) return st;
      if (!a.indices && r.rows != p->batch * p->beams)
        return fail(CC1D_ERR_VALUE, "without state_indices there is one row for each beam");
      const int64_t more = p->batch * t.blocks;
      if (more > kMax31) return fail(CC1D_ERR_VALUE, "the states are too large for one launch");
      if (t.columns > 0) {
        ++a.count;
        ctas += more;
      }
      const bool full = a.count == kBeamTensors || ctas > kMax31 / 2 || i + 1 == p->count;
      if (!full || a.count == 0) continue;
      if (pass == 1) {
        if (ctas > kMax31) return fail(CC1D_ERR_VALUE, "the states are too large for one launch");
        const cc1d_status done = launched(beam_reorder(a, ctas, static_cast<cudaStream_t>(stream)), "beam reordering launch", 1);
        if (done != CC1D_OK) return done;
      } else if (ctas > kMax31) {
        return fail(CC1D_ERR_VALUE, "the states are too large for one launch");
      }
      a.count = 0;
      ctas = 0;
    }
  }
  return CC1D_OK;
}

}  // extern "C"

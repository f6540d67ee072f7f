// fold_norm.hip -- pccl_hip_fold_norm, pccl_hip_fold_norm_backward: argument checks, team shape, how the rows are cut
// for the sums over rows, dispatch to the typed kernels.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "fold_norm_kernel.h"

using namespace pccl_dev;
using pccl_host::fail;

namespace {

// Rows of a launch: a grid times its lanes must fit 32 bits, 2^22 - 1 workgroups of 1024.
constexpr unsigned kLaunchRows = 1u << 21;

// One pack of 16 bytes a lane while a workgroup holds the row, else two (binary32 beyond 8192 columns: four): a wavefront where one is
// enough (no barrier in its sums), beyond a workgroup of as many as the width fills.  (binary32 up to 4096 columns with one pack
// and not two: forward 8192 x 2048 53 -> 48 us, 4096 x 4096 4 -> 2 95 -> 90; backward, where it is what leaves room for a row ahead,
// 4985 x 1025 50 -> 41, 16384 x 1024 83 -> 80; backward rows of 257 to 512 columns, where two packs still are one wavefront's, lose:
// 50000 x 400 98 -> 101, 30000 x 300 with biases 59 -> 69.)
NormShape shape_of(long width, int dtype, bool one_pack) {
  const int elems = dtype == PCCL_F32 && one_pack && width <= 4096 ? 4 : width <= 8192 ? 8 : 16;
  return {(int)((width + elems * kWave - 1) / (elems * kWave)) * kWave, elems};
}

bool row_dtype(int dtype) { return dtype == PCCL_F32 || dtype == PCCL_BF16 || dtype == PCCL_F16; }

struct Checker {
  int es, ps;  // element sizes of rows and parameters
  long rows, width;
  int rc = PCCL_OK;

  void aligned(const void *p, int size, const char *what) {
    if (rc == PCCL_OK && (uintptr_t)p % size) rc = fail(PCCL_ERR_MISALIGNED, "%s (%p) not %d-byte aligned", what, p, size);
  }
  void in(const void *p, long stride, const char *what) {
    aligned(p, es, what);
    if (rc == PCCL_OK && p && stride < 0) rc = fail(PCCL_ERR_INVALID_ARG, "stride %ld of %s below 0", stride, what);
  }
  void out(const void *p, long stride, const char *what, long n_rows, int size) {
    aligned(p, size, what);
    if (rc == PCCL_OK && p && n_rows > 1 && stride < width)
      rc = fail(PCCL_ERR_INVALID_ARG, "stride %ld of %s below the width %ld: its rows would overlap", stride, what, width);
  }
};

long gate_row_count(long rows, long gate_rows) { return rows / gate_rows + (rows % gate_rows != 0); }  // (gate_rows may be anything from 1)

// What both directions look at.
int check_desc(const pccl_fold_norm_desc *d, Checker *c) {
  if (!d) return fail(PCCL_ERR_INVALID_ARG, "fold_norm: description is null");
  if (!row_dtype(d->dtype)) return fail(PCCL_ERR_UNSUPPORTED, "fold_norm: rows of dtype code %d", d->dtype);
  if (d->param_dtype != d->dtype && d->param_dtype != PCCL_F32)
    return fail(PCCL_ERR_UNSUPPORTED, "fold_norm: parameters of dtype code %d for rows of %d", d->param_dtype, d->dtype);
  for (int kind : {d->post_kind, d->pre_kind})
    if (kind < PCCL_NORM_NONE || kind > PCCL_NORM_LAYER) return fail(PCCL_ERR_UNSUPPORTED, "unknown norm kind %d", kind);
  if (d->rows < 0 || d->rows > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "rows %ld outside [0, 2^31)", d->rows);
  if (d->width < 1 || d->width > PCCL_NORM_MAX_WIDTH)
    return fail(PCCL_ERR_INVALID_ARG, "width %ld outside [1, %d]", d->width, PCCL_NORM_MAX_WIDTH);
  if (d->n_in < 1 || d->n_in > PCCL_MAX_INPUTS) return fail(PCCL_ERR_INVALID_ARG, "n_in %d outside [1, 8]", d->n_in);
  if (d->n_out < 0 || d->n_out > PCCL_MAX_OUTPUTS) return fail(PCCL_ERR_INVALID_ARG, "n_out %d outside [0, 8]", d->n_out);
  // (comparisons that a NaN fails)
  if (d->post_kind != PCCL_NORM_NONE && !(d->post_eps >= FLT_MIN && d->post_eps <= FLT_MAX))
    return fail(PCCL_ERR_INVALID_ARG, "post_eps %g is no positive normal number", (double)d->post_eps);
  if (d->pre_kind != PCCL_NORM_NONE && !(d->pre_eps >= FLT_MIN && d->pre_eps <= FLT_MAX))
    return fail(PCCL_ERR_INVALID_ARG, "pre_eps %g is no positive normal number", (double)d->pre_eps);
  for (float f : {d->weight_offset, d->residual_scale, d->block_scale})
    if (!std::isfinite(f)) return fail(PCCL_ERR_INVALID_ARG, "weight_offset and scales must be finite");
  if (d->post_kind == PCCL_NORM_NONE && (d->post_weight || d->post_bias))
    return fail(PCCL_ERR_INVALID_ARG, "weight or bias of a post norm that there is not");
  if (d->pre_kind == PCCL_NORM_NONE && (d->pre_weight || d->pre_bias))
    return fail(PCCL_ERR_INVALID_ARG, "weight or bias of a pre norm that there is not");
  if (d->gate && d->gate_rows < 1) return fail(PCCL_ERR_INVALID_ARG, "gate_rows %ld < 1 with a gate", d->gate_rows);
  if (d->gate && d->gate_stride < 0) return fail(PCCL_ERR_INVALID_ARG, "stride %ld of the gate below 0", d->gate_stride);
  *c = Checker{pccl_host::pccl_dtype_bytes(d->dtype), pccl_host::pccl_dtype_bytes(d->param_dtype), d->rows, d->width};
  c->aligned(d->post_weight, c->ps, "post_weight");
  c->aligned(d->post_bias, c->ps, "post_bias");
  c->aligned(d->pre_weight, c->ps, "pre_weight");
  c->aligned(d->pre_bias, c->ps, "pre_bias");
  c->aligned(d->gate, c->ps, "gate");
  for (int k = 0; k < d->n_in; ++k) {
    if (!d->ins[k] && d->rows) return fail(PCCL_ERR_INVALID_ARG, "input %d is null", k);
    c->in(d->ins[k], d->in_stride, "an input");
  }
  return c->rc;
}

void fill(const pccl_fold_norm_desc *d, const Checker &c, NormArgs *a) {
  a->post_kind = d->post_kind;
  a->pre_kind = d->pre_kind;
  a->post_eps = d->post_eps;
  a->pre_eps = d->pre_eps;
  a->weight_offset = d->weight_offset;
  a->residual_scale = d->residual_scale;
  a->block_scale = d->block_scale;
  a->per_width = (float)(1.0 / (double)d->width);
  a->width = (int)d->width;
  a->n_in = d->n_in;
  a->n_out = d->n_out;
  a->rows = (unsigned)d->rows;
  a->post_weight = (const char *)d->post_weight;
  a->post_bias = (const char *)d->post_bias;
  a->pre_weight = (const char *)d->pre_weight;
  a->pre_bias = (const char *)d->pre_bias;
  a->gate = d->rows ? (const char *)d->gate : nullptr;  // (without rows it has none either)
  a->gate_bytes = d->gate_stride * c.ps;
  a->gate_rows = (unsigned)(d->gate ? std::min(d->gate_rows, std::max(1l, d->rows)) : std::max(1l, d->rows));
  for (int k = 0; k < d->n_in; ++k) a->ins[k] = (const char *)d->ins[k];
  a->in_bytes = d->in_stride * c.es;
}

// Calls f<DT, PF32>() for the row and parameter types.
template <class F>
hipError_t with_types(int dtype, int param_dtype, F &&f) {
  typedef std::integral_constant<bool, true> Wide;
  typedef std::integral_constant<bool, false> Same;
  const bool wide = param_dtype == PCCL_F32;
  if (dtype == PCCL_F32) return f(std::integral_constant<int, PCCL_F32>{}, Wide{});
  if (dtype == PCCL_BF16) return wide ? f(std::integral_constant<int, PCCL_BF16>{}, Wide{}) : f(std::integral_constant<int, PCCL_BF16>{}, Same{});
  return wide ? f(std::integral_constant<int, PCCL_F16>{}, Wide{}) : f(std::integral_constant<int, PCCL_F16>{}, Same{});
}

int launched(hipError_t e, const char *what) {
  return e == hipSuccess ? PCCL_OK : fail(PCCL_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
}

// Shape of the backward pass.  Beyond 8192 columns always sixteen wavefronts, some of which
// then have one pack, others two: a compute unit holds no second team (bf16 4096 x 9216 138 -> 124 us, 2048 x 12288 93 -> 89).
NormShape backward_shape(long width, int dtype) {
  if (width > 8192) return {kMostLanes, 16};
  return shape_of(width, dtype, width <= 4 * kWave || width > 8 * kWave);
}

// How the backward pass cuts the rows (see BackwardArgs).
struct Cut {
  unsigned groups, strips, n_strips, n_teams;
};

// Teams that fill the chip while there are few gate rows: enough for several wavefronts on every SIMD, few enough that writing and joining
// their sums (4 rows of binary32 a team) stays small beside the rows themselves.  Strips are of one gate row and `most / groups` is
// rounded down, so with about as many gate rows as teams the longest team has up to twice an even share: bf16 16384 x 8192 with no
// or one gate row 271 us, 149 391, 298 457; f32 16384 x 1024 80, with 820 119.  Twelve wavefronts a compute unit (or the team that
// passes twelve) where teams have their next row on its way, sixteen where they wait for it: without a row ahead, and with
// gate rows so short that a strip has none (12 against 16: 8000 x 1536 bf16, 8 gate rows, 51 -> 48 us, 100000 x 200 f32 96 -> 88;
// 8192 x 2048 with a gate a row 65 -> 68).
Cut cut_of(long rows, long width, long gate_rows, int dtype) {
  const NormShape n = backward_shape(width, dtype);
  const bool ahead = n.elems * pccl_host::pccl_dtype_bytes(dtype) == 16;
  const long per = gate_rows >= 1 ? std::min(gate_rows, std::max(1l, rows)) : std::max(1l, rows);
  int teams = kMostLanes / n.lanes;
  if (ahead && per >= 4) teams = std::min(teams, (12 * kWave + n.lanes - 1) / n.lanes);
  const long most = (long)pccl_host::compute_units() * teams;
  Cut c;
  c.groups = (unsigned)std::max(1l, gate_row_count(rows, per));
  c.strips = (unsigned)std::max(1l, std::min(per, most / (long)c.groups));
  c.n_strips = c.groups * c.strips;
  c.n_teams = (unsigned)std::min<long>(c.n_strips, most);
  return c;
}

long sums_bytes(const Cut &c, long width) { return (long)c.n_teams * 4 * width * 4; }
long gate_sums_bytes(const Cut &c, long width) { return c.strips > 1 ? (long)c.n_strips * width * 4 : 0; }

}  // namespace

extern "C" int pccl_hip_fold_norm(const pccl_fold_norm_desc *d, void *stream) {
  pccl_host::clear_error();
  Checker c;
  int rc = check_desc(d, &c);
  if (rc != PCCL_OK) return rc;
  c.in(d->residual, d->residual_stride, "the residual");
  c.out(d->residual_out, d->residual_out_stride, "residual_out", d->rows, c.es);
  c.out(d->folded, d->folded_stride, "folded", d->rows, c.es);
  for (int j = 0; j < d->n_out; ++j) {
    if (!d->outs[j] && d->rows) return fail(PCCL_ERR_INVALID_ARG, "output %d is null", j);
    c.out(d->outs[j], d->out_stride, "an output", d->rows, c.es);
  }
  if (c.rc != PCCL_OK) return c.rc;
  rc = pccl_host::check_stream(&stream);
  if (rc != PCCL_OK) return rc;
  if (d->rows == 0) return PCCL_OK;
  ForwardArgs a;
  memset(&a, 0, sizeof(a));
  fill(d, c, &a);
  a.residual = (const char *)d->residual;
  a.residual_bytes = d->residual_stride * c.es;
  a.residual_out = (char *)d->residual_out;
  a.residual_out_bytes = d->residual_out_stride * c.es;
  a.folded = (char *)d->folded;
  a.folded_bytes = d->folded_stride * c.es;
  for (int j = 0; j < d->n_out; ++j) a.outs[j] = (char *)d->outs[j];
  a.out_bytes = d->out_stride * c.es;
  const NormShape n = shape_of(d->width, d->dtype, true);
  // many inputs beyond the Infinity Cache are read non-temporally (8 -> 8 bf16 at 2048 x 8192 122 -> 120 us, 8 -> 1 at 4096 x 4096 67 -> 64;
  // one or two lose: 1 -> 1 at 16384 x 8192 178 -> 184, and so does what is in that cache: f32 2 -> 2 at 4096 x 2048 38 -> 45)
  const bool stream_in = (d->n_in + d->n_out + 2) * d->rows * d->width * c.es > (256l << 20);
  for (long lo = 0; lo < d->rows; lo += kLaunchRows) {
    a.row0 = (unsigned)lo;
    a.rows = (unsigned)std::min<long>(d->rows, lo + kLaunchRows);
    rc = launched(with_types(d->dtype, d->param_dtype, [&](auto t, auto p) {
      return launch_fold_norm<decltype(t)::value, decltype(p)::value>(n, stream_in, (hipStream_t)stream, a);
    }), "fold_norm");
    if (rc != PCCL_OK) return rc;
  }
  return PCCL_OK;
}

extern "C" int pccl_hip_fold_norm_workspace(long rows, long width, long gate_rows, long *bytes) {
  pccl_host::clear_error();
  if (!bytes) return fail(PCCL_ERR_INVALID_ARG, "pccl_hip_fold_norm_workspace: bytes is null");
  *bytes = 0;
  if (rows < 0 || rows > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "rows %ld outside [0, 2^31)", rows);
  if (width < 1 || width > PCCL_NORM_MAX_WIDTH) return fail(PCCL_ERR_INVALID_ARG, "width %ld outside [1, %d]", width, PCCL_NORM_MAX_WIDTH);
  if (gate_rows < 0) return fail(PCCL_ERR_INVALID_ARG, "gate_rows %ld < 0", gate_rows);
  for (int dtype : {PCCL_F32, PCCL_BF16}) {  // whichever type the rows have
    const Cut c = cut_of(rows, width, gate_rows, dtype);
    *bytes = std::max(*bytes, sums_bytes(c, width) + (gate_rows ? gate_sums_bytes(c, width) : 0));
  }
  return PCCL_OK;
}

extern "C" int pccl_hip_fold_norm_backward(const pccl_fold_norm_desc *d, const pccl_fold_norm_grads *g, void *stream) {
  pccl_host::clear_error();
  Checker c;
  int rc = check_desc(d, &c);
  if (rc != PCCL_OK) return rc;
  if (!g) return fail(PCCL_ERR_INVALID_ARG, "fold_norm_backward: gradients are null");
  if (g->n_grad_in < 0 || g->n_grad_in > PCCL_MAX_INPUTS) return fail(PCCL_ERR_INVALID_ARG, "n_grad_in %d outside [0, 8]", g->n_grad_in);
  const bool reads_r = d->pre_kind != PCCL_NORM_NONE && d->n_out > 0;
  if (reads_r && !d->residual_out && d->rows) return fail(PCCL_ERR_INVALID_ARG, "residual_out (the forward's r) is null");
  if (reads_r) c.in(d->residual_out, d->residual_out_stride, "residual_out");
  for (int j = 0; j < d->n_out; ++j) {
    if (!g->grad_outs[j] && d->rows) return fail(PCCL_ERR_INVALID_ARG, "gradient %d of the outputs is null", j);
    c.in(g->grad_outs[j], g->grad_out_stride, "a gradient of the outputs");
  }
  c.in(g->grad_residual_out, g->grad_residual_out_stride, "grad_residual_out");
  for (int k = 0; k < g->n_grad_in; ++k) {
    if (!g->grad_ins[k] && d->rows) return fail(PCCL_ERR_INVALID_ARG, "gradient %d of the inputs is null", k);
    c.out(g->grad_ins[k], g->grad_in_stride, "a gradient of the inputs", d->rows, c.es);
  }
  c.out(g->grad_residual, g->grad_residual_stride, "grad_residual", d->rows, c.es);
  if (g->grad_gate && g->grad_gate == d->gate) return fail(PCCL_ERR_INVALID_ARG, "grad_gate is the gate itself");
  if (g->grad_gate && !d->gate) return fail(PCCL_ERR_INVALID_ARG, "gradient of a gate that there is not");
  if (g->grad_gate) c.out(g->grad_gate, g->grad_gate_stride, "grad_gate", gate_row_count(d->rows, d->gate_rows), c.ps);
  const bool has[4] = {d->post_weight != nullptr, d->post_bias != nullptr, d->pre_weight != nullptr, d->pre_bias != nullptr};
  void *const to[4] = {g->grad_post_weight, g->grad_post_bias, g->grad_pre_weight, g->grad_pre_bias};
  static const char *const names[4] = {"grad_post_weight", "grad_post_bias", "grad_pre_weight", "grad_pre_bias"};
  bool any = false;
  for (int k = 0; k < 4; ++k) {
    if (to[k] && !has[k]) return fail(PCCL_ERR_INVALID_ARG, "%s of a parameter that there is not", names[k]);
    c.aligned(to[k], c.ps, names[k]);
    any = any || to[k];
  }
  if (c.rc != PCCL_OK) return c.rc;
  const bool single = d->n_in == 1 && d->n_out <= 1;
  const NormShape shape = backward_shape(d->width, d->dtype);
  const Cut cut = cut_of(d->rows, d->width, d->gate ? d->gate_rows : 0, d->dtype);
  const bool joined_gate = g->grad_gate && cut.strips > 1;
  const long need = (any ? sums_bytes(cut, d->width) : 0) + (joined_gate ? gate_sums_bytes(cut, d->width) : 0);
  if (need) {
    if (!g->workspace || g->workspace_bytes < need)
      return fail(PCCL_ERR_INVALID_ARG, "workspace of %ld bytes, %ld are needed", g->workspace ? g->workspace_bytes : 0, need);
    if ((uintptr_t)g->workspace % 16) return fail(PCCL_ERR_MISALIGNED, "workspace (%p) not 16-byte aligned", g->workspace);
  }
  rc = pccl_host::check_stream(&stream);
  if (rc != PCCL_OK) return rc;
  if (d->rows == 0 && !any) return PCCL_OK;

  BackwardArgs a;
  memset(&a, 0, sizeof(a));
  fill(d, c, &a);
  a.residual_out = (const char *)d->residual_out;
  a.residual_out_bytes = d->residual_out_stride * c.es;
  a.grad_residual_out = (const char *)g->grad_residual_out;
  a.grad_residual_out_bytes = g->grad_residual_out_stride * c.es;
  for (int j = 0; j < d->n_out; ++j) a.grad_outs[j] = (const char *)g->grad_outs[j];
  a.grad_out_bytes = g->grad_out_stride * c.es;
  a.grad_residual = (char *)g->grad_residual;
  a.grad_residual_bytes = g->grad_residual_stride * c.es;
  for (int k = 0; k < g->n_grad_in; ++k) a.grad_ins[k] = (char *)g->grad_ins[k];
  a.n_grad_in = g->n_grad_in;
  a.grad_in_bytes = g->grad_in_stride * c.es;
  a.n_strips = cut.n_strips;
  a.strips = cut.strips;
  a.n_teams = cut.n_teams;
  a.sums = (float *)g->workspace;
  a.gate_sums = joined_gate ? (float *)((char *)g->workspace + (any ? sums_bytes(cut, d->width) : 0)) : nullptr;
  a.grad_gate = d->rows ? (char *)g->grad_gate : nullptr;
  a.grad_gate_bytes = g->grad_gate_stride * c.ps;
  for (int k = 0; k < 4; ++k) a.want_sums[k] = to[k] != nullptr;
  // beyond the Infinity Cache (bf16 16384 x 8192 306 -> 281 us, 32768 x 1024 88 -> 83; inside: 8192 x 2048 with a gate a row 84.5 -> 86)
  const bool stream_in = (4 + g->n_grad_in) * d->rows * d->width * c.es > (256l << 20);
  const bool bias = to[1] || to[3] || (g->grad_gate && d->post_bias);
  rc = launched(with_types(d->dtype, d->param_dtype, [&](auto t, auto p) {
    return launch_fold_norm_backward<decltype(t)::value, decltype(p)::value>(shape, single, bias, stream_in, (hipStream_t)stream, a);
  }), "fold_norm_backward");
  if (rc != PCCL_OK || !need) return rc;

  SumsArgs j;
  memset(&j, 0, sizeof(j));
  j.sums = a.sums;
  j.gate_sums = a.gate_sums;
  for (int k = 0; k < 4; ++k) {
    j.out[k] = (char *)to[k];
    if (to[k]) j.listed[j.n_listed++] = k;
  }
  j.width = (int)d->width;
  j.n_partial = shape.workgroups(cut.n_teams);
  j.strips = cut.strips;
  j.grad_gate = a.grad_gate;
  j.grad_gate_bytes = a.grad_gate_bytes;
  const unsigned grid_y = j.n_listed + (joined_gate ? cut.groups : 0);
  return launched(with_types(d->dtype, d->param_dtype, [&](auto t, auto p) {
    return launch_fold_norm_sums<decltype(t)::value, decltype(p)::value>(grid_y, (hipStream_t)stream, j);
  }), "fold_norm_backward (sums over rows)");
}

// fold_norm_kernel.h -- the forward and backward kernels of the norms around a block (pccl_hip_fold_norm,
// pccl_hip_fold_norm_backward) and their typed launchers.
#pragma once

#include <type_traits>

#include "fold_norm_device.h"

namespace pccl_dev {

struct NormArgs {  // both directions
  int post_kind, pre_kind;
  float post_eps, pre_eps, weight_offset, residual_scale, block_scale;
  float per_width;  // 1 / width
  int width, n_in, n_out;
  unsigned rows;
  const char *post_weight, *post_bias, *pre_weight, *pre_bias, *gate;
  long gate_bytes;     // from one gate row to the next
  unsigned gate_rows;  // rows that share one (all of them where there is no gate)
  const char *ins[PCCL_MAX_INPUTS];
  long in_bytes;
};

struct ForwardArgs : NormArgs {
  unsigned row0;  // the launch's first row
  const char *residual;
  char *residual_out, *folded, *outs[PCCL_MAX_OUTPUTS];
  long residual_bytes, residual_out_bytes, folded_bytes, out_bytes;
};

// v's norm over the team in place: v - mean (layer) and one over the spread; masked elements stay 0.
template <class R, int LANES, int E>
__device__ __forceinline__ float standardise(const Share<R, LANES, E> &s, TeamSums<LANES> &sums, int kind, float per_width, float eps,
                                             float (&v)[E]) {
  float t[1];
  if (kind == PCCL_NORM_LAYER) {  // two passes over the registers: no cancellation between E[v^2] and E[v]^2
    t[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) t[0] += v[i];
    sums(t);
    const float mean = t[0] * per_width;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] -= mean;
    s.mask(v);
  }
  t[0] = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) t[0] = __builtin_fmaf(v[i], v[i], t[0]);
  sums(t);
  return one_over_spread(t[0], per_width, eps);
}

// x = v * rstd * (weight + offset) + bias
template <class R, bool PF32, int LANES, int E>
__device__ __forceinline__ void scale_and_shift(const Share<R, LANES, E> &s, const ParamShare<R, PF32, LANES, E> &weight, bool has_weight,
                                                float offset, const char *bias, float rstd, float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= rstd;
  if (has_weight) {
    float w[E];
    weight.up(w);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= w[i] + offset;
  }
  if (bias) {
    ParamShare<R, PF32, LANES, E> b;
    float x[E];
    b.load(s, bias);
    b.up(x);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] += x[i];
  }
}

// Lanes of a workgroup: teams of one wavefront come four to a workgroup (they meet at no barrier), others have their own.
constexpr int team_block(int lanes) { return lanes == kWave ? kBlock : lanes; }

template <int DT, bool PF32, int LANES, int E, int AT_ONCE>
__global__ void __launch_bounds__(team_block(LANES)) fold_norm_kernel(const ForwardArgs a) {
  typedef RowType<DT> R;
  constexpr int kTeams = team_block(LANES) / LANES;
  __shared__ float words[2][LANES / kWave][kSumsAtOnce];
  const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / LANES);
  const unsigned row = a.row0 + blockIdx.x * kTeams + team;
  if (row >= a.rows) return;  // a whole team; teams of one wavefront meet at no barrier
  const Share<R, LANES, E> s((int)threadIdx.x % LANES, a.width);
  TeamSums<LANES> sums{words, 0};

  ParamShare<R, PF32, LANES, E> post_weight, pre_weight, gate;
  u32x4 x[E / R::kPack];
  float v[E];
  if (a.residual) s.load(a.residual + (long)row * a.residual_bytes, x);
  fold_rows<R, LANES, E, AT_ONCE>(s, a.ins, a.n_in, (long)row * a.in_bytes, v);
  s.mask(v);
  // parameters come from the caches; asked for in front of the sums that they are waited for behind
  if (a.post_weight) post_weight.load(s, a.post_weight);
  if (a.gate) gate.load(s, a.gate + (row / a.gate_rows) * a.gate_bytes);
  if (a.pre_weight) pre_weight.load(s, a.pre_weight);

  if (a.folded) s.store(a.folded + (long)row * a.folded_bytes, v);
  if (a.post_kind != PCCL_NORM_NONE) {
    const float rstd = standardise(s, sums, a.post_kind, a.per_width, a.post_eps, v);
    scale_and_shift(s, post_weight, a.post_weight != nullptr, a.weight_offset, a.post_bias, rstd, v);
  }
  if (a.gate) {
    float g[E];
    gate.up(g);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= g[i];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= a.block_scale;
  if (a.residual) {
    float f[E];
    s.up(x, f);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = __builtin_fmaf(a.residual_scale, f[i], v[i]);
  }
  s.mask(v);  // (a bias and x have put values there)
  if (a.residual_out) s.store(a.residual_out + (long)row * a.residual_out_bytes, v);
  if (a.n_out == 0) return;
  if (a.pre_kind != PCCL_NORM_NONE) {
    const float rstd = standardise(s, sums, a.pre_kind, a.per_width, a.pre_eps, v);
    scale_and_shift(s, pre_weight, a.pre_weight != nullptr, a.weight_offset, a.pre_bias, rstd, v);
  }
  const long at = (long)row * a.out_bytes;
#pragma unroll
  for (int j = 0; j < PCCL_MAX_OUTPUTS; ++j)
    if (j < a.n_out) s.store(a.outs[j] + at, v);
}

// ---- backward ----------------------------------------------------------------------------------------
// The rows are cut into strips that lie within the rows of one gate row (strips of a gate row: `strips`, of
// `strip_rows` rows; without a gate all rows count as one gate row's), and a team goes through consecutive
// strips.  Lane l holds the same columns of every row, so the sums over rows stay in its registers; a team
// writes those of the parameters once, at its end, and those of the gate at the end of each strip.
struct BackwardArgs : NormArgs {
  const char *residual_out, *grad_residual_out, *grad_outs[PCCL_MAX_OUTPUTS];
  char *grad_residual, *grad_ins[PCCL_MAX_INPUTS];
  int n_grad_in;
  long residual_out_bytes, grad_residual_out_bytes, grad_out_bytes, grad_residual_bytes, grad_in_bytes;
  unsigned n_strips, strip_rows;  // in all; rows of one
  unsigned strips;                // of one gate row
  unsigned n_teams;
  // what the sums over rows go to: [n_teams][4][width] (post weight, post bias, pre weight, pre bias) and, with
  // several strips a gate row, [n_strips][width]; with one strip the gate's own gradient
  float *sums, *gate_sums;
  char *grad_gate;
  long grad_gate_bytes;
  bool want_sums[4];
};

template <class R, int LANES, int E>
__device__ __forceinline__ void store_sums(const Share<R, LANES, E> &s, float *row, const float (&x)[E]) {
#pragma unroll
  for (int j = 0; j < E / R::kPack; ++j) {
    if (s.lo[j] == 0) {
#pragma unroll
      for (int w = 0; w < R::kPack / 4; ++w)
        *(u32x4_a4 *)(row + s.off[j] + 4 * w) = RowType<PCCL_F32>::down(x + j * R::kPack + 4 * w);
    } else if (s.has(j)) {
#pragma unroll
      for (int i = 0; i < R::kPack; ++i)
        if (i >= s.lo[j]) row[s.off[j] + i] = x[j * R::kPack + i];
    }
  }
}

// x = the lane's share of a row of sums, or zeros
template <class R, int LANES, int E>
__device__ __forceinline__ void load_sums(const Share<R, LANES, E> &s, const float *row, bool there, float (&x)[E]) {
#pragma unroll
  for (int j = 0; j < E / R::kPack; ++j)
#pragma unroll
    for (int i = 0; i < R::kPack; ++i) x[j * R::kPack + i] = there && i >= s.lo[j] ? row[s.off[j] + i] : 0.0f;
}

// What a row of the backward pass sums over the team: a parameter's column sums come from two products per element.
// With yhat, rhat the standardised y and r:
//   s1 = sum dr * yhat, s0 = sum dr over the rows of a strip, which share a gate row g, give
//     the gate's gradient            c * ((w + o) * s1 + b * s0)        (c block_scale, w, o, b the post norm's)
//     the post norm's                weight c * g * s1, bias c * g * s0
//   p1 = sum dh * rhat, p0 = sum dh  weight and bias of the pre norm
// so that a row costs one fused multiply-add a column for each, and gate and weight are met once a strip.
//
// One team's registers hold the row (packed), the row after it on its way (SINGLE: one y and at most one dh, so that
// four streams are read), wpre = w + o of the pre norm, cgw = c * g * (w + o) of the post norm, and the sums.
// BIAS: some bias's gradient or a gate behind a biased norm is asked for (s0 and p0 are kept).
//
// The arguments (18 addresses and 12 strides) are read again from the argument segment wherever a row needs them: held
// in scalar registers over the loop they spill into vector registers, and those are what is short here.
typedef const BackwardArgs __attribute__((address_space(4))) *BackwardArgsAt;
__device__ __forceinline__ BackwardArgsAt read_again(BackwardArgsAt p) {
  asm volatile("" : "+s"(p));  // (no instruction: the compiler may not know what it points to any more)
  return p;
}
template <class R, int LANES, int E>
struct BackRow {
  u32x4 y[E / R::kPack], r[E / R::kPack], dh[E / R::kPack], dr[E / R::kPack];
};

template <int DT, bool PF32, int LANES, int E, bool SINGLE, bool BIAS>
__global__ void __launch_bounds__(team_block(LANES), 4) fold_norm_backward_kernel(const BackwardArgs) {
  typedef RowType<DT> R;
  typedef Share<R, LANES, E> S;
  typedef ParamShare<R, PF32, LANES, E> P;
  constexpr int kTeams = team_block(LANES) / LANES;
  constexpr int kFold = 4;  // gradients in flight together; more cost registers
  const BackwardArgsAt args = (BackwardArgsAt)__builtin_amdgcn_kernarg_segment_ptr();  // (the one argument stands at its start)
  const BackwardArgsAt a0 = args;
  __shared__ float words[2][LANES / kWave][kSumsAtOnce];
  const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / LANES);
  const unsigned t = blockIdx.x * kTeams + team;
  if (t >= a0->n_teams) return;
  const S s((int)threadIdx.x % LANES, a0->width);
  TeamSums<LANES> sums{words, 0};
  const bool post = a0->post_kind != PCCL_NORM_NONE, outs = a0->n_out > 0, pre = a0->pre_kind != PCCL_NORM_NONE && outs;
  const bool post_layer = a0->post_kind == PCCL_NORM_LAYER, pre_layer = pre && a0->pre_kind == PCCL_NORM_LAYER;
  const float per_width = a0->per_width;

  float wpre[E], p1[E], p0[BIAS ? E : 1];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    wpre[i] = 1.0f;
    p1[i] = 0.0f;
    if constexpr (BIAS) p0[i] = 0.0f;
  }
  if (a0->pre_weight) {
    P w;
    w.load(s, a0->pre_weight);
    w.up(wpre);
#pragma unroll
    for (int i = 0; i < E; ++i) wpre[i] += a0->weight_offset;
  }

  auto load_row = [&](unsigned long row, BackRow<R, LANES, E> &x) {
    const BackwardArgsAt a = read_again(args);
    if (a->grad_residual_out) s.load(a->grad_residual_out + row * a->grad_residual_out_bytes, x.dr);
    if (pre) s.load(a->residual_out + row * a->residual_out_bytes, x.r);
    if constexpr (SINGLE) {
      if (outs) s.load(a->grad_outs[0] + row * a->grad_out_bytes, x.dh);
      s.load(a->ins[0] + row * a->in_bytes, x.y);
    }
  };

  const unsigned first = (unsigned)((unsigned long)a0->n_strips * t / a0->n_teams);
  const unsigned end = (unsigned)((unsigned long)a0->n_strips * (t + 1) / a0->n_teams);
  for (unsigned strip = first; strip < end; ++strip) {
    const BackwardArgsAt a1 = read_again(args);
    const unsigned group = strip / a1->strips;
    // (the last gate row may have fewer rows than gate_rows, and its last strips then none: 64 bits, and no row)
    const unsigned long group_row = (unsigned long)group * a1->gate_rows;
    const unsigned long begin = group_row + (unsigned long)(strip - group * a1->strips) * a1->strip_rows;
    unsigned long stop = begin + a1->strip_rows;
    if (stop > group_row + a1->gate_rows) stop = group_row + a1->gate_rows;
    if (stop > a1->rows) stop = a1->rows;

    BackRow<R, LANES, E> next;
    if (SINGLE && begin < stop) load_row(begin, next);
    float cgw[E], s1[E], s0[BIAS ? E : 1];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      cgw[i] = a1->block_scale;
      s1[i] = 0.0f;
      if constexpr (BIAS) s0[i] = 0.0f;
    }
    if (a1->gate) {
      P g;
      float f[E];
      g.load(s, a1->gate + group * a1->gate_bytes);
      g.up(f);
#pragma unroll
      for (int i = 0; i < E; ++i) cgw[i] *= f[i];
    }
    if (a1->post_weight) {
      P w;
      float f[E];
      w.load(s, a1->post_weight);
      w.up(f);
#pragma unroll
      for (int i = 0; i < E; ++i) cgw[i] *= f[i] + a1->weight_offset;
    }

    for (unsigned long row = begin; row < stop; ++row) {
      BackRow<R, LANES, E> now;
      float y[E], dh[E], r[E];
      if constexpr (SINGLE) {
        now = next;
        if (row + 1 < stop) load_row(row + 1, next);
        s.up(now.y, y);
        if (outs) s.up(now.dh, dh);
      } else {
        load_row(row, now);
        const BackwardArgsAt a = read_again(args);
        if (outs) fold_rows<R, LANES, E, kFold>(s, a->grad_outs, a->n_out, row * a->grad_out_bytes, dh);
        fold_rows<R, LANES, E, kFold>(s, a->ins, a->n_in, row * a->in_bytes, y);
      }
      s.mask(y);
      if (outs) s.mask(dh);
      if (pre) {
        s.up(now.r, r);
        s.mask(r);
      }
      // both norms' statistics, and what the pre norm's backward sums, in one go over the team (two with a layer norm)
      if (post_layer || pre_layer) {
        float m[2] = {0.0f, 0.0f};
        if (post_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) m[0] += y[i];
        }
        if (pre_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) m[1] += r[i];
        }
        sums(m);
        if (post_layer) {
          const float mean = m[0] * per_width;
#pragma unroll
          for (int i = 0; i < E; ++i) y[i] -= mean;
          s.mask(y);
        }
        if (pre_layer) {
          const float mean = m[1] * per_width;
#pragma unroll
          for (int i = 0; i < E; ++i) r[i] -= mean;
          s.mask(r);
        }
      }
      float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // squares of y, squares of r, dh * w * r, dh * w
      if (post) {
#pragma unroll
        for (int i = 0; i < E; ++i) q[0] = __builtin_fmaf(y[i], y[i], q[0]);
      }
      if (pre) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          q[1] = __builtin_fmaf(r[i], r[i], q[1]);
          q[2] = __builtin_fmaf(dh[i] * wpre[i], r[i], q[2]);
        }
        if (pre_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) q[3] = __builtin_fmaf(dh[i], wpre[i], q[3]);
        }
      }
      if (post || pre) sums(q);
      const BackwardArgsAt a = read_again(args);
      float dr[E];
      if (a->grad_residual_out) {
        s.up(now.dr, dr);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] = 0.0f;
      }
      if (pre) {
        // dr += rstd * (d - rhat * mean(d * rhat) - mean(d)), d = dh * w
        const float rstd = one_over_spread(q[1], per_width, a->pre_eps);
        const float along = -(rstd * rstd * rstd) * (q[2] * per_width);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          p1[i] = __builtin_fmaf(dh[i], r[i] * rstd, p1[i]);
          dr[i] = __builtin_fmaf(dh[i] * wpre[i], rstd, __builtin_fmaf(r[i], along, dr[i]));
        }
        if (pre_layer) {
          const float mean = rstd * (q[3] * per_width);
#pragma unroll
          for (int i = 0; i < E; ++i) dr[i] -= mean;
        }
        if constexpr (BIAS) {
#pragma unroll
          for (int i = 0; i < E; ++i) p0[i] += dh[i];
        }
      } else if (outs) {
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] += dh[i];
      }
      s.mask(dr);
      if (a->grad_residual) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = a->residual_scale * dr[i];
        s.store(a->grad_residual + row * a->grad_residual_bytes, x);
      }
      if (post) {
        const float rstd = one_over_spread(q[0], per_width, a->post_eps);
        float m[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
          y[i] *= rstd;
          s1[i] = __builtin_fmaf(dr[i], y[i], s1[i]);
        }
        if constexpr (BIAS) {
#pragma unroll
          for (int i = 0; i < E; ++i) s0[i] += dr[i];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          dr[i] *= cgw[i];
          m[0] = __builtin_fmaf(dr[i], y[i], m[0]);
        }
        if (post_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) m[1] += dr[i];
        }
        sums(m);
        const float along = -rstd * (m[0] * per_width), mean = -rstd * (m[1] * per_width);
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] = __builtin_fmaf(dr[i], rstd, __builtin_fmaf(y[i], along, mean));
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          s1[i] = __builtin_fmaf(dr[i], y[i], s1[i]);
          dr[i] *= cgw[i];
        }
      }
      const unsigned long at = row * a->grad_in_bytes;
#pragma unroll 1
      for (int j = 0; j < a->n_grad_in; ++j) s.store(a->grad_ins[j] + at, dr);
    }

    // the strip's sums: to the gate's gradient or its workspace, and, times the gate, to the team's
    const BackwardArgsAt a = read_again(args);
    if (a->grad_gate) {
      float x[E];
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = s1[i] * a->block_scale;
      if (a->post_weight) {
        P w;
        float f[E];
        w.load(s, a->post_weight);
        w.up(f);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] *= f[i] + a->weight_offset;
      }
      if constexpr (BIAS) {
        if (a->post_bias) {
          P b;
          float f[E];
          b.load(s, a->post_bias);
          b.up(f);
#pragma unroll
          for (int i = 0; i < E; ++i) x[i] = __builtin_fmaf(f[i] * a->block_scale, s0[i], x[i]);
        }
      }
      if (a->gate_sums) {
        store_sums(s, a->gate_sums + (unsigned long)strip * a->width, x);
      } else if constexpr (PF32 && R::kBytes == 2) {
        store_sums(s, (float *)(a->grad_gate + group * a->grad_gate_bytes), x);
      } else {
        s.store(a->grad_gate + group * a->grad_gate_bytes, x);
      }
    }
    if (a->want_sums[0] || a->want_sums[1]) {
      float f[E];
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = a->block_scale;
      if (a->gate) {
        P g;
        float x[E];
        g.load(s, a->gate + group * a->gate_bytes);
        g.up(x);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] *= x[i];
      }
      // a team of several strips adds to what it wrote itself (each lane to its own columns)
      float *mine = a->sums + (unsigned long)t * 4 * a->width;
      float x[E];
      if (a->want_sums[0]) {
        load_sums(s, mine, strip != first, x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = __builtin_fmaf(f[i], s1[i], x[i]);
        store_sums(s, mine, x);
      }
      if constexpr (BIAS) {
        if (a->want_sums[1]) {
          load_sums(s, mine + a->width, strip != first, x);
#pragma unroll
          for (int i = 0; i < E; ++i) x[i] = __builtin_fmaf(f[i], s0[i], x[i]);
          store_sums(s, mine + a->width, x);
        }
      }
    }
  }
  float *mine = a0->sums + (unsigned long)t * 4 * a0->width;
  if (a0->want_sums[2]) store_sums(s, mine + 2 * a0->width, p1);
  if constexpr (BIAS) {
    if (a0->want_sums[3]) store_sums(s, mine + 3 * a0->width, p0);
  }
}

// Joins the teams' sums: a workgroup adds 64 columns of one parameter's (or one gate row's) partial rows, 16 wavefronts
// every sixteenth row each, then the 16 in order.
struct SumsArgs {
  const float *sums, *gate_sums;
  char *out[4];      // by parameter, null: not wanted
  int listed[4];     // which parameters blockIdx.y = 0 .. n_listed - 1 stand for
  int n_listed, width;
  unsigned n_teams, strips;
  char *grad_gate;   // blockIdx.y = n_listed + gate row
  long grad_gate_bytes;
};
constexpr int kJoinWaves = 16;

template <int DT, bool PF32>
__global__ void __launch_bounds__(kJoinWaves * kWave) fold_norm_sums_kernel(const SumsArgs a) {
  __shared__ float part[kJoinWaves][kWave];
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave;
  const int column = (int)blockIdx.x * kWave + lane;
  const bool of_gate = (int)blockIdx.y >= a.n_listed;
  const int which = of_gate ? 0 : a.listed[blockIdx.y];
  const long group = (int)blockIdx.y - a.n_listed;
  const float *from = of_gate ? a.gate_sums + group * a.strips * a.width : a.sums + (long)which * a.width;
  const long step = of_gate ? a.width : 4l * a.width;
  const unsigned n = of_gate ? a.strips : a.n_teams;
  float t = 0.0f;
  if (column < a.width) {
#pragma unroll 8
    for (unsigned k = wave; k < n; k += kJoinWaves) t += from[k * step + column];
  }
  part[wave][lane] = t;
  __syncthreads();
  if (wave != 0 || column >= a.width) return;
#pragma unroll
  for (int k = 1; k < kJoinWaves; ++k) t += part[k][lane];
  char *to = of_gate ? a.grad_gate + group * a.grad_gate_bytes : a.out[which];
  if constexpr (PF32) ((float *)to)[column] = t;
  else ((typename RowType<DT>::elem_t *)to)[column] = RowType<DT>::down1(t);
}

// ---- launchers, one translation unit per pair of types ---------------------------------------------------
// Lanes of a team and elements a lane, by width.
struct NormShape {
  int lanes, elems;
};

template <class F>
inline bool with_norm_shape(NormShape n, F &&f) {
#define PCCL_NORM_SHAPE(L, E)                                                              \
  if (n.lanes == L && n.elems == E) {                                                      \
    f(std::integral_constant<int, L>{}, std::integral_constant<int, E>{});                 \
    return true;                                                                           \
  }
  PCCL_NORM_SHAPE(64, 8)
  PCCL_NORM_SHAPE(128, 8)
  PCCL_NORM_SHAPE(256, 8)
  PCCL_NORM_SHAPE(512, 8)
  PCCL_NORM_SHAPE(1024, 8)
  PCCL_NORM_SHAPE(1024, 16)
#undef PCCL_NORM_SHAPE
  return false;
}

template <int DT, bool PF32> hipError_t launch_fold_norm(NormShape n, hipStream_t stream, const ForwardArgs &a);
template <int DT, bool PF32> hipError_t launch_fold_norm_backward(NormShape n, bool bias, hipStream_t stream, const BackwardArgs &a);
template <int DT, bool PF32> hipError_t launch_fold_norm_sums(unsigned grid_y, hipStream_t stream, const SumsArgs &a);

#define PCCL_DEFINE_FOLD_NORM(DT, PF32)                                                                                     \
  template <> hipError_t launch_fold_norm<DT, PF32>(NormShape n, hipStream_t stream, const ForwardArgs &a) {                \
    with_norm_shape(n, [&](auto l, auto e) {                                                                                \
      constexpr int L = decltype(l)::value, E = decltype(e)::value, kTeams = team_block(L) / L;                             \
      const unsigned grid = (a.rows - a.row0 + kTeams - 1) / kTeams;                                                        \
      if (a.n_in <= 2) hipLaunchKernelGGL((fold_norm_kernel<DT, PF32, L, E, 2>), dim3(grid), dim3(team_block(L)), 0, stream, a); \
      else hipLaunchKernelGGL((fold_norm_kernel<DT, PF32, L, E, 8>), dim3(grid), dim3(team_block(L)), 0, stream, a);        \
    });                                                                                                                     \
    return hipGetLastError();                                                                                               \
  }                                                                                                                         \
  template <> hipError_t launch_fold_norm_backward<DT, PF32>(NormShape n, bool bias, hipStream_t stream, const BackwardArgs &a) { \
    with_norm_shape(n, [&](auto l, auto e) {                                                                                \
      constexpr int L = decltype(l)::value, E = decltype(e)::value, kTeams = team_block(L) / L;                             \
      const unsigned grid = (a.n_teams + kTeams - 1) / kTeams;                                                              \
      const bool single = a.n_in == 1 && a.n_out <= 1;                                                                      \
      auto run = [&](auto sg, auto b) {                                                                                     \
        hipLaunchKernelGGL((fold_norm_backward_kernel<DT, PF32, L, E, decltype(sg)::value, decltype(b)::value>), dim3(grid), \
                           dim3(team_block(L)), 0, stream, a);                                                              \
      };                                                                                                                    \
      if (single) bias ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});                \
      else bias ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});                     \
    });                                                                                                                     \
    return hipGetLastError();                                                                                               \
  }                                                                                                                         \
  template <> hipError_t launch_fold_norm_sums<DT, PF32>(unsigned grid_y, hipStream_t stream, const SumsArgs &a) {          \
    hipLaunchKernelGGL((fold_norm_sums_kernel<DT, PF32>), dim3((a.width + kWave - 1) / kWave, grid_y), dim3(kJoinWaves * kWave), 0, stream, a); \
    return hipGetLastError();                                                                                               \
  }

}  // namespace pccl_dev

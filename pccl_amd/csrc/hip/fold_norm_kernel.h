// fold_norm_kernel.h -- the forward and backward kernels of the norms around a block (pccl_hip_fold_norm,
// pccl_hip_fold_norm_backward) and their typed launchers.
#pragma once

#include <type_traits>

#include "fold_norm_device.h"
#include "reduce_copy_kernel.h"

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

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct ForwardArgs : NormArgs {
  unsigned row0;  // the launch's first row
  const char *residual;
  char *residual_out, *folded, *outs[PCCL_MAX_OUTPUTS];
  long residual_bytes, residual_out_bytes, folded_bytes, out_bytes;
};

// v's norm over the team in place: v - mean (layer) and one over the spread; masked elements stay 0.
template <class R, bool TEAM, int E>
__device__ __forceinline__ float standardise(const Share<R, TEAM, E> &s, TeamSums<TEAM> &sums, int kind, float per_width, float eps,
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
template <class R, bool PF32, bool TEAM, int E>
__device__ __forceinline__ void scale_and_shift(const Share<R, TEAM, E> &s, const ParamShare<R, PF32, TEAM, E> &weight, bool has_weight,
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
    ParamShare<R, PF32, TEAM, E> b;
    float x[E];
    b.load(s, bias);
    b.up(x);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] += x[i];
  }
}

constexpr int kMostLanes = kMostWaves * kWave;
constexpr int team_block(bool team) { return team ? kMostLanes : kBlock; }  // lanes of a workgroup, at most

// STREAM: the inputs are read non-temporally.  Workgroups of the launch take rows in the order of rotated_chunk, for the reasons given
// there (8 -> 8 bf16 at 2048 x 8192 119 -> 111 us, 8 -> 1 at 4096 x 4096 64 -> 61, narrow rows unchanged).
template <int DT, bool PF32, bool TEAM, int E, int AT_ONCE, bool STREAM>
__global__ void __launch_bounds__(team_block(TEAM)) fold_norm_kernel(const ForwardArgs a) {
  typedef RowType<DT> R;
  constexpr int kTeams = TEAM ? 1 : kBlock / kWave;
  __shared__ float words[2][TEAM ? kMostWaves : 1][kSumsAtOnce];
  const int team = TEAM ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lanes = TEAM ? (int)blockDim.x : kWave;
  const unsigned row = a.row0 + rotated_chunk(blockIdx.x, gridDim.x) * kTeams + team;
  if (row >= a.rows) return;  // a whole team; teams of one wavefront meet at no barrier
  const Share<R, TEAM, E> s((int)threadIdx.x % lanes, lanes, a.width);
  TeamSums<TEAM> sums{words, lanes / kWave, 0};

  ParamShare<R, PF32, TEAM, E> post_weight, pre_weight, gate;
  u32x4 x[E / R::kPack];
  float v[E];
  if (a.residual) s.template load<STREAM>(a.residual + (long)row * a.residual_bytes, x);
  fold_rows<STREAM, AT_ONCE, 0>(s, a.ins, a.n_in, (long)row * a.in_bytes, v);
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
// The rows of one gate row (without a gate: all rows) are dealt out to `strips` strips, row i to strip i mod strips, and a
// team goes through consecutive strips.  Teams at work at the same time so read neighbouring rows: a window that moves through
// memory in address order.  (With strips of consecutive rows the teams stood a power of two of bytes apart, bf16
// 16384 x 8192 at 64 rows a team 1 MiB, and fell on the same channels.)  Lane l holds the same columns of every row, so the sums over
// rows stay in its registers; a team writes those of the parameters once, at its end, and those of the gate at the end of each strip.
struct BackwardArgs : NormArgs {
  const char *residual_out, *grad_residual_out, *grad_outs[PCCL_MAX_OUTPUTS];
  char *grad_residual, *grad_ins[PCCL_MAX_INPUTS];
  int n_grad_in;
  long residual_out_bytes, grad_residual_out_bytes, grad_out_bytes, grad_residual_bytes, grad_in_bytes;
  unsigned n_strips;              // in all
  unsigned strips;                // of one gate row
  unsigned n_teams;
  // what the sums over rows go to: [n_teams][4][width] (post weight, post bias, pre weight, pre bias) and, with
  // several strips a gate row, [n_strips][width]; with one strip the gate's own gradient
  float *sums, *gate_sums;
  char *grad_gate;
  long grad_gate_bytes;
  bool want_sums[4];
};

// A lane's share of a row of sums in the workspace (binary32).
template <class R, bool TEAM, int E>
__device__ __forceinline__ void store_sums(const Share<R, TEAM, E> &s, float *row, const float (&x)[E]) {
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

template <class R, bool TEAM, int E>
__device__ __forceinline__ void load_sums(const Share<R, TEAM, E> &s, const float *row, float (&x)[E]) {
#pragma unroll
  for (int j = 0; j < E / R::kPack; ++j) {
    float *to = x + j * R::kPack;
    if (s.lo[j] == 0) {
#pragma unroll
      for (int w = 0; w < R::kPack / 4; ++w) {
        const u32x4 v = *(const u32x4_a4 *)(row + s.off[j] + 4 * w);
#pragma unroll
        for (int i = 0; i < 4; ++i) to[4 * w + i] = as_f32(v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < R::kPack; ++i) to[i] = i >= s.lo[j] ? row[s.off[j] + i] : 0.0f;
    }
  }
}

// Sums over rows that a lane keeps for its columns, in registers or (IN_LDS) in the workgroup's LDS, four columns to a 16-byte
// word, words of one lane `step` apart.
template <int E, bool IN_LDS>
struct Columns {
  float x[IN_LDS ? 1 : E];
  f32x4 *at;
  int step;

  __device__ __forceinline__ void zero() {
    if constexpr (IN_LDS) {
#pragma unroll
      for (int k = 0; k < E / 4; ++k) at[k * step] = f32x4{0, 0, 0, 0};
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = 0.0f;
    }
  }
  // += a * b, element by element: N columns from `first` on
  template <int N>
  __device__ __forceinline__ void add(int first, const float (&a)[N], const float (&b)[N]) {
    if constexpr (IN_LDS) {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) {
        f32x4 &to = at[(first / 4 + k) * step];
        f32x4 v = to;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(a[4 * k + i], b[4 * k + i], v[i]);
        to = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[first + i] = __builtin_fmaf(a[i], b[i], x[first + i]);
    }
  }
  __device__ __forceinline__ void get(float (&to)[E]) const {
#pragma unroll
    for (int i = 0; i < E; ++i) to[i] = IN_LDS ? at[i / 4 * step][i % 4] : x[i];
  }
};

// What a row of the backward pass sums over the team: a parameter's column sums come from two products per element.
// With yhat, rhat the standardised y and r:
//   s1 = sum dr * yhat, s0 = sum dr over the rows of a strip, which share a gate row g, give
//     the gate's gradient            c * ((w + o) * s1 + b * s0)        (c block_scale, w, o, b the post norm's)
//     the post norm's                weight c * g * s1, bias c * g * s0
//   p1 = sum dh * rhat, p0 = sum dh  weight and bias of the pre norm
// so that a row costs one fused multiply-add a column for each, and gate and weight are met once a strip.
//
// One team's registers hold the row (packed), wpre = w + o of the pre norm, cgw = c * g * (w + o) of the post norm, s1 and p1.
// Rows of one pack a lane (16-bit up to 8192 columns, binary32 up to 4096) have room for the row after it, on its way; of several partial
// y or dh (SINGLE: there are none) the first, the others are loaded four at once when the row's turn comes (bf16 4096 x 4096 of two
// gradients 58 -> 55 us).  binary32 with two packs spilled with it (8192 x 2048 87 -> 84 us without, 78 with one pack and the row ahead).  s0 and p0 and the post norm's sums over a team's strips stay in LDS.
// Rows beyond 8192 columns (E = 16) have sixteen wavefronts, all of a compute unit's registers, 8 for each column.  They go pack by pack,
// in order: what a pack needs of wpre and cgw is read from the caches as it comes, y, r and dh stay as they were loaded and are unpacked and
// centred anew in each phase, s1 and p1 are in LDS, the post norm's sums over strips go to the workspace and back, and only 16-bit rows
// without BIAS have the next row on its way.  (2048 x 16384 bf16 113 -> 106 us, with biases 226 -> 128; f32 1024 x 16384 148 -> 105, with
// biases 212 -> 186; the floors are 59.)  They still spill, less than the whole row at once did: without BIAS 0 to 2 of 128 registers
// for one gradient of 16-bit rows, 0 or 1 for several, 12 and 43 for binary32; with BIAS 18 to 22, 57 to 77, 98 and 132.  Of the narrower
// instances only some with BIAS spill: two packs of binary32 5 (a team) and 13 (one wavefront), one wavefront of 16-bit rows 4 to 8.
// BIAS: some bias's gradient or a gate behind a biased norm is asked for (s0 and p0 are kept).
// STREAM: rows are read non-temporally.
//
// The arguments (18 addresses and 12 strides) are read again from the argument segment wherever a row needs them: held
// in scalar registers over the loop they spill into vector registers, and those are what is short here.
typedef const BackwardArgs __attribute__((address_space(4))) *BackwardArgsAt;
__device__ __forceinline__ BackwardArgsAt read_again(BackwardArgsAt p) {
  asm volatile("" : "+s"(p));  // (no instruction: the compiler may not know what it points to any more)
  return p;
}
template <class R, int E>
struct BackRow {
  u32x4 y[E / R::kPack], r[E / R::kPack], dh[E / R::kPack], dr[E / R::kPack];
};

// Whether calls of one y and at most one dh have instances of their own: all but two packs of binary32 in one wavefront (50000 x 400
// 98 us with and without, where 92 was reached before calls of several gradients took this form; beyond 4096 columns 2048 x 8192 88 -> 84).
template <int DT, bool TEAM, int E>
constexpr bool row_single() { return E == RowType<DT>::kPack || TEAM; }

template <int DT, bool PF32, bool TEAM, int E, bool SINGLE, bool BIAS, bool STREAM>
__global__ void __launch_bounds__(team_block(TEAM), 4) fold_norm_backward_kernel(const BackwardArgs) {
  typedef RowType<DT> R;
  typedef Share<R, TEAM, E> S;
  typedef ParamShare<R, PF32, TEAM, E> P;
  constexpr int kTeams = TEAM ? 1 : kBlock / kWave;
  constexpr bool kWide = E > 8;
  constexpr int kPack = R::kPack, kPacks = E / kPack;
  constexpr bool kNext = E == R::kPack || (SINGLE && R::kBytes == 2 && !BIAS);  // the next row is on its way
  constexpr int kFold = E * R::kBytes > 32 ? 1 : E * R::kBytes > 16 ? 2 : 4;  // gradients in flight together; more cost registers
  const BackwardArgsAt args = (BackwardArgsAt)__builtin_amdgcn_kernarg_segment_ptr();  // (the one argument stands at its start)
  const BackwardArgsAt a0 = args;
  __shared__ float words[2][TEAM ? kMostWaves : 1][kSumsAtOnce];
  extern __shared__ f32x4 column_words[];  // backward_lds() of them
  const int team = TEAM ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave), lanes = TEAM ? (int)blockDim.x : kWave;
  const unsigned t = blockIdx.x * kTeams + team;
  const bool there = t < a0->n_teams;  // (a workgroup's last teams may have nothing to do, but they meet the others at its end)
  const S s((int)threadIdx.x % lanes, lanes, a0->width);
  TeamSums<TEAM> sums{words, lanes / kWave, 0};
  auto columns = [&](int n) { return column_words + (n * (E / 4)) * (int)blockDim.x + (int)threadIdx.x; };
  const bool post = a0->post_kind != PCCL_NORM_NONE, outs = a0->n_out > 0, pre = a0->pre_kind != PCCL_NORM_NONE && outs;
  const bool post_layer = a0->post_kind == PCCL_NORM_LAYER, pre_layer = pre && a0->pre_kind == PCCL_NORM_LAYER;
  const float per_width = a0->per_width;

  float wpre_kept[kWide ? 1 : E], ones[kPack];
  Columns<E, kWide> p1{{}, columns(0), (int)blockDim.x}, s1{{}, columns(1), (int)blockDim.x};
  Columns<E, !kWide> p0{{}, columns(2), (int)blockDim.x}, s0{{}, columns(3), (int)blockDim.x};                   // (BIAS)
  Columns<E, true> post_sums{{}, columns(0), (int)blockDim.x}, post_bias_sums{{}, columns(1), (int)blockDim.x};  // (E up to 8)
  p1.zero();
  if constexpr (BIAS) p0.zero();
#pragma unroll
  for (int i = 0; i < kPack; ++i) ones[i] = 1.0f;
  // wpre and cgw: with E = 16 read again (from the caches), pack by pack, wherever a row needs them
  auto get_wpre = [&](int j, float (&to)[kPack]) {
    const BackwardArgsAt a = read_again(args);
#pragma unroll
    for (int i = 0; i < kPack; ++i) to[i] = 1.0f;
    if (a->pre_weight) {
      P::pack(s, a->pre_weight, j, to);
#pragma unroll
      for (int i = 0; i < kPack; ++i) to[i] += a->weight_offset;
    }
  };
  auto get_cgw = [&](unsigned group, int j, float (&to)[kPack]) {
    const BackwardArgsAt a = read_again(args);
#pragma unroll
    for (int i = 0; i < kPack; ++i) to[i] = a->block_scale;
    if (a->gate) {
      float f[kPack];
      P::pack(s, a->gate + group * a->gate_bytes, j, f);
#pragma unroll
      for (int i = 0; i < kPack; ++i) to[i] *= f[i];
    }
    if (a->post_weight) {
      float f[kPack];
      P::pack(s, a->post_weight, j, f);
#pragma unroll
      for (int i = 0; i < kPack; ++i) to[i] *= f[i] + a->weight_offset;
    }
  };
  auto all = [&](auto &&get, float (&to)[kWide ? 1 : E]) {
    if constexpr (!kWide) {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        float x[kPack];
        get(j, x);
#pragma unroll
        for (int i = 0; i < kPack; ++i) to[j * kPack + i] = x[i];
      }
    }
  };
  all(get_wpre, wpre_kept);

  auto load_row = [&](unsigned long row, BackRow<R, E> &x) {
    const BackwardArgsAt a = read_again(args);
    if (a->grad_residual_out) s.template load<STREAM>(a->grad_residual_out + row * a->grad_residual_out_bytes, x.dr);
    if (pre) s.template load<STREAM>(a->residual_out + row * a->residual_out_bytes, x.r);
    if (outs) s.template load<STREAM>(a->grad_outs[0] + row * a->grad_out_bytes, x.dh);
    s.template load<STREAM>(a->ins[0] + row * a->in_bytes, x.y);
  };

  const unsigned first = (unsigned)((unsigned long)a0->n_strips * t / a0->n_teams);
  const unsigned end = there ? (unsigned)((unsigned long)a0->n_strips * (t + 1) / a0->n_teams) : first;
  for (unsigned strip = first; strip < end; ++strip) {
    const BackwardArgsAt a1 = read_again(args);
    const unsigned group = strip / a1->strips;
    const unsigned long group_row = (unsigned long)group * a1->gate_rows, begin = group_row + (strip - group * a1->strips);
    unsigned long stop = group_row + a1->gate_rows;  // (the last gate row may have fewer rows than gate_rows, and some of its strips none)
    if (stop > a1->rows) stop = a1->rows;
    const unsigned step = a1->strips;

    BackRow<R, E> next;
    if (kNext && begin < stop) load_row(begin, next);
    s1.zero();
    if constexpr (BIAS) s0.zero();
    float cgw_kept[kWide ? 1 : E];
    all([&](int j, float (&to)[kPack]) { get_cgw(group, j, to); }, cgw_kept);

    for (unsigned long row = begin; row < stop; row += step) {
      BackRow<R, E> now;
      float y_kept[E], dh_kept[E], r_kept[E];  // (those that are not unpacked anew)
      if constexpr (kNext) {
        now = next;
        if (row + step < stop) load_row(row + step, next);
      } else {
        load_row(row, now);
      }
      if constexpr (!(SINGLE && kWide)) {
        s.up(now.y, y_kept);
        if (outs) s.up(now.dh, dh_kept);
      }
      if constexpr (!SINGLE) {
        const BackwardArgsAt a = read_again(args);
        fold_rows<STREAM, kFold, 1>(s, a->grad_outs, a->n_out, row * a->grad_out_bytes, dh_kept);
        fold_rows<STREAM, kFold, 1>(s, a->ins, a->n_in, row * a->in_bytes, y_kept);
      }
      if constexpr (!(SINGLE && kWide)) {
        s.mask(y_kept);
        if (outs) s.mask(dh_kept);
      }
      if constexpr (!kWide) {
        if (pre) {
          s.up(now.r, r_kept);
          s.mask(r_kept);
        }
      }
      // pack j of y, dh and r, y and r less their means once those are known
      float mean_y = 0.0f, mean_r = 0.0f;
      auto unpacked = [&](u32x4 v, int j, float mean, float (&to)[kPack]) {
        asm volatile("" : "+v"(v));  // (no instruction: the compiler may not keep what it unpacked before)
        R::up(v, to);
#pragma unroll
        for (int i = 0; i < kPack; ++i) to[i] -= mean;
        s.mask_pack(j, to);
      };
      auto kept = [&](const float (&x)[E], int j, float (&to)[kPack]) {
#pragma unroll
        for (int i = 0; i < kPack; ++i) to[i] = x[j * kPack + i];
      };
      auto get_y = [&](int j, float (&to)[kPack]) {
        if constexpr (SINGLE && kWide) unpacked(now.y[j], j, mean_y, to);
        else kept(y_kept, j, to);
      };
      auto get_dh = [&](int j, float (&to)[kPack]) {
        if constexpr (SINGLE && kWide) unpacked(now.dh[j], j, 0.0f, to);
        else kept(dh_kept, j, to);
      };
      auto get_r = [&](int j, float (&to)[kPack]) {
        if constexpr (kWide) unpacked(now.r[j], j, mean_r, to);
        else kept(r_kept, j, to);
      };
      auto wpre = [&](int j, float (&to)[kPack]) {
        if constexpr (kWide) get_wpre(j, to);
        else kept(wpre_kept, j, to);
      };
      auto cgw = [&](int j, float (&to)[kPack]) {
        if constexpr (kWide) get_cgw(group, j, to);
        else kept(cgw_kept, j, to);
      };
      // packs one after the other: what one of them needs is not loaded before the last is done with
      auto packs = [&](auto &&work) {
#pragma unroll
        for (int j = 0; j < kPacks; ++j) {
          if (!kWide || j == 0 || __builtin_amdgcn_readfirstlane(s.lo[j]) < kPack) work(j);  // (a wavefront may be behind the row's end)
          if constexpr (kWide) __builtin_amdgcn_sched_barrier(0);
        }
      };
      // both norms' statistics, and what the pre norm's backward sums, in one go over the team (two with a layer norm)
      if (post_layer || pre_layer) {
        float m[2] = {0.0f, 0.0f};
        packs([&](int j) {
          float x[kPack];
          if (post_layer) {
            get_y(j, x);
#pragma unroll
            for (int i = 0; i < kPack; ++i) m[0] += x[i];
          }
          if (pre_layer) {
            get_r(j, x);
#pragma unroll
            for (int i = 0; i < kPack; ++i) m[1] += x[i];
          }
        });
        sums(m);
        if (post_layer) {
          mean_y = m[0] * per_width;
          if constexpr (!(SINGLE && kWide)) {
#pragma unroll
            for (int i = 0; i < E; ++i) y_kept[i] -= mean_y;
            s.mask(y_kept);
          }
        }
        if (pre_layer) {
          mean_r = m[1] * per_width;
          if constexpr (!kWide) {
#pragma unroll
            for (int i = 0; i < E; ++i) r_kept[i] -= mean_r;
            s.mask(r_kept);
          }
        }
      }
      float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // squares of y, squares of r, dh * w * r, dh * w
      packs([&](int j) {
        if (post) {
          float y[kPack];
          get_y(j, y);
#pragma unroll
          for (int i = 0; i < kPack; ++i) q[0] = __builtin_fmaf(y[i], y[i], q[0]);
        }
        if (pre) {
          float r[kPack], dh[kPack], w[kPack];
          wpre(j, w);
          get_r(j, r);
          get_dh(j, dh);
#pragma unroll
          for (int i = 0; i < kPack; ++i) {
            q[1] = __builtin_fmaf(r[i], r[i], q[1]);
            q[2] = __builtin_fmaf(dh[i] * w[i], r[i], q[2]);
          }
          if (pre_layer) {
#pragma unroll
            for (int i = 0; i < kPack; ++i) q[3] = __builtin_fmaf(dh[i], w[i], q[3]);
          }
        }
      });
      if (post || pre) sums(q);
      const BackwardArgsAt a = read_again(args);
      float dr[E] = {};
      // dr += rstd * (d - rhat * mean(d * rhat) - mean(d)), d = dh * w
      const float pre_rstd = one_over_spread(q[1], per_width, a->pre_eps);
      const float pre_along = -pre_rstd * (q[2] * per_width);  // (no power of rstd on its own: with a tiny eps that could pass the largest binary32)
      const float pre_mean = pre_rstd * (q[3] * per_width);
      packs([&](int j) {
        float d[kPack], dh[kPack];
        if (a->grad_residual_out) {
          R::up(now.dr[j], d);
        } else {
#pragma unroll
          for (int i = 0; i < kPack; ++i) d[i] = 0.0f;
        }
        if (pre) {
          float w[kPack], r[kPack];
          wpre(j, w);
          get_r(j, r);
          get_dh(j, dh);
#pragma unroll
          for (int i = 0; i < kPack; ++i) {
            r[i] *= pre_rstd;
            d[i] = __builtin_fmaf(pre_rstd, __builtin_fmaf(r[i], pre_along, dh[i] * w[i]), d[i]);
          }
          p1.add(j * kPack, dh, r);
          if (pre_layer) {
#pragma unroll
            for (int i = 0; i < kPack; ++i) d[i] -= pre_mean;
          }
          if constexpr (BIAS) p0.add(j * kPack, dh, ones);
        } else if (outs) {
          get_dh(j, dh);
#pragma unroll
          for (int i = 0; i < kPack; ++i) d[i] += dh[i];
        }
        s.mask_pack(j, d);
        if (a->grad_residual) {
          float x[kPack];
#pragma unroll
          for (int i = 0; i < kPack; ++i) x[i] = a->residual_scale * d[i];
          s.store_pack(a->grad_residual + row * a->grad_residual_bytes, j, x);
        }
#pragma unroll
        for (int i = 0; i < kPack; ++i) dr[j * kPack + i] = d[i];
      });
      const float post_rstd = post ? one_over_spread(q[0], per_width, a->post_eps) : 1.0f;
      float m[2] = {0.0f, 0.0f};
      packs([&](int j) {
        float d[kPack], y[kPack], w[kPack];
        kept(dr, j, d);
        cgw(j, w);
        get_y(j, y);
#pragma unroll
        for (int i = 0; i < kPack; ++i) y[i] *= post_rstd;
        s1.add(j * kPack, d, y);
        if constexpr (BIAS)
          if (post) s0.add(j * kPack, d, ones);
#pragma unroll
        for (int i = 0; i < kPack; ++i) {
          d[i] *= w[i];
          m[0] = __builtin_fmaf(d[i], y[i], m[0]);
          dr[j * kPack + i] = d[i];
          if constexpr (!(SINGLE && kWide)) y_kept[j * kPack + i] = y[i];
        }
        if (post_layer) {
#pragma unroll
          for (int i = 0; i < kPack; ++i) m[1] += d[i];
        }
      });
      if (post) {
        sums(m);
        const float along = -post_rstd * (m[0] * per_width), mean = -post_rstd * (m[1] * per_width);
        packs([&](int j) {
          float y[kPack];
          get_y(j, y);
#pragma unroll
          for (int i = 0; i < kPack; ++i) {
            if constexpr (SINGLE && kWide) y[i] *= post_rstd;
            dr[j * kPack + i] = __builtin_fmaf(dr[j * kPack + i], post_rstd, __builtin_fmaf(y[i], along, mean));
          }
        });
      }
      const unsigned long at = row * a->grad_in_bytes;
#pragma unroll 1
      for (int j = 0; j < a->n_grad_in; ++j) s.store(a->grad_ins[j] + at, dr);
    }

    // the strip's sums: to the gate's gradient or its workspace, and, times the gate, to the team's
    const BackwardArgsAt a = read_again(args);
    float x[E], x0[E];
    s1.get(x);
    if constexpr (BIAS) s0.get(x0);
    if (a->grad_gate) {
      float d[E];
#pragma unroll
      for (int i = 0; i < E; ++i) d[i] = x[i] * a->block_scale;
      if (a->post_weight) {
        P w;
        float f[E];
        w.load(s, a->post_weight);
        w.up(f);
#pragma unroll
        for (int i = 0; i < E; ++i) d[i] *= f[i] + a->weight_offset;
      }
      if constexpr (BIAS) {
        if (a->post_bias) {
          P b;
          float f[E];
          b.load(s, a->post_bias);
          b.up(f);
#pragma unroll
          for (int i = 0; i < E; ++i) d[i] = __builtin_fmaf(f[i] * a->block_scale, x0[i], d[i]);
        }
      }
      if (a->gate_sums) {
        store_sums(s, a->gate_sums + (unsigned long)strip * a->width, d);
      } else if constexpr (PF32 && R::kBytes == 2) {
        store_sums(s, (float *)(a->grad_gate + group * a->grad_gate_bytes), d);
      } else {
        s.store(a->grad_gate + group * a->grad_gate_bytes, d);
      }
    }
    if (a->want_sums[0] || a->want_sums[1]) {
      float f[E];
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = a->block_scale;
      if (a->gate) {
        P g;
        float e[E];
        g.load(s, a->gate + group * a->gate_bytes);
        g.up(e);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] *= e[i];
      }
      if constexpr (!kWide) {
        if (strip == first) {
          post_sums.zero();
          if constexpr (BIAS) post_bias_sums.zero();
        }
        post_sums.add(0, f, x);
        if constexpr (BIAS) post_bias_sums.add(0, f, x0);
      } else {
        // (each lane adds to the columns that it wrote itself)
        float *mine = a->sums + (unsigned long)t * 4 * a->width;
        auto add = [&](float *row, const float (&v)[E]) {
          float had[E] = {};
          if (strip != first) load_sums(s, row, had);
#pragma unroll
          for (int i = 0; i < E; ++i) had[i] = __builtin_fmaf(f[i], v[i], had[i]);
          store_sums(s, row, had);
        };
        if (a->want_sums[0]) add(mine, x);
        if constexpr (BIAS)
          if (a->want_sums[1]) add(mine + a->width, x0);
      }
    }
  }
  // the team's sums; those of the four teams of a workgroup are added first
  float *mine = a0->sums + (unsigned long)(TEAM ? t : blockIdx.x) * 4 * a0->width;
  auto put = [&](int which, bool set, float (&x)[E]) {
    if constexpr (!TEAM) {
      __syncthreads();  // (every team comes here; what LDS held before is done with)
#pragma unroll
      for (int k = 0; k < E / 4; ++k) column_words[k * kBlock + (int)threadIdx.x] = set ? f32x4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]} : f32x4{0, 0, 0, 0};
      __syncthreads();
      if (team != 0) return;
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = column_words[i / 4 * kBlock + (int)threadIdx.x][i % 4];
#pragma unroll
      for (int other = 1; other < kTeams; ++other)
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] += column_words[i / 4 * kBlock + other * kWave + (int)threadIdx.x][i % 4];
    }
    store_sums(s, mine + which * a0->width, x);
  };
  // (taken out of LDS before the first of them goes through it)
  float x_post[E], x_post_bias[E], x_p1[E], x_p0[E];
  if constexpr (!kWide) post_sums.get(x_post);
  if constexpr (!kWide && BIAS) post_bias_sums.get(x_post_bias);
  p1.get(x_p1);
  if constexpr (BIAS) p0.get(x_p0);
  if constexpr (!kWide) {  // (a team has a strip, so these were set)
    if (a0->want_sums[0]) put(0, there, x_post);
    if constexpr (BIAS)
      if (a0->want_sums[1]) put(1, there, x_post_bias);
  }
  if (a0->want_sums[2]) put(2, there, x_p1);
  if constexpr (BIAS)
    if (a0->want_sums[3]) put(3, there, x_p0);
}

// Bytes of LDS for sums by column: with E up to 8 the post norm's, with biases theirs, p0 and s0 too; with E = 16 p1 and s1.
inline unsigned backward_lds(int lanes_of_workgroup, int elems, bool bias) {
  return (unsigned)lanes_of_workgroup * elems * 4 * (elems > 8 ? 2 : bias ? 4 : 1);
}

// Joins the teams' sums: a workgroup adds 64 columns of one parameter's (or one gate row's) partial rows.  A lane has four columns, so
// that four rows of 256 bytes are one load of a wavefront and sixteen wavefronts have 64 rows at work at once, each every 64th
// row; then the four of a wavefront, then the wavefronts, always in the same order.  What bounds it is the round trip to memory (the
// rows were written by other chiplets): few workgroups, all resident, eight loads of each lane in flight.  (One column a lane and 16 or 64
// columns a workgroup: 512 rows x 4096 x 8 20 us, 1024 rows x 300 x 2 9 us and, with 64, 17.)
struct SumsArgs {
  const float *sums, *gate_sums;
  char *out[4];      // by parameter, null: not wanted
  int listed[4];     // which parameters blockIdx.y = 0 .. n_listed - 1 stand for
  int n_listed, width;
  unsigned n_partial, strips;
  char *grad_gate;   // blockIdx.y = n_listed + gate row
  long grad_gate_bytes;
};
constexpr int kJoinWaves = 16, kJoinColumns = 64, kJoinRows = 4;

template <int DT, bool PF32>
__global__ void __launch_bounds__(kJoinWaves * kWave) fold_norm_sums_kernel(const SumsArgs a) {
  __shared__ f32x4 part[kJoinWaves][kWave / kJoinRows];
  const int lane = (int)threadIdx.x % kWave, wave = (int)threadIdx.x / kWave, at = lane % (kWave / kJoinRows);
  // the last lanes move back to end with the row: they add, and store, what their neighbours do (rows of less than four: one by one)
  int column = (int)blockIdx.x * kJoinColumns + at * 4;
  const bool mine = column < a.width, narrow = a.width < 4;
  if (!narrow && column > a.width - 4) column = a.width - 4;
  const bool of_gate = (int)blockIdx.y >= a.n_listed;
  const int which = of_gate ? 0 : a.listed[blockIdx.y];
  const long group = (int)blockIdx.y - a.n_listed;
  const float *from = of_gate ? a.gate_sums + group * a.strips * a.width : a.sums + (long)which * a.width;
  const long step = of_gate ? a.width : 4l * a.width;
  const unsigned n = of_gate ? a.strips : a.n_partial;
  f32x4 t{0, 0, 0, 0};
  if (mine) {
    if (!narrow) {
      typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
#pragma unroll 8
      for (unsigned k = wave * kJoinRows + lane / (kWave / kJoinRows); k < n; k += kJoinWaves * kJoinRows) t += *(const f32x4_a4 *)(from + k * step + column);
    } else {
      for (unsigned k = wave * kJoinRows + lane / (kWave / kJoinRows); k < n; k += kJoinWaves * kJoinRows)
        for (int i = 0; i < a.width; ++i) t[i] += from[k * step + i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] += __shfl_xor(t[i], 16, kWave);
    t[i] += __shfl_xor(t[i], 32, kWave);
  }
  if (lane == at) part[wave][at] = t;
  __syncthreads();
  if (wave != 0 || lane != at || !mine) return;
  t = part[0][at];
#pragma unroll
  for (int k = 1; k < kJoinWaves; ++k) t += part[k][at];
  char *to = of_gate ? a.grad_gate + group * a.grad_gate_bytes : a.out[which];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (column + i >= a.width) break;
    if constexpr (PF32) ((float *)to)[column + i] = t[i];
    else ((typename RowType<DT>::elem_t *)to)[column + i] = RowType<DT>::down1(t[i]);
  }
}

// ---- launchers, one translation unit per pair of types ---------------------------------------------------
// The lanes of a row's team and the elements of a lane.
struct NormShape {
  int lanes, elems;
  int block() const { return lanes == kWave ? kBlock : lanes; }  // lanes of a workgroup
  unsigned workgroups(unsigned rows) const { return lanes == kWave ? (rows + kBlock / kWave - 1) / (kBlock / kWave) : rows; }
};

template <int DT, class F>
inline void with_norm_shape(NormShape n, F &&f) {
  typedef std::integral_constant<int, 4> Four;
  typedef std::integral_constant<int, 8> Eight;
  typedef std::integral_constant<int, 16> Sixteen;
  if constexpr (DT == PCCL_F32) {
    if (n.elems == 4) return n.lanes == kWave ? f(std::false_type{}, Four{}) : f(std::true_type{}, Four{});
  }
  if (n.lanes == kWave) f(std::false_type{}, Eight{});
  else if (n.elems == 8) f(std::true_type{}, Eight{});
  else f(std::true_type{}, Sixteen{});
}

template <int DT, bool PF32> hipError_t launch_fold_norm(NormShape n, bool stream_in, hipStream_t stream, const ForwardArgs &a);
template <int DT, bool PF32> hipError_t launch_fold_norm_backward(NormShape n, bool single, bool bias, bool stream_in, hipStream_t stream, const BackwardArgs &a);
template <int DT, bool PF32> hipError_t launch_fold_norm_sums(unsigned grid_y, hipStream_t stream, const SumsArgs &a);

#define PCCL_DEFINE_FOLD_NORM(DT, PF32)                                                                                         \
  template <> hipError_t launch_fold_norm<DT, PF32>(NormShape n, bool stream_in, hipStream_t stream, const ForwardArgs &a) {    \
    with_norm_shape<DT>(n, [&](auto team, auto e) {                                                                             \
      constexpr bool TEAM = decltype(team)::value;                                                                              \
      constexpr int E = decltype(e)::value;                                                                                     \
      constexpr int kMany = DT == PCCL_F32 && E == 16 ? 2 : 8; /* eight inputs of 64 bytes a lane would spill */                \
      const dim3 grid(n.workgroups(a.rows - a.row0)), block(n.block());                                                         \
      if constexpr (DT != PCCL_F32 || TEAM || E == 4) { /* (two packs of binary32 in one wavefront: only backward) */           \
        if (a.n_in <= 2) hipLaunchKernelGGL((fold_norm_kernel<DT, PF32, TEAM, E, 2, false>), grid, block, 0, stream, a);        \
        else if (stream_in) hipLaunchKernelGGL((fold_norm_kernel<DT, PF32, TEAM, E, kMany, true>), grid, block, 0, stream, a);  \
        else hipLaunchKernelGGL((fold_norm_kernel<DT, PF32, TEAM, E, kMany, false>), grid, block, 0, stream, a);                \
      }                                                                                                                         \
    });                                                                                                                         \
    return hipGetLastError();                                                                                                   \
  }                                                                                                                             \
  template <> hipError_t launch_fold_norm_backward<DT, PF32>(NormShape n, bool single, bool bias, bool stream_in, hipStream_t stream, const BackwardArgs &a) { \
    with_norm_shape<DT>(n, [&](auto team, auto e) {                                                                             \
      constexpr bool TEAM = decltype(team)::value;                                                                              \
      constexpr int E = decltype(e)::value;                                                                                     \
      const dim3 grid(n.workgroups(a.n_teams)), block(n.block());                                                               \
      const unsigned lds = backward_lds(n.block(), E, bias);                                                                    \
      auto run = [&](auto ahead, auto b, auto st) {                                                                             \
        hipLaunchKernelGGL((fold_norm_backward_kernel<DT, PF32, TEAM, E, decltype(ahead)::value, decltype(b)::value, decltype(st)::value>), \
                           grid, block, lds, stream, a);                                                                        \
      };                                                                                                                        \
      constexpr bool kSingle = row_single<DT, TEAM, E>();                                                                       \
      if (kSingle && single) {                                                                                                  \
        typedef std::integral_constant<bool, kSingle> Single;                                                                    \
        if (stream_in) bias ? run(Single{}, std::true_type{}, std::true_type{}) : run(Single{}, std::false_type{}, std::true_type{}); \
        else bias ? run(Single{}, std::true_type{}, std::false_type{}) : run(Single{}, std::false_type{}, std::false_type{});   \
      } else {                                                                                                                  \
        typedef std::integral_constant<bool, !kSingle> Streams; /* (16-bit rows of several gradients: 85 against 88 us, not worth a variant) */ \
        if (stream_in) bias ? run(std::false_type{}, std::true_type{}, Streams{}) : run(std::false_type{}, std::false_type{}, Streams{}); \
        else bias ? run(std::false_type{}, std::true_type{}, std::false_type{}) : run(std::false_type{}, std::false_type{}, std::false_type{}); \
      }                                                                                                                         \
    });                                                                                                                         \
    return hipGetLastError();                                                                                                   \
  }                                                                                                                             \
  template <> hipError_t launch_fold_norm_sums<DT, PF32>(unsigned grid_y, hipStream_t stream, const SumsArgs &a) {              \
    hipLaunchKernelGGL((fold_norm_sums_kernel<DT, PF32>), dim3((a.width + kJoinColumns - 1) / kJoinColumns, grid_y), dim3(kJoinWaves * kWave), 0, stream, a); \
    return hipGetLastError();                                                                                                   \
  }

}  // namespace pccl_dev

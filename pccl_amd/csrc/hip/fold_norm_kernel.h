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

constexpr int team_block(int lanes) { return lanes < kBlock ? kBlock : lanes; }

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

// FULL: sums for biases and gate as well (registers for five rows of sums instead of two)
template <int DT, bool PF32, int LANES, int E, bool FULL>
__global__ void __launch_bounds__(team_block(LANES)) fold_norm_backward_kernel(const BackwardArgs a) {
  typedef RowType<DT> R;
  typedef Share<R, LANES, E> S;
  typedef ParamShare<R, PF32, LANES, E> P;
  constexpr int kPacks = E / R::kPack;
  constexpr int kTeams = team_block(LANES) / LANES;
  constexpr int kFold = 4;  // gradients in flight together; more cost registers
  __shared__ float words[2][LANES / kWave][kSumsAtOnce];
  const int team = kTeams == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / LANES);
  const unsigned t = blockIdx.x * kTeams + team;
  if (t >= a.n_teams) return;
  const S s((int)threadIdx.x % LANES, a.width);
  TeamSums<LANES> sums{words, 0};
  const bool post = a.post_kind != PCCL_NORM_NONE, pre = a.pre_kind != PCCL_NORM_NONE;
  const bool post_layer = a.post_kind == PCCL_NORM_LAYER, pre_layer = a.pre_kind == PCCL_NORM_LAYER;

  float sum_post[E], sum_pre[E], sum_post_bias[FULL ? E : 1], sum_pre_bias[FULL ? E : 1], sum_gate[FULL ? E : 1];
#pragma unroll
  for (int i = 0; i < E; ++i) sum_post[i] = sum_pre[i] = 0.0f;
  if constexpr (FULL) {
#pragma unroll
    for (int i = 0; i < E; ++i) sum_post_bias[i] = sum_pre_bias[i] = 0.0f;
  }

  const unsigned first = (unsigned)((unsigned long)a.n_strips * t / a.n_teams);
  const unsigned end = (unsigned)((unsigned long)a.n_strips * (t + 1) / a.n_teams);
  for (unsigned strip = first; strip < end; ++strip) {
    const unsigned group = strip / a.strips;
    // (the last gate row may have fewer rows than gate_rows, and its last strips then none: 64 bits, and no row)
    const unsigned long group_row = (unsigned long)group * a.gate_rows;
    const unsigned long begin = group_row + (unsigned long)(strip - group * a.strips) * a.strip_rows;
    unsigned long stop = begin + a.strip_rows;
    if (stop > group_row + a.gate_rows) stop = group_row + a.gate_rows;
    if (stop > a.rows) stop = a.rows;
    const char *gate_row = a.gate ? a.gate + group * a.gate_bytes : nullptr;
    if constexpr (FULL) {
#pragma unroll
      for (int i = 0; i < E; ++i) sum_gate[i] = 0.0f;
    }
    for (unsigned long row = begin; row < stop; ++row) {
      u32x4 v_r[kPacks], v_dr[kPacks];
      float y[E], dh[E], dr[E];
      P w_pre, w_post, gate;
      if (a.grad_residual_out) s.load(a.grad_residual_out + row * a.grad_residual_out_bytes, v_dr);
      if (pre && a.n_out) s.load(a.residual_out + (long)row * a.residual_out_bytes, v_r);
      if (a.n_out) fold_rows<R, LANES, E, kFold>(s, a.grad_outs, a.n_out, row * a.grad_out_bytes, dh);
      fold_rows<R, LANES, E, kFold>(s, a.ins, a.n_in, (long)row * a.in_bytes, y);
      if (a.pre_weight) w_pre.load(s, a.pre_weight);
      if (a.post_weight) w_post.load(s, a.post_weight);
      if (gate_row) gate.load(s, gate_row);
      if (a.grad_residual_out) {
        s.up(v_dr, dr);
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] = 0.0f;
      }

      s.mask(y);
      s.mask(dr);
      if (a.n_out) s.mask(dh);
      // both norms' statistics, and what the pre norm's backward sums, in one go over the team (two with a layer norm)
      float r[E], mean_y = 0.0f;
      const bool through_pre = pre && a.n_out;
      if (through_pre) {
        s.up(v_r, r);
        s.mask(r);
      }
      if ((post && post_layer) || (through_pre && pre_layer)) {
        float m[2] = {0.0f, 0.0f};
        if (post && post_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) m[0] += y[i];
        }
        if (through_pre && pre_layer) {
#pragma unroll
          for (int i = 0; i < E; ++i) m[1] += r[i];
        }
        sums(m);
        if (post && post_layer) {
          mean_y = m[0] * a.per_width;
#pragma unroll
          for (int i = 0; i < E; ++i) y[i] -= mean_y;
          s.mask(y);
        }
        if (through_pre && pre_layer) {
          const float mean_r = m[1] * a.per_width;
#pragma unroll
          for (int i = 0; i < E; ++i) r[i] -= mean_r;
          s.mask(r);
        }
      }
      float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // squares of y, squares of r, dh * w * r, dh * w
      if (post) {
#pragma unroll
        for (int i = 0; i < E; ++i) q[0] = __builtin_fmaf(y[i], y[i], q[0]);
      }
      float d[E];  // dh * w
      if (through_pre) {
        if (a.pre_weight) {
          float w[E];
          w_pre.up(w);
#pragma unroll
          for (int i = 0; i < E; ++i) d[i] = dh[i] * (w[i] + a.weight_offset);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) d[i] = dh[i];
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
          q[1] = __builtin_fmaf(r[i], r[i], q[1]);
          q[2] = __builtin_fmaf(d[i], r[i], q[2]);
          q[3] += d[i];
        }
      }
      if (post || through_pre) sums(q);
      if (through_pre) {
        const float rstd = one_over_spread(q[1], a.per_width, a.pre_eps);
        const float along = q[2] * rstd * a.per_width, mean_d = pre_layer ? q[3] * a.per_width : 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float hat = r[i] * rstd;
          sum_pre[i] = __builtin_fmaf(dh[i], hat, sum_pre[i]);
          dr[i] = __builtin_fmaf(rstd, d[i] - __builtin_fmaf(hat, along, mean_d), dr[i]);
        }
        if constexpr (FULL) {
#pragma unroll
          for (int i = 0; i < E; ++i) sum_pre_bias[i] += dh[i];
        }
        if (pre_layer) s.mask(dr);  // (the mean of d went into masked elements)
      } else if (a.n_out) {
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] += dh[i];
      }
      if (a.grad_residual) {
        float x[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = a.residual_scale * dr[i];
        s.store(a.grad_residual + row * a.grad_residual_bytes, x);
      }
#pragma unroll
      for (int i = 0; i < E; ++i) dr[i] *= a.block_scale;
      float rstd_y = 1.0f;
      if (post) {
        rstd_y = one_over_spread(q[0], a.per_width, a.post_eps);
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] *= rstd_y;
      }
      float w[E];
      if (a.post_weight) {
        w_post.up(w);
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] += a.weight_offset;
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = 1.0f;
      }
      if (gate_row) {
        float g[E];
        gate.up(g);
        if constexpr (FULL) {
          float b[E];
          if (a.post_bias) {
            P bias;
            bias.load(s, a.post_bias);
            bias.up(b);
          } else {
#pragma unroll
            for (int i = 0; i < E; ++i) b[i] = 0.0f;
          }
#pragma unroll
          for (int i = 0; i < E; ++i) sum_gate[i] = __builtin_fmaf(dr[i], __builtin_fmaf(y[i], w[i], b[i]), sum_gate[i]);
        }
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] *= g[i];
      }
      if (post) {  // dr is the gradient of n now, y standardised
        if constexpr (FULL) {
#pragma unroll
          for (int i = 0; i < E; ++i) sum_post_bias[i] += dr[i];
        }
        float m[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
          sum_post[i] = __builtin_fmaf(dr[i], y[i], sum_post[i]);
          dr[i] *= w[i];
          m[0] = __builtin_fmaf(dr[i], y[i], m[0]);
          m[1] += dr[i];
        }
        sums(m);
        const float along = m[0] * a.per_width, mean_d = post_layer ? m[1] * a.per_width : 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) dr[i] = rstd_y * (dr[i] - __builtin_fmaf(y[i], along, mean_d));
      }
      const long at = row * a.grad_in_bytes;
#pragma unroll
      for (int j = 0; j < PCCL_MAX_INPUTS; ++j)
        if (j < a.n_grad_in) s.store(a.grad_ins[j] + at, dr);
    }
    if constexpr (FULL) {
      if (a.gate_sums) store_sums(s, a.gate_sums + strip * a.width, sum_gate);
      else if (a.grad_gate) {
        if constexpr (PF32 && R::kBytes == 2) store_sums(s, (float *)(a.grad_gate + group * a.grad_gate_bytes), sum_gate);
        else s.store(a.grad_gate + group * a.grad_gate_bytes, sum_gate);
      }
    }
  }
  float *mine = a.sums + (long)t * 4 * a.width;
  if (a.want_sums[0]) store_sums(s, mine, sum_post);
  if (a.want_sums[2]) store_sums(s, mine + 2 * a.width, sum_pre);
  if constexpr (FULL) {
    if (a.want_sums[1]) store_sums(s, mine + a.width, sum_post_bias);
    if (a.want_sums[3]) store_sums(s, mine + 3 * a.width, sum_pre_bias);
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
  PCCL_NORM_SHAPE(64, 16)
  PCCL_NORM_SHAPE(256, 8)
  PCCL_NORM_SHAPE(256, 16)
  PCCL_NORM_SHAPE(512, 16)
  PCCL_NORM_SHAPE(1024, 16)
#undef PCCL_NORM_SHAPE
  return false;
}

template <int DT, bool PF32> hipError_t launch_fold_norm(NormShape n, hipStream_t stream, const ForwardArgs &a);
template <int DT, bool PF32> hipError_t launch_fold_norm_backward(NormShape n, bool full, hipStream_t stream, const BackwardArgs &a);
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
  template <> hipError_t launch_fold_norm_backward<DT, PF32>(NormShape n, bool full, hipStream_t stream, const BackwardArgs &a) { \
    with_norm_shape(n, [&](auto l, auto e) {                                                                                \
      constexpr int L = decltype(l)::value, E = decltype(e)::value, kTeams = team_block(L) / L;                             \
      const unsigned grid = (a.n_teams + kTeams - 1) / kTeams;                                                              \
      if (full) hipLaunchKernelGGL((fold_norm_backward_kernel<DT, PF32, L, E, true>), dim3(grid), dim3(team_block(L)), 0, stream, a); \
      else hipLaunchKernelGGL((fold_norm_backward_kernel<DT, PF32, L, E, false>), dim3(grid), dim3(team_block(L)), 0, stream, a); \
    });                                                                                                                     \
    return hipGetLastError();                                                                                               \
  }                                                                                                                         \
  template <> hipError_t launch_fold_norm_sums<DT, PF32>(unsigned grid_y, hipStream_t stream, const SumsArgs &a) {          \
    hipLaunchKernelGGL((fold_norm_sums_kernel<DT, PF32>), dim3((a.width + kWave - 1) / kWave, grid_y), dim3(kJoinWaves * kWave), 0, stream, a); \
    return hipGetLastError();                                                                                               \
  }

}  // namespace pccl_dev

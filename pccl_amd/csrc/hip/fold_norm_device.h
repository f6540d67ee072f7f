// fold_norm_device.h -- device code shared by the forward and backward kernels of the norms around a
// block: how a row lies over the lanes of a team, loads and stores of a lane's share, sums over a team.
//
// A row of `width` elements is worked on by a team of lanes (TEAM false: one wavefront, four of them to a workgroup; TEAM true: a
// workgroup of as many wavefronts as the width needs) and stays in their registers from the first load to the last
// store: E elements a lane, as E / kPack packs of 16 bytes; pack j of lane l is pack j * lanes + l of the row, so that an
// instruction of a wavefront covers 1 KiB.
// Where the width is no multiple of a pack, the row's last pack is moved back to end with the row and the `lo`
// elements at its front, which the pack before it holds as well, are masked: left out of sums, not stored.
// (So every load is one 16-byte load inside the row at any width of at least a pack and any element alignment;
// narrower rows are loaded element by element.)
#pragma once

#include "plugin_common.h"
#include "reduce_copy_device.h"

namespace pccl_dev {

template <int DT> struct RowType;

template <> struct RowType<PCCL_F32> {
  static constexpr int kBytes = 4, kPack = 4;
  typedef u32x4_a4 pack_t;
  typedef unsigned int elem_t;
  static __device__ __forceinline__ void up(u32x4 v, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = as_f32(v[i]);
  }
  static __device__ __forceinline__ u32x4 down(const float *x) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = as_u32(x[i]);
    return v;
  }
  static __device__ __forceinline__ float up1(elem_t e) { return as_f32(e); }
  static __device__ __forceinline__ elem_t down1(float x) { return as_u32(x); }
};

template <> struct RowType<PCCL_BF16> {
  static constexpr int kBytes = 2, kPack = 8;
  typedef u32x4_a2 pack_t;
  typedef unsigned short elem_t;
  static __device__ __forceinline__ void up(u32x4 v, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = as_f32(v[i] << 16);
      x[2 * i + 1] = as_f32(v[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ u32x4 down(const float *x) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 p = {x[2 * i], x[2 * i + 1]};
      v[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector(p, bf16x2));
    }
    return v;
  }
  static __device__ __forceinline__ float up1(elem_t e) { return as_f32((unsigned int)e << 16); }
  static __device__ __forceinline__ elem_t down1(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
};

template <> struct RowType<PCCL_F16> {
  static constexpr int kBytes = 2, kPack = 8;
  typedef u32x4_a2 pack_t;
  typedef unsigned short elem_t;
  static __device__ __forceinline__ void up(u32x4 v, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned int w = v[i];  // (a bit cast of the vector's element itself takes the vector's first)
      const f32x2 p = __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
      x[2 * i] = p.x;
      x[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ u32x4 down(const float *x) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo = x[2 * i], hi = x[2 * i + 1];
      Dtype<PCCL_F16>::rounded_to_f32(lo);
      Dtype<PCCL_F16>::rounded_to_f32(hi);
      const f32x2 p = {lo, hi};
      v[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector(p, f16x2));
    }
    return v;
  }
  static __device__ __forceinline__ float up1(elem_t e) { return (float)__builtin_bit_cast(_Float16, e); }
  static __device__ __forceinline__ elem_t down1(float x) {
    Dtype<PCCL_F16>::rounded_to_f32(x);
    return __builtin_bit_cast(unsigned short, (_Float16)x);
  }
};

// One lane's share of a row: E elements of the packs of type R::kPack.
template <class R, bool TEAM, int E>
struct Share {
  static constexpr int kPacks = E / R::kPack;
  static constexpr bool kMayBeNarrow = !TEAM;  // rows of less than a pack are given to one wavefront
  int off[kPacks];  // where pack j starts in the row (below 0 in a narrow row: its first elements are masked)
  int lo[kPacks];   // elements at its front that are not this lane's; R::kPack or more: no pack
  bool narrow;      // the row is shorter than a pack
  bool ragged;      // some element of some lane is masked

  __device__ __forceinline__ Share(int lane, int lanes, int width) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      const int first = (j * lanes + lane) * R::kPack;
      off[j] = first < width - R::kPack ? first : width - R::kPack;
      lo[j] = first - off[j];
    }
    narrow = kMayBeNarrow && width < R::kPack;
    ragged = width != lanes * E;
  }
  __device__ __forceinline__ bool has(int j) const { return lo[j] < R::kPack; }

  // this lane's pack j of the row at `row` (wave-uniform), zeros where it has none
  // (STREAM: non-temporal)
  template <bool STREAM = false> __device__ __forceinline__ u32x4 load_pack(const char *row, int j) const {
    u32x4 v{0, 0, 0, 0};
    if (has(j)) {
      if (narrow) {
        typename R::elem_t e[R::kPack];
#pragma unroll
        for (int i = 0; i < R::kPack; ++i) e[i] = i >= lo[j] ? ((const typename R::elem_t *)row)[off[j] + i] : (typename R::elem_t)0;
        v = __builtin_bit_cast(u32x4, e);
      } else {
        const typename R::pack_t *at = (const typename R::pack_t *)(row + (unsigned)off[j] * (unsigned)R::kBytes);
        if constexpr (STREAM) v = __builtin_nontemporal_load(at);
        else v = *at;
      }
    }
    return v;
  }
  template <bool STREAM = false> __device__ __forceinline__ void load(const char *row, u32x4 (&v)[kPacks]) const {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) v[j] = load_pack<STREAM>(row, j);
  }
  // Rows are stored non-temporally at every size (forward f32 2 -> 2 at 4096 x 2048 45 -> 38 us, bf16 8 -> 8 at 2048 x 8192 129 -> 122).
  __device__ __forceinline__ void store_pack(char *row, int j, const float *x) const {
    if (lo[j] == 0) {
      __builtin_nontemporal_store(R::down(x), (typename R::pack_t *)(row + (unsigned)off[j] * (unsigned)R::kBytes));
    } else if (has(j)) {
#pragma unroll
      for (int i = 0; i < R::kPack; ++i)
        if (i >= lo[j]) ((typename R::elem_t *)row)[off[j] + i] = R::down1(x[i]);
    }
  }
  __device__ __forceinline__ void store(char *row, const float (&x)[E]) const {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) store_pack(row, j, x + j * R::kPack);
  }
  __device__ __forceinline__ void mask_pack(int j, float (&x)[R::kPack]) const {
    if (ragged && lo[j] != 0) {
#pragma unroll
      for (int i = 0; i < R::kPack; ++i)
        if (i < lo[j]) x[i] = 0.0f;
    }
  }
  // x = 0 in the elements that are not this lane's; wavefronts whose packs are all whole step over it
  __device__ __forceinline__ void mask(float (&x)[E]) const {
    if (ragged) {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        if (lo[j] != 0) {
#pragma unroll
          for (int i = 0; i < R::kPack; ++i)
            if (i < lo[j]) x[j * R::kPack + i] = 0.0f;
        }
      }
    }
  }
  static __device__ __forceinline__ void up(const u32x4 (&v)[kPacks], float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) R::up(v[j], x + j * R::kPack);
  }
};

// One lane's share of a parameter row (weight, bias, gate): elements of the rows' type or binary32.
template <class R, bool PF32, bool TEAM, int E>
struct ParamShare {
  static constexpr int kPacks = E / R::kPack;
  static constexpr bool kWide = PF32 && R::kBytes == 2;  // a pack's parameters are two 16-byte loads
  static constexpr int kWords = kWide ? 2 * kPacks : kPacks;
  u32x4 v[kWords];

  // one pack's
  static __device__ __forceinline__ void load_pack(const Share<R, TEAM, E> &s, const char *row, int j, u32x4 (&v)[kWords / kPacks]) {
    if constexpr (!kWide) {
      v[0] = s.load_pack(row, j);
    } else {
      v[0] = v[1] = u32x4{0, 0, 0, 0};
      if (s.has(j)) {
        if (s.narrow) {
          unsigned int e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = i >= s.lo[j] ? ((const unsigned int *)row)[s.off[j] + i] : 0u;
          v[0] = u32x4{e[0], e[1], e[2], e[3]};
          v[1] = u32x4{e[4], e[5], e[6], e[7]};
        } else {
          const u32x4_a4 *at = (const u32x4_a4 *)(row + (unsigned)s.off[j] * 4u);
          v[0] = at[0];
          v[1] = at[1];
        }
      }
    }
  }
  static __device__ __forceinline__ void up_pack(const u32x4 *v, float *x) {
    if constexpr (!kWide) {
      R::up(v[0], x);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = as_f32(v[i / 4][i % 4]);
    }
  }
  static __device__ __forceinline__ void pack(const Share<R, TEAM, E> &s, const char *row, int j, float (&x)[R::kPack]) {
    u32x4 w[kWords / kPacks];
    load_pack(s, row, j, w);
    up_pack(w, x);
  }
  __device__ __forceinline__ void load(const Share<R, TEAM, E> &s, const char *row) {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) {
      u32x4 w[kWords / kPacks];
      load_pack(s, row, j, w);
#pragma unroll
      for (int k = 0; k < kWords / kPacks; ++k) v[j * (kWords / kPacks) + k] = w[k];
    }
  }
  __device__ __forceinline__ void up(float (&x)[E]) const {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) up_pack(v + j * (kWords / kPacks), x + j * R::kPack);
  }
};

// y = the left fold of this lane's share of n rows; FROM = 1: y holds the first of them already.  AT_ONCE inputs are in flight together.
template <bool STREAM, int AT_ONCE, int FROM, class R, bool TEAM, int E, class Ins>
__device__ __forceinline__ void fold_rows(const Share<R, TEAM, E> &s, const Ins &ins, int n, long at, float (&y)[E]) {
  constexpr int kPacks = E / R::kPack;
  for (int k0 = FROM; k0 < n; k0 += AT_ONCE) {
    u32x4 v[AT_ONCE][kPacks];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (k == 0 || k0 + k < n) s.template load<STREAM>(ins[k0 + k] + at, v[k]);
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      if (k == 0 || k0 + k < n) {
        float x[E];
        s.up(v[k], x);
        if (k == 0 && k0 == 0) {
#pragma unroll
          for (int i = 0; i < E; ++i) y[i] = x[i];
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i) y[i] += x[i];
        }
      }
    }
  }
}

// Sums over lanes by data-parallel-primitive adds, no LDS access: shifts inside rows of 16 lanes leave a row's sum in its last
// lane, broadcasts of those the wavefront's sum in lane 63.  All 64 lanes are active.
template <int CTRL, int ROWS>
__device__ __forceinline__ float plus_dpp(float x) {
  return x + as_f32((unsigned)__builtin_amdgcn_update_dpp(0, (int)as_u32(x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float row_sum(float x) {  // in lanes 15, 31, 47, 63
  x = plus_dpp<0x111, 0xf>(x);  // row_shr:1
  x = plus_dpp<0x112, 0xf>(x);  // row_shr:2
  x = plus_dpp<0x114, 0xf>(x);  // row_shr:4
  return plus_dpp<0x118, 0xf>(x);  // row_shr:8
}
__device__ __forceinline__ float wave_sum(float x) {  // in lane 63
  x = row_sum(x);
  x = plus_dpp<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  return plus_dpp<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ float of_lane(float x, int lane) { return as_f32((unsigned)__builtin_amdgcn_readlane((int)as_u32(x), lane)); }

// Sums over a team, the same value in every lane, added in the same order every time: the wavefronts' sums go to LDS,
// the sixteen lanes of a row read one each and add them as above (reading all of them into every lane cost 64 registers).
// `turn` alternates between two sets of LDS words, so that one barrier a sum is enough: a wavefront writes a set again only
// after the barrier of the sum in between, which every reader of the set has reached.
constexpr int kSumsAtOnce = 4, kMostWaves = 16;
template <bool TEAM>
struct TeamSums {
  float (*words)[TEAM ? kMostWaves : 1][kSumsAtOnce];  // [2]
  int waves, turn;  // a row of 16 lanes has one for each wavefront

  template <int N>
  __device__ __forceinline__ void operator()(float (&x)[N]) {
    if constexpr (!TEAM) {
#pragma unroll
      for (int n = 0; n < N; ++n) x[n] = of_lane(wave_sum(x[n]), kWave - 1);
    } else {
      float (*w)[kSumsAtOnce] = words[turn];
      const int wave = (int)threadIdx.x / kWave, lane = (int)threadIdx.x % kWave;
#pragma unroll
      for (int n = 0; n < N; ++n) x[n] = wave_sum(x[n]);
      if (lane == kWave - 1) {
#pragma unroll
        for (int n = 0; n < N; ++n) w[wave][n] = x[n];
      }
      __syncthreads();
      const int from = lane % kMostWaves;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        x[n] = w[from][n];
        x[n] = from < waves ? x[n] : 0.0f;  // (words of wavefronts that there are not hold anything)
      }
#pragma unroll
      for (int n = 0; n < N; ++n) x[n] = of_lane(row_sum(x[n]), kMostWaves - 1);
      turn ^= 1;
    }
  }
};

__device__ __forceinline__ float one_over_spread(float sum_of_squares, float per_width, float eps) {
  // v_rsq_f32: within one unit in the last place; eps keeps the argument a normal number
  return __builtin_amdgcn_rsqf(sum_of_squares * per_width + eps);
}

}  // namespace pccl_dev

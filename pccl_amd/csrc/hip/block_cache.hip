// block_cache.hip -- pccl_hip_cache_write, pccl_hip_cache_read: keys and values coded in blocks of 32 elements with
// a shared power-of-two scale as they are written to their pages, and read back through page tables.
//
// Four neighbouring lanes work on one block, eight elements each: 16 bytes of a 16-bit row a load or store, and the block's
// largest magnitude is two data-parallel-primitive steps inside the quad away.  A lane keeps its head and its place in
// the head for all tokens that its wavefront goes through, so that the multiplications which find them (quarter rate) are
// paid once; where a token has 16 blocks or more, a wavefront works on one token at a time and finds slot, page and
// addresses on the scalar unit.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "fold_norm_device.h"

using pccl_host::fail;

namespace pccl_dev {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef unsigned int u32_a1 __attribute__((aligned(1)));

constexpr int kQuad = 4, kPerLane = 8;  // lanes of a block, elements of a lane
constexpr int kWaveBlocks = kWave / kQuad;
constexpr int kWaves = kBlock / kWave;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery's round-up method).
struct Divisor {
  unsigned d, multiplier, shift;
  void set(unsigned by) {
    d = by;
    shift = 0;
    while (shift < 31 && (1u << shift) < by) ++shift;
    multiplier = (unsigned)((((1ull << 32) * ((1ull << shift) - by)) / by) + 1);
  }
  __device__ __forceinline__ unsigned divide(unsigned n) const { return (__umulhi(n, multiplier) + n) >> shift; }
};

// ---- the formats ---------------------------------------------------------------------------------------
// kTop: mantissa bits of the largest value as a binary32, kExponent: its exponent; kBits: of an element.
template <int FMT> struct CacheFormat;
template <> struct CacheFormat<PCCL_CACHE_F8E4M3> {
  static constexpr int kBits = 8, kExponent = 8;
  static constexpr unsigned kTop = 0x600000u;  // 1.75 * 2^8
};
template <> struct CacheFormat<PCCL_CACHE_F8E5M2> {
  static constexpr int kBits = 8, kExponent = 15;
  static constexpr unsigned kTop = 0x600000u;  // 1.75 * 2^15
};
template <> struct CacheFormat<PCCL_CACHE_I8> {
  static constexpr int kBits = 8, kExponent = 0;
  static constexpr unsigned kTop = 0x7e0000u;  // 127/64
};
template <> struct CacheFormat<PCCL_CACHE_F4E2M1> {
  static constexpr int kBits = 4, kExponent = 2;
  static constexpr unsigned kTop = 0x400000u;  // 1.5 * 2^2
};

// A lane's eight codes: two words or one.
template <int BITS> struct LaneCodes { typedef u32x2 type; typedef u32x2_a1 any; };
template <> struct LaneCodes<4> { typedef unsigned type; typedef u32_a1 any; };

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// The 8- and 4-bit floats go through the scaled conversions (v_cvt_scalef32_pk_*): two elements an instruction, the scale's
// exponent byte applied on the way, round to nearest even; checked over every code, scale byte and 16-bit source pattern.  The
// format is a template argument of each, the word half or byte (an immediate) as well.
#define PCCL_PACKED(T, x) __builtin_bit_cast(T, x)
template <int DT, int FMT, int AT>
__device__ __forceinline__ unsigned two_up(unsigned c, float scale) {  // codes AT * 2, AT * 2 + 1 of a word -> two 16-bit elements
  if constexpr (DT == PCCL_BF16) {
    if constexpr (FMT == PCCL_CACHE_F8E4M3) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, scale, AT));
    else if constexpr (FMT == PCCL_CACHE_F8E5M2) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(c, scale, AT));
    else return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, AT));
  } else {
    if constexpr (FMT == PCCL_CACHE_F8E4M3) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, scale, AT));
    else if constexpr (FMT == PCCL_CACHE_F8E5M2) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(c, scale, AT));
    else return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, AT));
  }
}
template <int FMT, int AT>
__device__ __forceinline__ f32x2 two_up_f32(unsigned c, float scale) {
  if constexpr (FMT == PCCL_CACHE_F8E4M3) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, scale, AT);
  else if constexpr (FMT == PCCL_CACHE_F8E5M2) return __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(c, scale, AT);
  else return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, AT);
}
// two 16-bit elements into codes AT * 2, AT * 2 + 1 of word c
template <int DT, int FMT, int AT>
__device__ __forceinline__ unsigned two_down(unsigned c, unsigned w, float scale) {
  if constexpr (DT == PCCL_BF16) {
    const bf16x2 x = PCCL_PACKED(bf16x2, w);
    if constexpr (FMT == PCCL_CACHE_F8E4M3) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(PCCL_PACKED(s16x2, c), x, scale, AT));
    else if constexpr (FMT == PCCL_CACHE_F8E5M2) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(PCCL_PACKED(s16x2, c), x, scale, AT));
    else return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, x, scale, AT);
  } else {
    const f16x2 x = PCCL_PACKED(f16x2, w);
    if constexpr (FMT == PCCL_CACHE_F8E4M3) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(PCCL_PACKED(s16x2, c), x, scale, AT));
    else if constexpr (FMT == PCCL_CACHE_F8E5M2) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(PCCL_PACKED(s16x2, c), x, scale, AT));
    else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, x, scale, AT);
  }
}
template <int FMT, int AT>
__device__ __forceinline__ unsigned two_down_f32(unsigned c, float a, float b, float scale) {
  if constexpr (FMT == PCCL_CACHE_F8E4M3) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(PCCL_PACKED(s16x2, c), a, b, scale, AT));
  else if constexpr (FMT == PCCL_CACHE_F8E5M2) return PCCL_PACKED(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(PCCL_PACKED(s16x2, c), a, b, scale, AT));
  else return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, a, b, scale, AT);
}
#undef PCCL_PACKED

// A lane's eight elements as they stand in memory.
template <class R> struct Eight { u32x4 v[8 / R::kPack]; };

// codes of scale byte s -> elements
template <int DT, int FMT>
__device__ __forceinline__ Eight<RowType<DT>> decode(typename LaneCodes<CacheFormat<FMT>::kBits>::type c, unsigned s) {
  typedef RowType<DT> R;
  Eight<R> e;
  if constexpr (FMT == PCCL_CACHE_I8) {
    // a scale's 64th is exact down to 2^-133, and so is its product with a whole number
    const float step = as_f32(s == 255 ? 0x7fc00000u : s == 0 ? 0x400000u : s << 23) * (1.0f / 64);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(signed char)(c[i / 4] >> (8 * (i % 4))) * step;
#pragma unroll
    for (int j = 0; j < 8 / R::kPack; ++j) e.v[j] = R::down(x + j * R::kPack);
  } else {
    const float scale = as_f32(s << 23);
    unsigned w0, w1;  // words of codes 0-3 and 4-7; the 4-bit codes are all in one
    if constexpr (CacheFormat<FMT>::kBits == 8) w0 = c[0], w1 = c[1];
    else w0 = w1 = c;
    constexpr int kNext = CacheFormat<FMT>::kBits == 8 ? 0 : 2;
    if constexpr (DT == PCCL_F32) {
      const f32x2 a = two_up_f32<FMT, 0>(w0, scale), b = two_up_f32<FMT, 1>(w0, scale);
      const f32x2 d = two_up_f32<FMT, kNext>(w1, scale), f = two_up_f32<FMT, kNext + 1>(w1, scale);
      e.v[0] = u32x4{as_u32(a.x), as_u32(a.y), as_u32(b.x), as_u32(b.y)};
      e.v[1] = u32x4{as_u32(d.x), as_u32(d.y), as_u32(f.x), as_u32(f.y)};
    } else {
      e.v[0] = u32x4{two_up<DT, FMT, 0>(w0, scale), two_up<DT, FMT, 1>(w0, scale), two_up<DT, FMT, kNext>(w1, scale), two_up<DT, FMT, kNext + 1>(w1, scale)};
    }
  }
  return e;
}

// elements of a block with scale byte s -> codes; none passes the format's largest value, and a block of scale 255 has codes 0
template <int DT, int FMT>
__device__ __forceinline__ typename LaneCodes<CacheFormat<FMT>::kBits>::type encode(const Eight<RowType<DT>> &e, unsigned s) {
  typedef RowType<DT> R;
  typename LaneCodes<CacheFormat<FMT>::kBits>::type c{};
  if constexpr (FMT == PCCL_CACHE_I8) {
    float x[8];
    unsigned q[8];
#pragma unroll
    for (int j = 0; j < 8 / R::kPack; ++j) R::up(e.v[j], x + j * R::kPack);
    // 64 x / scale + 1.5 * 2^23 is rounded once, to a whole number, whose low byte is the code
    if (s >= 6 && s < 254) {  // 64 / scale is a binary32, one fused step
      const float f = as_f32((260u - s) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = as_u32(__builtin_fmaf(x[i], f, 12582912.0f));
    } else {  // 1 / scale and 64 apart (exact; a subnormal product rounds to 0 either way); only here a block whose scale would be 2^128 saturates
      const float f = as_f32(s == 254 ? 0x400000u : (254u - s) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = as_u32(__builtin_fmaf(__builtin_amdgcn_fmed3f(x[i] * f, -127.0f / 64, 127.0f / 64), 64.0f, 12582912.0f));
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const unsigned lo = __builtin_amdgcn_perm(q[4 * w + 1], q[4 * w], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[4 * w + 3], q[4 * w + 2], 0x04000c0cu);
      c[w] = s == 255 ? 0 : lo | hi;
    }
  } else {
    const float scale = as_f32(s << 23);
    unsigned w0 = 0, w1 = 0;
    if constexpr (DT == PCCL_F32) {
      const u32x4 a = e.v[0], b = e.v[1];
      w0 = two_down_f32<FMT, 0>(w0, as_f32(a[0]), as_f32(a[1]), scale);
      w0 = two_down_f32<FMT, 1>(w0, as_f32(a[2]), as_f32(a[3]), scale);
      if constexpr (CacheFormat<FMT>::kBits == 8) {
        w1 = two_down_f32<FMT, 0>(w1, as_f32(b[0]), as_f32(b[1]), scale);
        w1 = two_down_f32<FMT, 1>(w1, as_f32(b[2]), as_f32(b[3]), scale);
      } else {
        w0 = two_down_f32<FMT, 2>(w0, as_f32(b[0]), as_f32(b[1]), scale);
        w0 = two_down_f32<FMT, 3>(w0, as_f32(b[2]), as_f32(b[3]), scale);
      }
    } else {
      const u32x4 a = e.v[0];
      const unsigned a0 = a[0], a1 = a[1], a2 = a[2], a3 = a[3];
      w0 = two_down<DT, FMT, 0>(w0, a0, scale);
      w0 = two_down<DT, FMT, 1>(w0, a1, scale);
      if constexpr (CacheFormat<FMT>::kBits == 8) {
        w1 = two_down<DT, FMT, 0>(w1, a2, scale);
        w1 = two_down<DT, FMT, 1>(w1, a3, scale);
      } else {
        w0 = two_down<DT, FMT, 2>(w0, a2, scale);
        w0 = two_down<DT, FMT, 3>(w0, a3, scale);
      }
    }
    if (s == 255) w0 = w1 = 0;
    if constexpr (CacheFormat<FMT>::kBits == 8) c = u32x2{w0, w1};
    else c = w0;
  }
  return c;
}

// binary32 bits of the largest magnitude of a lane's elements; magnitudes compare as whole numbers, infinities and NaN come out on top
template <int DT>
__device__ __forceinline__ unsigned most_of(const Eight<RowType<DT>> &e) {
  if constexpr (DT == PCCL_F32) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max(m, e.v[j][i] & 0x7fffffffu);
    return m;
  } else {
    const u32x4 v = e.v[0] & 0x7fff7fffu;
    const unsigned v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
    const u16x2 a = __builtin_elementwise_max(__builtin_bit_cast(u16x2, v0), __builtin_bit_cast(u16x2, v1));
    const u16x2 b = __builtin_elementwise_max(__builtin_bit_cast(u16x2, v2), __builtin_bit_cast(u16x2, v3));
    const u16x2 m = __builtin_elementwise_max(a, b);
    return as_u32(RowType<DT>::up1(max(m.x, m.y)));
  }
}

__device__ __forceinline__ unsigned quad_max(unsigned m) {
  m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

// Scale byte of a block from the bits of its largest magnitude: the exponent, one more if the mantissa is beyond that of the
// format's largest value, less that value's exponent.
template <class F>
__device__ __forceinline__ unsigned scale_of(unsigned most) {
  int s = (int)((most + (0x7fffffu - F::kTop)) >> 23) - F::kExponent;
  // a subnormal's mantissa counts from 2^-127 up, not from its leading bit: only a format whose exponent is 0 gets above 0 there
  if (F::kExponent == 0 && most < 0x800000u) s = most > ((F::kTop + 0x800000u) >> 1) ? 1 : 0;
  s = s < 0 ? 0 : s > 254 ? 254 : s;
  return most >= 0x7f800000u ? 255u : (unsigned)s;
}

struct CacheArgs {
  char *codes[PCCL_CACHE_MAX_TENSORS], *scales[PCCL_CACHE_MAX_TENSORS];
  long code_page, code_token, code_head, scale_page, scale_token, scale_head;
  long row_head;            // bytes from one head of a source or output row to the next
  int head_dim;
  unsigned blocks;          // of a token: heads times blocks of a head
  unsigned group;           // tokens that a wavefront has side by side (1 from 16 blocks on)
  Divisor by_blocks, head_blocks, page_tokens, chunks;  // blocks of a token; of a head; tokens of a page; wavefronts' shares of a token
};

// Where a lane stands: its token among those side by side, its head's and block's offsets.
struct Place {
  bool on;
  unsigned token, block;
  int n, q;               // elements inside the head (0..8), lane of the quad
  long code, scale, row;  // bytes behind the token's start
};
template <bool ONE>  // one token at a time
__device__ __forceinline__ Place place_of(const CacheArgs &a, unsigned chunk, int bits, int elem_bytes) {
  Place p;
  const unsigned lane = threadIdx.x % kWave, at = lane / kQuad;
  p.q = (int)(lane % kQuad);
  p.token = ONE ? 0 : a.by_blocks.divide(at);
  const unsigned r = ONE ? chunk * kWaveBlocks + at : at - p.token * a.blocks;
  p.on = ONE ? r < a.blocks : p.token < a.group;
  const unsigned head = a.head_blocks.divide(r);
  p.block = r - head * a.head_blocks.d;
  const int first = (int)p.block * PCCL_CACHE_BLOCK + p.q * kPerLane;
  p.n = min(max(a.head_dim - first, 0), kPerLane);
  p.code = (long)head * a.code_head + first * bits / 8;
  p.scale = (long)head * a.scale_head + p.block;
  p.row = (long)head * a.row_head + first * elem_bytes;
  return p;
}

// eight elements from `at` on, n of them there, zeros behind
template <class R>
__device__ __forceinline__ Eight<R> load_eight(const char *at, int n) {
  Eight<R> e;
#pragma unroll
  for (int j = 0; j < 8 / R::kPack; ++j) {
    if (n == 8) {
      e.v[j] = ((const typename R::pack_t *)at)[j];
    } else {
      typename R::elem_t x[R::kPack];
#pragma unroll
      for (int i = 0; i < R::kPack; ++i) x[i] = j * R::kPack + i < n ? ((const typename R::elem_t *)at)[j * R::kPack + i] : (typename R::elem_t)0;
      e.v[j] = __builtin_bit_cast(u32x4, x);
    }
  }
  return e;
}
template <class R>
__device__ __forceinline__ void store_eight(char *at, int n, const Eight<R> &e) {
#pragma unroll
  for (int j = 0; j < 8 / R::kPack; ++j) {
    if (n == 8) {
      ((typename R::pack_t *)at)[j] = e.v[j];
    } else {
#pragma unroll
      for (int i = 0; i < R::kPack; ++i)
        if (j * R::kPack + i < n) {
          const unsigned w = e.v[j][i * R::kBytes / 4];
          ((typename R::elem_t *)at)[j * R::kPack + i] = (typename R::elem_t)(R::kBytes == 2 && i % 2 ? w >> 16 : w);
        }
    }
  }
}

struct WriteArgs : CacheArgs {
  const char *srcs[PCCL_CACHE_MAX_TENSORS];
  long src_token;  // bytes
  const long *slots;
  unsigned long n_slots;
  unsigned tokens;  // of the launch
};

template <int DT, int FMT, int TIMES, bool ONE>
__global__ void __launch_bounds__(kBlock) cache_write_kernel(const WriteArgs a) {
  typedef RowType<DT> R;
  typedef CacheFormat<FMT> F;
  typedef LaneCodes<F::kBits> L;
  const unsigned wave = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const unsigned tile = a.chunks.divide(wave), chunk = wave - tile * a.chunks.d;
  const unsigned token0 = tile * TIMES * a.group;
  if (token0 >= a.tokens) return;
  const Place p = place_of<ONE>(a, chunk, F::kBits, R::kBytes);
  const char *src = a.srcs[blockIdx.y];
  char *codes = a.codes[blockIdx.y], *scales = a.scales[blockIdx.y];
  unsigned long slot[TIMES];
  Eight<R> e[TIMES];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned token = token0 + t * a.group + p.token;
    const bool there = token < a.tokens;
    slot[t] = (unsigned long)a.slots[there ? token : 0];  // (no branch around the load: all of them go out together)
    if (!there) slot[t] = ~0ul;
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t)
    if (slot[t] < a.n_slots && p.on) e[t] = load_eight<R>(src + (unsigned long)(token0 + t * a.group + p.token) * a.src_token + p.row, p.n);
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    if (slot[t] >= a.n_slots || !p.on) continue;  // whole quads
    const unsigned s = scale_of<F>(quad_max(most_of<DT>(e[t])));
    const typename L::type c = encode<DT, FMT>(e[t], s);
    const unsigned page = a.page_tokens.divide((unsigned)slot[t]), token = (unsigned)slot[t] - page * a.page_tokens.d;
    char *to = codes + ((unsigned long)page * a.code_page + (unsigned long)token * a.code_token) + p.code;
    if (p.n == 8) {
      *(typename L::any *)to = c;
    } else {
      const int bytes = (p.n * F::kBits + 7) / 8;
#pragma unroll
      for (int i = 0; i < F::kBits; ++i) {
        unsigned w;
        if constexpr (F::kBits == 8) w = c[i / 4];
        else w = c;
        if (i < bytes) to[i] = (char)(w >> (8 * (i % 4)));
      }
    }
    if (p.q == 0) scales[((unsigned long)page * a.scale_page + (unsigned long)token * a.scale_token) + p.scale] = (char)s;
  }
}

struct ReadArgs : CacheArgs {
  char *outs[PCCL_CACHE_MAX_TENSORS];
  long out_token;  // bytes
  long out_rows, max_len, table_stride, n_pages;
  const int *page_table, *lengths;
  const long *row_start;
  unsigned token0;  // the launch's first token of every sequence
  int seq0;
};

template <int DT, int FMT, int TIMES, bool ONE>
__global__ void __launch_bounds__(kBlock) cache_read_kernel(const ReadArgs a) {
  typedef RowType<DT> R;
  typedef CacheFormat<FMT> F;
  typedef LaneCodes<F::kBits> L;
  const long seq = a.seq0 + (long)blockIdx.y;
  const unsigned wave = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const unsigned tile = a.chunks.divide(wave), chunk = wave - tile * a.chunks.d;
  const unsigned long token0 = a.token0 + (unsigned long)tile * TIMES * a.group;
  long length = a.lengths[seq];
  if (length > a.max_len) length = a.max_len;
  if ((long)token0 >= length) return;
  const Place p = place_of<ONE>(a, chunk, F::kBits, R::kBytes);
  const char *codes = a.codes[blockIdx.z], *scales = a.scales[blockIdx.z];
  char *out = a.outs[blockIdx.z];
  const long first_row = a.row_start ? a.row_start[seq] : seq * a.max_len;
  const int *table = a.page_table + seq * a.table_stride;
  unsigned long page[TIMES];
  typename L::type c[TIMES];
  unsigned s[TIMES];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned pos = (unsigned)token0 + t * a.group + p.token, entry = a.page_tokens.divide(pos);
    const bool named = (long)pos < length && (long)entry < a.table_stride && (unsigned long)(first_row + pos) < (unsigned long)a.out_rows;
    page[t] = (unsigned long)(long)table[named ? entry : 0];  // (no branch around the load: all of them go out together)
    if (!named) page[t] = ~0ul;
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    if (page[t] >= (unsigned long)a.n_pages || !p.on) continue;
    const unsigned pos = (unsigned)token0 + t * a.group + p.token, token = pos - a.page_tokens.divide(pos) * a.page_tokens.d;
    const char *from = codes + (page[t] * a.code_page + (unsigned long)token * a.code_token) + p.code;
    s[t] = (unsigned char)(scales + (page[t] * a.scale_page + (unsigned long)token * a.scale_token))[p.scale];
    if (p.n == 8) {
      c[t] = *(const typename L::any *)from;
    } else {
      const int bytes = (p.n * F::kBits + 7) / 8;
      unsigned w[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < F::kBits; ++i)
        if (i < bytes) w[i / 4] |= (unsigned)(unsigned char)from[i] << (8 * (i % 4));
      if constexpr (F::kBits == 8) c[t] = u32x2{w[0], w[1]};
      else c[t] = w[0];
    }
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    if (page[t] >= (unsigned long)a.n_pages || !p.on) continue;
    const unsigned pos = (unsigned)token0 + t * a.group + p.token;
    store_eight<R>(out + (unsigned long)(first_row + pos) * a.out_token + p.row, p.n, decode<DT, FMT>(c[t], s[t]));
  }
}

}  // namespace pccl_dev

using namespace pccl_dev;

namespace {

// Strides of a tensor whose heads start at page * s[0] + token * s[1] + head * s[2], `bytes` bytes each: they keep the
// heads apart if, from the smallest stride to the largest, each covers what lies inside of it.
bool apart(const long (&count)[3], const long (&stride)[3], long bytes) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
  long extent = bytes;
  for (int k : order) {
    if (count[k] <= 1) continue;
    if (stride[k] < extent) return false;
    extent += (count[k] - 1) * stride[k];
  }
  return true;
}

int check_cache(const pccl_cache_desc *c, int dtype, const void *const *tensors, const char *what, CacheArgs *a) {
  if (!c) return fail(PCCL_ERR_INVALID_ARG, "cache: description is null");
  if (c->format < PCCL_CACHE_F8E4M3 || c->format > PCCL_CACHE_F4E2M1) return fail(PCCL_ERR_UNSUPPORTED, "unknown cache format %d", c->format);
  if (dtype != PCCL_F32 && dtype != PCCL_BF16 && dtype != PCCL_F16) return fail(PCCL_ERR_UNSUPPORTED, "cache: rows of dtype code %d", dtype);
  if (c->n_tensors < 1 || c->n_tensors > PCCL_CACHE_MAX_TENSORS) return fail(PCCL_ERR_INVALID_ARG, "n_tensors %d outside [1, 8]", c->n_tensors);
  if (c->heads < 1 || c->heads > 65536 || c->head_dim < 1 || c->head_dim > 65536)
    return fail(PCCL_ERR_INVALID_ARG, "heads %d or head_dim %d outside [1, 65536]", c->heads, c->head_dim);
  if (c->page_tokens < 1 || c->page_tokens > (1l << 20)) return fail(PCCL_ERR_INVALID_ARG, "page_tokens %ld outside [1, 2^20]", c->page_tokens);
  if (c->n_pages < 0 || c->n_pages > 0x7fffffffl / c->page_tokens)
    return fail(PCCL_ERR_INVALID_ARG, "%ld pages of %ld tokens: below 0 or more than 2^31 - 1 tokens", c->n_pages, c->page_tokens);
  const int bits = c->format == PCCL_CACHE_F4E2M1 ? 4 : 8;
  const int blocks = (c->head_dim + PCCL_CACHE_BLOCK - 1) / PCCL_CACHE_BLOCK;
  const long counts[3] = {c->n_pages, c->page_tokens, c->heads};
  for (long s : {c->code_page, c->code_token, c->code_head, c->scale_page, c->scale_token, c->scale_head})
    if (s < 0 || s > (1l << 40)) return fail(PCCL_ERR_INVALID_ARG, "cache stride %ld outside [0, 2^40]", s);
  if (!apart(counts, {c->code_page, c->code_token, c->code_head}, (c->head_dim * bits + 7) / 8))
    return fail(PCCL_ERR_INVALID_ARG, "code strides %ld, %ld, %ld let heads overlap", c->code_page, c->code_token, c->code_head);
  if (!apart(counts, {c->scale_page, c->scale_token, c->scale_head}, blocks))
    return fail(PCCL_ERR_INVALID_ARG, "scale strides %ld, %ld, %ld let heads overlap", c->scale_page, c->scale_token, c->scale_head);
  if (!tensors) return fail(PCCL_ERR_INVALID_ARG, "array of %s is null", what);
  const int es = pccl_host::pccl_dtype_bytes(dtype);
  memset((void *)a, 0, sizeof(*a));
  for (int k = 0; k < c->n_tensors; ++k) {
    if (c->n_pages && (!c->codes[k] || !c->scales[k])) return fail(PCCL_ERR_INVALID_ARG, "codes or scales of tensor %d are null", k);
    if ((uintptr_t)tensors[k] % es) return fail(PCCL_ERR_MISALIGNED, "%s %d (%p) not %d-byte aligned", what, k, tensors[k], es);
    a->codes[k] = (char *)c->codes[k];
    a->scales[k] = (char *)c->scales[k];
  }
  a->code_page = c->code_page;
  a->code_token = c->code_token;
  a->code_head = c->code_head;
  a->scale_page = c->scale_page;
  a->scale_token = c->scale_token;
  a->scale_head = c->scale_head;
  a->head_dim = c->head_dim;
  a->blocks = (unsigned)c->heads * (unsigned)blocks;  // at most 2^27
  a->group = std::max(1u, kWaveBlocks / a->blocks);
  a->by_blocks.set(a->blocks);
  a->head_blocks.set((unsigned)blocks);
  a->page_tokens.set((unsigned)c->page_tokens);
  a->chunks.set(a->group > 1 ? 1 : (a->blocks + kWaveBlocks - 1) / kWaveBlocks);
  return PCCL_OK;
}

template <class F>
void with_types(int dtype, int format, F &&f) {
  auto of_format = [&](auto t) {
    switch (format) {
      case PCCL_CACHE_F8E4M3: f(t, std::integral_constant<int, PCCL_CACHE_F8E4M3>{}); break;
      case PCCL_CACHE_F8E5M2: f(t, std::integral_constant<int, PCCL_CACHE_F8E5M2>{}); break;
      case PCCL_CACHE_I8: f(t, std::integral_constant<int, PCCL_CACHE_I8>{}); break;
      default: f(t, std::integral_constant<int, PCCL_CACHE_F4E2M1>{}); break;
    }
  };
  if (dtype == PCCL_F32) of_format(std::integral_constant<int, PCCL_F32>{});
  else if (dtype == PCCL_BF16) of_format(std::integral_constant<int, PCCL_BF16>{});
  else of_format(std::integral_constant<int, PCCL_F16>{});
}

constexpr int kTimes = 4;  // groups of tokens that a wavefront has in flight where there are enough of them

// whether n wavefronts' worth of tokens give every compute unit eight workgroups of kTimes groups a wavefront
bool many(long n) { return n >= (long)pccl_host::compute_units() * 8 * kWaves * kTimes; }

// Tokens of a launch: wavefronts stay below 2^26 (a grid times its lanes must fit 32 bits) and below what Divisor divides.
long launch_tokens(const CacheArgs &a) { return std::max(1l, (1l << 26) / a.chunks.d); }

// Workgroups of a launch over n tokens.
unsigned workgroups(const CacheArgs &a, long tokens, int times) {
  const long tiles = (tokens + (long)times * a.group - 1) / ((long)times * a.group);
  return (unsigned)((tiles * a.chunks.d + kWaves - 1) / kWaves);
}

// Calls f(times, one token at a time) with both as constants.
template <class F>
void with_shape(bool four, bool one, F &&f) {
  typedef std::integral_constant<int, kTimes> Four;
  typedef std::integral_constant<int, 1> Once;
  if (four) one ? f(Four{}, std::true_type{}) : f(Four{}, std::false_type{});
  else one ? f(Once{}, std::true_type{}) : f(Once{}, std::false_type{});
}

int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PCCL_OK : fail(PCCL_ERR_HIP, "%s launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" int pccl_hip_cache_write(const pccl_cache_desc *c, int dtype, const void *const *srcs, long src_token_stride, long src_head_stride,
                                    const long *slots, long tokens, void *stream) {
  pccl_host::clear_error();
  WriteArgs a;
  int rc = check_cache(c, dtype, srcs, "source", &a);
  if (rc != PCCL_OK) return rc;
  if (tokens < 0 || tokens > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "tokens %ld outside [0, 2^31)", tokens);
  if (src_token_stride < 0 || src_head_stride < 0)
    return fail(PCCL_ERR_INVALID_ARG, "source strides %ld, %ld below 0", src_token_stride, src_head_stride);
  if ((uintptr_t)slots % 8) return fail(PCCL_ERR_MISALIGNED, "slots (%p) not 8-byte aligned", (const void *)slots);
  if (tokens && !slots) return fail(PCCL_ERR_INVALID_ARG, "slots are null");
  for (int k = 0; k < c->n_tensors; ++k)
    if (tokens && !srcs[k]) return fail(PCCL_ERR_INVALID_ARG, "source %d is null", k);
  rc = pccl_host::check_stream(stream);
  if (rc != PCCL_OK) return rc;
  if (tokens == 0 || c->n_pages == 0) return PCCL_OK;
  const int es = pccl_host::pccl_dtype_bytes(dtype);
  a.src_token = src_token_stride * es;
  a.row_head = src_head_stride * es;
  a.n_slots = (unsigned long)(c->n_pages * c->page_tokens);
  const long most = launch_tokens(a);
  for (long lo = 0; lo < tokens; lo += most) {
    const long n = std::min(most, tokens - lo);
    for (int k = 0; k < c->n_tensors; ++k) a.srcs[k] = (const char *)srcs[k] + lo * a.src_token;
    a.slots = slots + lo;
    a.tokens = (unsigned)n;
    const bool four = many((n + a.group - 1) / a.group * a.chunks.d * c->n_tensors);
    with_types(dtype, c->format, [&](auto t, auto f) {
      with_shape(four, a.group == 1, [&](auto times, auto one) {
        hipLaunchKernelGGL((cache_write_kernel<decltype(t)::value, decltype(f)::value, decltype(times)::value, decltype(one)::value>),
                           dim3(workgroups(a, n, decltype(times)::value), c->n_tensors), dim3(kBlock), 0, (hipStream_t)stream, a);
      });
    });
    rc = launched("cache_write");
    if (rc != PCCL_OK) return rc;
  }
  return PCCL_OK;
}

extern "C" int pccl_hip_cache_read(const pccl_cache_desc *c, int dtype, void *const *outs, long out_token_stride, long out_head_stride,
                                   long out_rows, const int *page_table, long table_stride, const int *lengths, const long *row_start,
                                   int n_seq, long max_len, void *stream) {
  pccl_host::clear_error();
  ReadArgs a;
  int rc = check_cache(c, dtype, (const void *const *)outs, "output", &a);
  if (rc != PCCL_OK) return rc;
  if (n_seq < 0) return fail(PCCL_ERR_INVALID_ARG, "n_seq %d < 0", n_seq);
  if (max_len < 0 || max_len > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "max_len %ld outside [0, 2^31)", max_len);
  if (out_rows < 0 || table_stride < 0) return fail(PCCL_ERR_INVALID_ARG, "out_rows %ld or table_stride %ld below 0", out_rows, table_stride);
  if (out_token_stride < 0 || out_head_stride < 0 || out_token_stride > (1l << 40) || out_head_stride > (1l << 40))
    return fail(PCCL_ERR_INVALID_ARG, "output strides %ld, %ld outside [0, 2^40]", out_token_stride, out_head_stride);
  if (!apart({1, out_rows, c->heads}, {0, out_token_stride, out_head_stride}, c->head_dim))
    return fail(PCCL_ERR_INVALID_ARG, "output strides %ld, %ld let heads overlap", out_token_stride, out_head_stride);
  if ((uintptr_t)page_table % 4 || (uintptr_t)lengths % 4 || (uintptr_t)row_start % 8)
    return fail(PCCL_ERR_MISALIGNED, "page_table, lengths or row_start not aligned to their elements");
  const bool nothing = n_seq == 0 || max_len == 0 || out_rows == 0 || table_stride == 0 || c->n_pages == 0;
  if (!nothing && (!page_table || !lengths)) return fail(PCCL_ERR_INVALID_ARG, "page_table or lengths are null");
  for (int k = 0; k < c->n_tensors; ++k)
    if (!nothing && !outs[k]) return fail(PCCL_ERR_INVALID_ARG, "output %d is null", k);
  rc = pccl_host::check_stream(stream);
  if (rc != PCCL_OK || nothing) return rc;
  const int es = pccl_host::pccl_dtype_bytes(dtype);
  for (int k = 0; k < c->n_tensors; ++k) a.outs[k] = (char *)outs[k];
  a.out_token = out_token_stride * es;
  a.row_head = out_head_stride * es;
  a.out_rows = out_rows;
  a.max_len = max_len;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.row_start = row_start;
  a.n_pages = c->n_pages;
  const long most = launch_tokens(a);
  for (int seq = 0; seq < n_seq; seq += 65535) {
    a.seq0 = seq;
    const int seqs = std::min(65535, n_seq - seq);
    for (long lo = 0; lo < max_len; lo += most) {
      a.token0 = (unsigned)lo;
      const long n = std::min(most, max_len - lo);
      const bool four = many((n + a.group - 1) / a.group * a.chunks.d * seqs * c->n_tensors);
      with_types(dtype, c->format, [&](auto t, auto f) {
        with_shape(four, a.group == 1, [&](auto times, auto one) {
          hipLaunchKernelGGL((cache_read_kernel<decltype(t)::value, decltype(f)::value, decltype(times)::value, decltype(one)::value>),
                             dim3(workgroups(a, n, decltype(times)::value), seqs, c->n_tensors), dim3(kBlock), 0, (hipStream_t)stream, a);
        });
      });
      rc = launched("cache_read");
      if (rc != PCCL_OK) return rc;
    }
  }
  return PCCL_OK;
}

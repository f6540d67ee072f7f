// block_cache.hip -- pccl_hip_cache_write, pccl_hip_cache_read: keys and values coded in blocks of 32 elements with
// a shared power-of-two scale as they are written to their pages, and read back through page tables.
//
// A lane works on 16 bytes of a row: four neighbouring lanes on one block of a 16-bit row, eight on one of binary32, so that the
// block's largest magnitude is two or three data-parallel-primitive steps away.  A lane keeps its head and its place in
// the head for all tokens that its wavefront goes through, so that the multiplications which find them (quarter rate) are
// paid once; where a token fills a wavefront, it works on one token at a time and finds slot, page and
// addresses on the scalar unit.  (Reading needs no block's lanes side by side: there a short last block takes only the lanes it fills.)
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "fold_norm_device.h"
#include "pieces.h"

using pccl_host::fail;

namespace pccl_dev {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef unsigned int u32_a1 __attribute__((aligned(1)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
typedef unsigned int u32_a2 __attribute__((aligned(2)));
typedef unsigned short u16_a1 __attribute__((aligned(1)));

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

// A lane's codes: eight of 8 bits in two words, or as many as there are in the low bits of one.
template <int BITS> struct LaneCodes { typedef unsigned type; };
template <> struct LaneCodes<64> { typedef u32x2 type; };
template <int BITS> struct StoredCodes;
template <> struct StoredCodes<64> { typedef u32x2_a1 type; };
template <> struct StoredCodes<32> { typedef u32_a1 type; };
template <> struct StoredCodes<16> { typedef u16_a1 type; };

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

template <int DT, int FMT>
struct Lane {
  typedef RowType<DT> R;
  static constexpr int kElems = R::kPack, kBits = kElems * CacheFormat<FMT>::kBits;
  static constexpr int kBlockLanes = PCCL_CACHE_BLOCK / kElems;
  typedef typename LaneCodes<kBits>::type Codes;

  // codes of scale byte s -> elements as they stand in memory
  static __device__ __forceinline__ u32x4 decode(Codes c, unsigned s) {
    unsigned w0, w1;  // the words that elements 0-3 and 4-7 are in
    if constexpr (kBits == 64) w0 = c[0], w1 = c[1];
    else w0 = w1 = c;
    if constexpr (FMT == PCCL_CACHE_I8) {
      // a scale's 64th is exact down to 2^-133, and so is its product with a whole number
      const float step = as_f32(s == 255 ? 0x7fc00000u : s == 0 ? 0x400000u : s << 23) * (1.0f / 64);
      float x[kElems];
#pragma unroll
      for (int i = 0; i < kElems; ++i) x[i] = (float)(signed char)((i < 4 ? w0 : w1) >> (8 * (i % 4))) * step;
      return R::down(x);
    } else {
      const float scale = as_f32(s << 23);
      if constexpr (DT == PCCL_F32) {
        const f32x2 a = two_up_f32<FMT, 0>(w0, scale), b = two_up_f32<FMT, 1>(w0, scale);
        return u32x4{as_u32(a.x), as_u32(a.y), as_u32(b.x), as_u32(b.y)};
      } else {
        constexpr int kNext = kBits == 64 ? 0 : 2;
        return u32x4{two_up<DT, FMT, 0>(w0, scale), two_up<DT, FMT, 1>(w0, scale), two_up<DT, FMT, kNext>(w1, scale), two_up<DT, FMT, kNext + 1>(w1, scale)};
      }
    }
  }

  // elements of a block with scale byte s -> codes; none passes the format's largest value, and a block of scale 255 has codes 0
  static __device__ __forceinline__ Codes encode(u32x4 v, unsigned s) {
    unsigned w0 = 0, w1 = 0;
    if constexpr (FMT == PCCL_CACHE_I8) {
      float x[kElems];
      unsigned q[kElems];
      R::up(v, x);
      // 64 x / scale + 1.5 * 2^23 is rounded once, to a whole number, whose low byte is the code
      if (s >= 6 && s < 254) {  // 64 / scale is a binary32: one fused step
        const float f = as_f32((260u - s) << 23);
#pragma unroll
        for (int i = 0; i < kElems; ++i) q[i] = as_u32(__builtin_fmaf(x[i], f, 12582912.0f));
      } else {  // 1 / scale and 64 apart (exact; a subnormal product rounds to 0 either way); only here a block whose scale would be 2^128 saturates
        const float f = as_f32(s == 254 ? 0x400000u : (254u - s) << 23);
#pragma unroll
        for (int i = 0; i < kElems; ++i) q[i] = as_u32(__builtin_fmaf(__builtin_amdgcn_fmed3f(x[i] * f, -127.0f / 64, 127.0f / 64), 64.0f, 12582912.0f));
      }
      w0 = __builtin_amdgcn_perm(q[1], q[0], 0x0c0c0400u) | __builtin_amdgcn_perm(q[3], q[2], 0x04000c0cu);
      if constexpr (kElems == 8) w1 = __builtin_amdgcn_perm(q[5], q[4], 0x0c0c0400u) | __builtin_amdgcn_perm(q[7], q[6], 0x04000c0cu);
    } else {
      const float scale = as_f32(s << 23);
      const unsigned v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
      if constexpr (DT == PCCL_F32) {
        w0 = two_down_f32<FMT, 0>(w0, as_f32(v0), as_f32(v1), scale);
        w0 = two_down_f32<FMT, 1>(w0, as_f32(v2), as_f32(v3), scale);
      } else {
        w0 = two_down<DT, FMT, 0>(w0, v0, scale);
        w0 = two_down<DT, FMT, 1>(w0, v1, scale);
        if constexpr (kBits == 64) {
          w1 = two_down<DT, FMT, 0>(w1, v2, scale);
          w1 = two_down<DT, FMT, 1>(w1, v3, scale);
        } else {
          w0 = two_down<DT, FMT, 2>(w0, v2, scale);
          w0 = two_down<DT, FMT, 3>(w0, v3, scale);
        }
      }
    }
    if (s == 255) w0 = w1 = 0;
    if constexpr (kBits == 64) return u32x2{w0, w1};
    else return w0;
  }

  // The last piece of a head may be short (n elements of kElems, none for a lane behind it).  It is loaded as the whole piece that ends
  // with the head and shifted down, where the head is long enough for that (`long_head`), and stored as pieces of 8, 4, 2 and 1
  // bytes: element by element the one short piece of an odd head cost as much as all the others together.
  static __device__ __forceinline__ Codes load_codes(const char *at, int n, bool long_head) {
    typedef typename StoredCodes<kBits>::type T;
    if (n == kElems) return *(const T *)at;
    const int bytes = (n * CacheFormat<FMT>::kBits + 7) / 8;
    if (long_head) {
      const Codes c = *(const T *)(at + bytes - kBits / 8);
      if constexpr (kBits == 64) {
        const unsigned long w = __builtin_bit_cast(unsigned long, c) >> (8 * (8 - bytes));
        return __builtin_bit_cast(u32x2, w);
      } else {
        return c >> (8 * (kBits / 8 - bytes));
      }
    }
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kBits / 8; ++i)
      if (i < bytes) w[i / 4] |= (unsigned)(unsigned char)at[i] << (8 * (i % 4));
    if constexpr (kBits == 64) return u32x2{w[0], w[1]};
    else return w[0];
  }
  static __device__ __forceinline__ void store_codes(char *at, int n, Codes c) {
    const int bytes = (n * CacheFormat<FMT>::kBits + 7) / 8;
    if (bytes == kBits / 8) {  // (with 4-bit codes also where the last code's half of the byte is empty)
      typedef typename StoredCodes<kBits>::type T;
      __builtin_nontemporal_store((T)c, (T *)at);
    } else {
      unsigned w;  // what is left to store
      if constexpr (kBits == 64) w = bytes & 4 ? c[1] : c[0];
      else w = c;
      if constexpr (kBits == 64) {
        if (bytes & 4) {
          const unsigned first = c[0];
          *(u32_a1 *)at = first;
          at += 4;
        }
      }
      if (bytes & 2) {
        *(u16_a1 *)at = (unsigned short)w;
        at += 2;
        w >>= 16;
      }
      if (bytes & 1) *at = (char)w;
    }
  }
  // elements from `at` on, n of them there, zeros behind
  template <bool STREAM> static __device__ __forceinline__ u32x4 load(const char *at, int n, bool long_head) {
    typedef typename R::pack_t T;
    if (n == kElems) {
      if constexpr (STREAM) return __builtin_nontemporal_load((const T *)at);
      else return *(const T *)at;
    }
    if (n > 0 && long_head) {
      u32x4 v = *(const T *)(at + (n - kElems) * R::kBytes);
      const int skip = (kElems - n) * R::kBytes;  // bytes to shift down by: 8, 4 and 2 of them
      if (skip & 8) v = u32x4{v[2], v[3], 0, 0};
      if (skip & 4) v = u32x4{v[1], v[2], v[3], 0};
      if (R::kBytes == 2 && (skip & 2))
        v = u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], 2), __builtin_amdgcn_alignbyte(v[2], v[1], 2), __builtin_amdgcn_alignbyte(v[3], v[2], 2), v[3] >> 16};
      return v;
    }
    typename R::elem_t x[kElems];
#pragma unroll
    for (int i = 0; i < kElems; ++i) x[i] = i < n ? ((const typename R::elem_t *)at)[i] : (typename R::elem_t)0;
    return __builtin_bit_cast(u32x4, x);
  }
  static __device__ __forceinline__ void store(char *at, int n, u32x4 v) {
    if (n == kElems) {
      __builtin_nontemporal_store(v, (typename R::pack_t *)at);
    } else {
      const int bytes = n * R::kBytes;
      if (bytes & 8) {
        *(u32x2_a2 *)at = u32x2{v[0], v[1]};
        at += 8;
      }
      unsigned w = bytes & 8 ? v[2] : v[0];
      const unsigned after = bytes & 8 ? v[3] : v[1];
      if (bytes & 4) {
        *(u32_a2 *)at = w;
        at += 4;
        w = after;
      }
      if (R::kBytes == 2 && (bytes & 2)) *(unsigned short *)at = (unsigned short)w;
    }
  }
};

// binary32 bits of the largest magnitude of a lane's elements; magnitudes compare as whole numbers, infinities and NaN come out on top
template <int DT>
__device__ __forceinline__ unsigned most_of(u32x4 v) {
  if constexpr (DT == PCCL_F32) {
    v &= 0x7fffffffu;
    return max(max(v[0], v[1]), max(v[2], v[3]));
  } else {
    v &= 0x7fff7fffu;
    const unsigned v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
    const u16x2 a = __builtin_elementwise_max(__builtin_bit_cast(u16x2, v0), __builtin_bit_cast(u16x2, v1));
    const u16x2 b = __builtin_elementwise_max(__builtin_bit_cast(u16x2, v2), __builtin_bit_cast(u16x2, v3));
    const u16x2 m = __builtin_elementwise_max(a, b);
    return as_u32(RowType<DT>::up1(max(m.x, m.y)));
  }
}

// the largest of a block's 4 or 8 lanes, in each of them
template <int LANES>
__device__ __forceinline__ unsigned block_max(unsigned m) {
  m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  if constexpr (LANES == 8) m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, true));  // row_half_mirror
  return m;
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
  long code_head, scale_head;
  unsigned code_page, code_token, scale_page, scale_token;  // (a 32-bit product is two scalar multiplications, a 64-bit one six)
  long row_head;            // bytes from one head of a source or output row to the next
  int head_dim;
  unsigned group;           // tokens that a wavefront has side by side
  int parts;                // 16-byte pieces of a token that a lane has (see Place)
  Divisor token_lanes, head_lanes, page_tokens, chunks;  // lanes that a token and a head take; tokens of a page; wavefronts' shares of a token
};

// Where a lane stands: its token among those side by side, its head's and block's offsets.  PARTS: 16-byte pieces of a token that a
// lane has, 64 lanes apart; 0: the token has room for others beside it.
struct Place {
  bool on;
  unsigned token;
  int n, first;           // elements inside the head, the first of them
  long code, scale, row;  // bytes behind the token's start
};
template <class L, int PARTS, int REPEAT>
__device__ __forceinline__ Place place_of(const CacheArgs &a, unsigned chunk, int part) {
  Place p;
  const unsigned lane = threadIdx.x % kWave;
  p.token = PARTS ? 0 : a.token_lanes.divide(lane);
  unsigned r = PARTS ? (chunk * PARTS + part) * kWave + lane : lane - p.token * a.token_lanes.d;
  p.on = PARTS ? (chunk * PARTS + part) * kWave < a.token_lanes.d : p.token < a.group;
  // lanes behind the token's last do what its last block's (or last) lanes do, to the same bytes: the wavefront stays whole
  if (PARTS && r >= a.token_lanes.d) r = a.token_lanes.d - REPEAT + r % REPEAT;
  const unsigned head = a.head_lanes.divide(r);
  p.first = (int)(r - head * a.head_lanes.d) * L::kElems;
  p.n = min(max(a.head_dim - p.first, 0), L::kElems);
  p.code = (long)head * a.code_head + p.first / L::kElems * (L::kBits / 8);
  p.scale = (long)head * a.scale_head + p.first / PCCL_CACHE_BLOCK;
  p.row = (long)head * a.row_head + p.first * L::R::kBytes;
  return p;
}

__device__ __forceinline__ unsigned long times(unsigned a, unsigned b) { return (unsigned long)a * b; }

// How much of a wavefront's work may be missing.  kAny: tokens, lanes, the ends of pieces.  kEven: heads are whole pieces, so a lane has
// its piece or nothing, under one mask.  kWhole: every lane has a piece of every token; no mask and no branch.  The scalar unit, one
// instruction a clock for a compute unit's 32 wavefronts, is what the masks of the general form keep busy (4-bit read of
// 131072 tokens x 8 x 128 x 2: 143 us without kWhole, 120 with it).
constexpr int kAny = 0, kEven = 1, kWhole = 2;
template <class L, int PARTS>
__device__ __forceinline__ bool all_whole(const Place (&p)[PARTS]) {
  bool whole = true;
#pragma unroll
  for (int h = 0; h < PARTS; ++h) whole = whole && p[h].on && p[h].n == L::kElems;
  return __builtin_amdgcn_ballot_w64(whole) == ~0ull;
}

struct WriteArgs : CacheArgs {
  const char *srcs[PCCL_CACHE_MAX_TENSORS];
  unsigned src_token;  // bytes
  const long *slots;
  unsigned long n_slots;
  unsigned tokens;  // of the launch
};

template <int DT, int FMT, int TIMES, int PARTS, bool STREAM>
__global__ void __launch_bounds__(kBlock) cache_write_kernel(const WriteArgs a) {
  typedef Lane<DT, FMT> L;
  constexpr int kParts = PARTS ? PARTS : 1;
  const unsigned wave = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const unsigned tile = a.chunks.divide(wave), chunk = wave - tile * a.chunks.d;
  const unsigned token0 = tile * TIMES * a.group;
  if (token0 >= a.tokens) return;
  const char *src = a.srcs[blockIdx.y];
  char *codes = a.codes[blockIdx.y], *scales = a.scales[blockIdx.y];
  Place p[kParts];
#pragma unroll
  for (int h = 0; h < kParts; ++h) p[h] = place_of<L, PARTS, L::kBlockLanes>(a, chunk, h);
  unsigned long slot[TIMES];
  u32x4 v[TIMES][kParts];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned token = token0 + t * a.group + p[0].token;
    const bool there = token < a.tokens;
    slot[t] = (unsigned long)a.slots[there ? token : 0];  // (no branch around the load: all of them go out together)
    if (!there) slot[t] = ~0ul;
  }
  const bool long_head = a.head_dim >= L::kElems;
  auto work = [&](auto level) {
    constexpr int kLevel = decltype(level)::value;
#pragma unroll
    for (int t = 0; t < TIMES; ++t)
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const char *at = src + times(token0 + t * a.group + p[0].token, a.src_token) + p[h].row;
        if constexpr (kLevel == kWhole) {
          v[t][h] = L::template load<STREAM>(at, L::kElems, true);
        } else {
          if (kLevel == kEven) v[t][h] = u32x4{0, 0, 0, 0};
          if (slot[t] < a.n_slots && p[h].on && (kLevel == kAny || p[h].n)) v[t][h] = L::template load<STREAM>(at, kLevel == kEven ? L::kElems : p[h].n, long_head);
        }
      }
#pragma unroll
    for (int t = 0; t < TIMES; ++t) {
      const unsigned page = a.page_tokens.divide((unsigned)slot[t]), token = (unsigned)slot[t] - page * a.page_tokens.d;
      char *to = codes + (times(page, a.code_page) + times(token, a.code_token));
      char *scale_to = scales + (times(page, a.scale_page) + times(token, a.scale_token));
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const bool there = slot[t] < a.n_slots && p[h].on;  // the same for a block's lanes
        if (kLevel == kAny && !there) continue;
        const unsigned s = scale_of<CacheFormat<FMT>>(block_max<L::kBlockLanes>(most_of<DT>(v[t][h])));
        const typename L::Codes c = L::encode(v[t][h], s);
        if (kLevel != kEven || (there && p[h].n)) {
          L::store_codes(to + p[h].code, kLevel == kAny ? p[h].n : L::kElems, c);
          if (p[h].first % PCCL_CACHE_BLOCK == 0) scale_to[p[h].scale] = (char)s;
        }
      }
    }
  };
  typedef std::integral_constant<int, kAny> Any;
  typedef std::integral_constant<int, kEven> Even;
  typedef std::integral_constant<int, kWhole> Whole;
  if (a.head_dim % L::kElems != 0) return work(Any{});
  if constexpr (PARTS != 0) {
    bool all = true;  // (on the scalar unit)
#pragma unroll
    for (int t = 0; t < TIMES; ++t) all = all && slot[t] < a.n_slots;
    if (all && all_whole<L>(p)) return work(Whole{});
  }
  work(Even{});
}

struct ReadArgs : CacheArgs {
  char *outs[PCCL_CACHE_MAX_TENSORS];
  unsigned out_token;  // bytes
  long out_rows, max_len, table_stride, n_pages;
  const int *page_table, *lengths;
  const long *row_start;
  unsigned token0;  // the launch's first token of every sequence
  int seq0;
};

template <int DT, int FMT, int TIMES, int PARTS>
__global__ void __launch_bounds__(kBlock) cache_read_kernel(const ReadArgs a) {
  typedef Lane<DT, FMT> L;
  constexpr int kParts = PARTS ? PARTS : 1;
  const long seq = a.seq0 + (long)blockIdx.y;
  const unsigned wave = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const unsigned tile = a.chunks.divide(wave), chunk = wave - tile * a.chunks.d;
  const unsigned long token0 = a.token0 + (unsigned long)tile * TIMES * a.group;
  if ((long)token0 >= a.max_len) return;
  Place p[kParts];
#pragma unroll
  for (int h = 0; h < kParts; ++h) p[h] = place_of<L, PARTS, 1>(a, chunk, h);
  // Table entries, length and first row are asked for together (an entry that is not the sequence's is inside the table all the
  // same): what a wavefront waits for is one chain of two loads.
  const int *table = a.page_table + seq * a.table_stride;
  unsigned long page[TIMES];
  bool named[TIMES];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned pos = (unsigned)token0 + t * a.group + p[0].token, entry = a.page_tokens.divide(pos);
    named[t] = (long)entry < a.table_stride;
    page[t] = (unsigned long)(long)table[named[t] ? entry : 0];
  }
  long length = a.lengths[seq];
  const long first_row = a.row_start ? a.row_start[seq] : seq * a.max_len;
  const char *codes = a.codes[blockIdx.z], *scales = a.scales[blockIdx.z];
  char *out = a.outs[blockIdx.z];
  if (length > a.max_len) length = a.max_len;
  typename L::Codes c[TIMES][kParts];
  unsigned s[TIMES][kParts];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned pos = (unsigned)token0 + t * a.group + p[0].token;
    named[t] = named[t] && (long)pos < length && (unsigned long)first_row + pos < (unsigned long)a.out_rows && page[t] < (unsigned long)a.n_pages;
  }
  const bool long_head = a.head_dim >= L::kElems;
  auto work = [&](auto level) {
    constexpr int kLevel = decltype(level)::value;
#pragma unroll
    for (int t = 0; t < TIMES; ++t) {
      const unsigned pos = (unsigned)token0 + t * a.group + p[0].token, token = pos - a.page_tokens.divide(pos) * a.page_tokens.d;
      const char *from = codes + (times((unsigned)page[t], a.code_page) + times(token, a.code_token));
      const char *scale_from = scales + (times((unsigned)page[t], a.scale_page) + times(token, a.scale_token));
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        if (kLevel != kWhole && !(named[t] && p[h].on)) continue;
        s[t][h] = (unsigned char)scale_from[p[h].scale];
        c[t][h] = L::load_codes(from + p[h].code, kLevel == kAny ? p[h].n : L::kElems, long_head);
      }
    }
#pragma unroll
    for (int t = 0; t < TIMES; ++t) {
      const unsigned pos = (unsigned)token0 + t * a.group + p[0].token;
      char *to = out + times((unsigned)(first_row + pos), a.out_token);
#pragma unroll
      for (int h = 0; h < kParts; ++h)
        if (kLevel == kWhole || (named[t] && p[h].on)) L::store(to + p[h].row, kLevel == kAny ? p[h].n : L::kElems, L::decode(c[t][h], s[t][h]));
    }
  };
  typedef std::integral_constant<int, kAny> Any;
  typedef std::integral_constant<int, kEven> Even;
  typedef std::integral_constant<int, kWhole> Whole;
  if (a.head_dim % L::kElems != 0) return work(Any{});
  if constexpr (PARTS != 0) {
    bool all = true;  // (on the scalar unit)
#pragma unroll
    for (int t = 0; t < TIMES; ++t) all = all && named[t];
    if (all && all_whole<L>(p)) return work(Whole{});
  }
  work(Even{});
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

int check_cache(const pccl_cache_desc *c, int dtype, const void *const *tensors, const char *what, bool whole_blocks, CacheArgs *a) {
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
  for (long s : {c->code_page, c->code_token, c->scale_page, c->scale_token})
    if (s > 0xffffffffl) return fail(PCCL_ERR_UNSUPPORTED, "cache stride %ld of a page or token is not below 4 GiB", s);
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
  a->code_page = (unsigned)c->code_page;
  a->code_token = (unsigned)c->code_token;
  a->code_head = c->code_head;
  a->scale_page = (unsigned)c->scale_page;
  a->scale_token = (unsigned)c->scale_token;
  a->scale_head = c->scale_head;
  a->head_dim = c->head_dim;
  // lanes of a head: as many as its elements fill, when writing as many as its blocks have (at most 2^14, of a token 2^30)
  const int elems = 16 / es, head_lanes = whole_blocks ? blocks * (PCCL_CACHE_BLOCK / elems) : (c->head_dim + elems - 1) / elems;
  const unsigned token_lanes = (unsigned)c->heads * (unsigned)head_lanes;
  a->group = std::max(1u, kWave / token_lanes);
  a->token_lanes.set(token_lanes);
  a->head_lanes.set((unsigned)head_lanes);
  a->page_tokens.set((unsigned)c->page_tokens);
  a->parts = a->group > 1 ? 0 : token_lanes > kWave ? 2 : 1;
  a->chunks.set(a->parts < 2 ? 1 : (token_lanes + 2 * kWave - 1) / (2 * kWave));
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

constexpr int kWriteTimes = 2, kReadTimes = 4;  // groups of tokens that a wavefront has in flight where there are enough of them

// whether n wavefronts' worth of tokens, `times` of them to a wavefront, give every compute unit eight workgroups
bool many(long n, int times) { return n >= (long)pccl_host::compute_units() * 8 * kWaves * times; }

// Tokens of a launch: wavefronts stay below 2^26 (a grid times its lanes must fit 32 bits) and below what Divisor divides.
long launch_tokens(const CacheArgs &a) { return std::max(1l, (1l << 26) / a.chunks.d); }

// Workgroups of a launch over n tokens.
unsigned workgroups(const CacheArgs &a, long tokens, int times) {
  const long tiles = (tokens + (long)times * a.group - 1) / ((long)times * a.group);
  return (unsigned)((tiles * a.chunks.d + kWaves - 1) / kWaves);
}

// Calls f(times, parts) with both as constants.
template <int TIMES, class F>
void with_shape(bool several, int parts, F &&f) {
  auto of_parts = [&](auto times) {
    if (parts == 0) f(times, std::integral_constant<int, 0>{});
    else if (parts == 1) f(times, std::integral_constant<int, 1>{});
    else f(times, std::integral_constant<int, 2>{});
  };
  if (several) of_parts(std::integral_constant<int, TIMES>{});
  else of_parts(std::integral_constant<int, 1>{});
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
  int rc = check_cache(c, dtype, srcs, "source", true, &a);
  if (rc != PCCL_OK) return rc;
  if (tokens < 0 || tokens > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "tokens %ld outside [0, 2^31)", tokens);
  const int es = pccl_host::pccl_dtype_bytes(dtype);
  if (src_token_stride < 0 || src_head_stride < 0 || src_head_stride > (1l << 40))
    return fail(PCCL_ERR_INVALID_ARG, "source strides %ld, %ld below 0 or beyond 2^40", src_token_stride, src_head_stride);
  if (src_token_stride > 0xffffffffl / es) return fail(PCCL_ERR_UNSUPPORTED, "source stride %ld of a token is not below 4 GiB", src_token_stride);
  if ((uintptr_t)slots % 8) return fail(PCCL_ERR_MISALIGNED, "slots (%p) not 8-byte aligned", (const void *)slots);
  if (tokens && !slots) return fail(PCCL_ERR_INVALID_ARG, "slots are null");
  for (int k = 0; k < c->n_tensors; ++k)
    if (tokens && !srcs[k]) return fail(PCCL_ERR_INVALID_ARG, "source %d is null", k);
  rc = pccl_host::check_stream(&stream);
  if (rc != PCCL_OK) return rc;
  if (tokens == 0 || c->n_pages == 0) return PCCL_OK;
  a.src_token = (unsigned)(src_token_stride * es);
  a.row_head = src_head_stride * es;
  a.n_slots = (unsigned long)(c->n_pages * c->page_tokens);
  const bool stream_in = (double)c->heads * c->head_dim * es * tokens * c->n_tensors >= (double)(48l << 20);  // (up to 2^68)
  return pccl_host::in_pieces(tokens, launch_tokens(a), [&](long lo, long n) {
    for (int k = 0; k < c->n_tensors; ++k) a.srcs[k] = (const char *)srcs[k] + lo * (long)a.src_token;
    a.slots = slots + lo;
    a.tokens = (unsigned)n;
    with_types(dtype, c->format, [&](auto t, auto f) {
      with_shape<kWriteTimes>(many((n + a.group - 1) / a.group * a.chunks.d * c->n_tensors, kWriteTimes), a.parts, [&](auto times, auto parts) {
        constexpr int DT = decltype(t)::value, FMT = decltype(f)::value, TIMES = decltype(times)::value, PARTS = decltype(parts)::value;
        const dim3 grid(workgroups(a, n, TIMES), c->n_tensors);
        if (stream_in) hipLaunchKernelGGL((cache_write_kernel<DT, FMT, TIMES, PARTS, true>), grid, dim3(kBlock), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((cache_write_kernel<DT, FMT, TIMES, PARTS, false>), grid, dim3(kBlock), 0, (hipStream_t)stream, a);
      });
    });
    return launched("cache_write");
  });
}

extern "C" int pccl_hip_cache_read(const pccl_cache_desc *c, int dtype, void *const *outs, long out_token_stride, long out_head_stride,
                                   long out_rows, const int *page_table, long table_stride, const int *lengths, const long *row_start,
                                   int n_seq, long max_len, void *stream) {
  pccl_host::clear_error();
  ReadArgs a;
  int rc = check_cache(c, dtype, (const void *const *)outs, "output", false, &a);
  if (rc != PCCL_OK) return rc;
  if (n_seq < 0) return fail(PCCL_ERR_INVALID_ARG, "n_seq %d < 0", n_seq);
  if (max_len < 0 || max_len > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "max_len %ld outside [0, 2^31)", max_len);
  if (out_rows > 0x7fffffffl) return fail(PCCL_ERR_INVALID_ARG, "out_rows %ld outside [0, 2^31)", out_rows);
  if (out_rows < 0 || table_stride < 0) return fail(PCCL_ERR_INVALID_ARG, "out_rows %ld or table_stride %ld below 0", out_rows, table_stride);
  if (out_token_stride < 0 || out_head_stride < 0 || out_token_stride > (1l << 40) || out_head_stride > (1l << 40))
    return fail(PCCL_ERR_INVALID_ARG, "output strides %ld, %ld outside [0, 2^40]", out_token_stride, out_head_stride);
  const int es = pccl_host::pccl_dtype_bytes(dtype);
  if (out_token_stride > 0xffffffffl / es) return fail(PCCL_ERR_UNSUPPORTED, "output stride %ld of a token is not below 4 GiB", out_token_stride);
  if (!apart({1, out_rows, c->heads}, {0, out_token_stride, out_head_stride}, c->head_dim))
    return fail(PCCL_ERR_INVALID_ARG, "output strides %ld, %ld let heads overlap", out_token_stride, out_head_stride);
  if ((uintptr_t)page_table % 4 || (uintptr_t)lengths % 4 || (uintptr_t)row_start % 8)
    return fail(PCCL_ERR_MISALIGNED, "page_table, lengths or row_start not aligned to their elements");
  const bool nothing = n_seq == 0 || max_len == 0 || out_rows == 0 || table_stride == 0 || c->n_pages == 0;
  if (!nothing && (!page_table || !lengths)) return fail(PCCL_ERR_INVALID_ARG, "page_table or lengths are null");
  for (int k = 0; k < c->n_tensors; ++k)
    if (!nothing && !outs[k]) return fail(PCCL_ERR_INVALID_ARG, "output %d is null", k);
  rc = pccl_host::check_stream(&stream);
  if (rc != PCCL_OK || nothing) return rc;
  for (int k = 0; k < c->n_tensors; ++k) a.outs[k] = (char *)outs[k];
  a.out_token = (unsigned)(out_token_stride * es);
  a.row_head = out_head_stride * es;
  a.out_rows = out_rows;
  a.max_len = max_len;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.row_start = row_start;
  a.n_pages = c->n_pages;
  // (no wavefronts for tokens that the table has no page for: max_len may be any upper bound, with row_start up to 2^31 - 1 tokens of
  // every sequence, and those would be 2^29 wavefronts a sequence with nothing to do)
  const long tokens = pccl_host::tokens_in_pages(max_len, table_stride, c->page_tokens);
  return pccl_host::in_pieces(n_seq, 65535, [&](long seq, long seqs) {
    a.seq0 = (int)seq;
    return pccl_host::in_pieces(tokens, launch_tokens(a), [&](long lo, long n) {
      a.token0 = (unsigned)lo;
      with_types(dtype, c->format, [&](auto t, auto f) {
        with_shape<kReadTimes>(many((n + a.group - 1) / a.group * a.chunks.d * seqs * c->n_tensors, kReadTimes), a.parts, [&](auto times, auto parts) {
          constexpr int DT = decltype(t)::value, FMT = decltype(f)::value, TIMES = decltype(times)::value, PARTS = decltype(parts)::value;
          hipLaunchKernelGGL((cache_read_kernel<DT, FMT, TIMES, PARTS>), dim3(workgroups(a, n, TIMES), (unsigned)seqs, c->n_tensors), dim3(kBlock), 0,
                             (hipStream_t)stream, a);
        });
      });
      return launched("cache_read");
    });
  });
}

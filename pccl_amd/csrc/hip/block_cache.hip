// block_cache.hip -- pccl_hip_cache_write, pccl_hip_cache_read: keys and values coded in blocks of 32 elements with
// a shared power-of-two scale as they are written to their pages, and read back through page tables.
//
// Four neighbouring lanes work on one block, eight elements each: 16 bytes of a 16-bit source a load, and the block's
// largest magnitude is two data-parallel-primitive steps inside the quad away.  Blocks are numbered row by row
// (row = token and head), so that consecutive quads walk a token's heads in memory order on both sides.
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
constexpr int kBlocksAtOnce = kBlock / kQuad;

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
// down(): eight scaled elements (none beyond the largest value) to 8 * kBits bits, nearest, ties to even.
template <int FMT> struct CacheFormat;

template <bool E5M2> struct CacheF8 {
  static constexpr int kBits = 8;
  static constexpr unsigned kTop = 0x600000u;  // 1.75 * 2^15 and 1.75 * 2^8
  static constexpr int kExponent = E5M2 ? 15 : 8;
  typedef F8Fmt<E5M2> F;
  static __device__ __forceinline__ u32x2 down(const float *x) { return u32x2{F::down4(x[0], x[1], x[2], x[3]), F::down4(x[4], x[5], x[6], x[7])}; }
  static __device__ __forceinline__ void up(u32x2 c, float scale, float *x) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const typename F::f32x2 lo = F::template up2<false>(c[w]), hi = F::template up2<true>(c[w]);
      x[4 * w] = lo.x * scale;
      x[4 * w + 1] = lo.y * scale;
      x[4 * w + 2] = hi.x * scale;
      x[4 * w + 3] = hi.y * scale;
    }
  }
};
template <> struct CacheFormat<PCCL_CACHE_F8E4M3> : CacheF8<false> {};
template <> struct CacheFormat<PCCL_CACHE_F8E5M2> : CacheF8<true> {};

template <> struct CacheFormat<PCCL_CACHE_I8> {
  static constexpr int kBits = 8;
  static constexpr unsigned kTop = 0x7e0000u;  // 127/64
  static constexpr int kExponent = 0;
  static __device__ __forceinline__ u32x2 down(const float *x) {
    // 64 x + 1.5 * 2^23 is rounded to a whole number, whose low byte is the code (one fused step: one rounding);
    // only a block whose scale would be 2^128 comes beyond 127
    unsigned q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = as_u32(__builtin_fmaf(__builtin_amdgcn_fmed3f(x[i], -127.0f / 64, 127.0f / 64), 64.0f, 12582912.0f));
    u32x2 c;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const unsigned lo = __builtin_amdgcn_perm(q[4 * w + 1], q[4 * w], 0x0c0c0400u), hi = __builtin_amdgcn_perm(q[4 * w + 3], q[4 * w + 2], 0x0c0c0400u);
      c[w] = lo | hi << 16;
    }
    return c;
  }
  static __device__ __forceinline__ void up(u32x2 c, float scale, float *x) {
    const float step = scale * (1.0f / 64);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)(c[i / 4] << (24 - 8 * (i % 4))) >> 24) * step;
  }
};

template <> struct CacheFormat<PCCL_CACHE_F4E2M1> {
  static constexpr int kBits = 4;
  static constexpr unsigned kTop = 0x400000u;  // 1.5 * 2^2
  static constexpr int kExponent = 2;
  static __device__ __forceinline__ unsigned down(const float *x) {
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], 1.0f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], 1.0f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], 1.0f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], 1.0f, 3);
    return c;
  }
  static __device__ __forceinline__ void up(unsigned c, float scale, float *x) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    x[0] = a.x * scale;
    x[1] = a.y * scale;
    x[2] = b.x * scale;
    x[3] = b.y * scale;
    x[4] = d.x * scale;
    x[5] = d.y * scale;
    x[6] = e.x * scale;
    x[7] = e.y * scale;
  }
};

// A lane's eight codes: two words or one.
template <int BITS> struct LaneCodes { typedef u32x2 type; typedef u32x2_a1 any; };
template <> struct LaneCodes<4> { typedef unsigned type; typedef u32_a1 any; };

struct CacheArgs {
  char *codes[PCCL_CACHE_MAX_TENSORS], *scales[PCCL_CACHE_MAX_TENSORS];
  long code_page, code_token, code_head, scale_page, scale_token, scale_head;
  long n_slots;
  int heads, head_dim;
  Divisor blocks, by_heads, page_tokens;  // blocks of a head, heads, tokens of a page
};

struct WriteArgs : CacheArgs {
  const char *srcs[PCCL_CACHE_MAX_TENSORS];
  long src_token, src_head;  // bytes
  const long *slots;
  unsigned n_blocks;  // of the launch
};

// The eight elements of a lane, from `at` on, `n` of them (0..8) inside the head; zeros behind.
template <class R>
struct Eight {
  static constexpr int kPacks = 8 / R::kPack;
  u32x4 v[kPacks];
  __device__ __forceinline__ void load(const char *at, int n) {
    if (n == 8) {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) v[j] = ((const typename R::pack_t *)at)[j];
    } else {
#pragma unroll
      for (int j = 0; j < kPacks; ++j) {
        typename R::elem_t e[R::kPack];
#pragma unroll
        for (int i = 0; i < R::kPack; ++i) e[i] = j * R::kPack + i < n ? ((const typename R::elem_t *)at)[j * R::kPack + i] : (typename R::elem_t)0;
        v[j] = __builtin_bit_cast(u32x4, e);
      }
    }
  }
  __device__ __forceinline__ void up(float *x) const {
#pragma unroll
    for (int j = 0; j < kPacks; ++j) R::up(v[j], x + j * R::kPack);
  }
  // binary32 bits of the largest magnitude; magnitudes compare as whole numbers, infinities and NaN come out on top
  __device__ __forceinline__ unsigned most() const {
    float x[8];
    up(x);
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, as_u32(x[i]) & 0x7fffffffu);
    return m;
  }
};

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

template <int DT, int FMT, int TIMES>
__global__ void __launch_bounds__(kBlock) cache_write_kernel(const WriteArgs a) {
  typedef RowType<DT> R;
  typedef CacheFormat<FMT> F;
  typedef LaneCodes<F::kBits> L;
  const char *src = a.srcs[blockIdx.y];
  char *codes = a.codes[blockIdx.y], *scales = a.scales[blockIdx.y];
  const int q = (int)threadIdx.x % kQuad;
  Eight<R> e[TIMES];
  long slot[TIMES];
  unsigned block[TIMES], head[TIMES];
  int n[TIMES];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned u = (blockIdx.x * TIMES + t) * kBlocksAtOnce + threadIdx.x / kQuad;
    slot[t] = -1;
    if (u < a.n_blocks) {
      const unsigned row = a.blocks.divide(u), token = a.by_heads.divide(row);
      block[t] = u - row * a.blocks.d;
      head[t] = row - token * a.by_heads.d;
      slot[t] = a.slots[token];
      const int first = (int)block[t] * PCCL_CACHE_BLOCK + q * kPerLane;
      n[t] = min(max(a.head_dim - first, 0), kPerLane);
      if ((unsigned long)slot[t] < (unsigned long)a.n_slots)
        e[t].load(src + token * a.src_token + head[t] * a.src_head + (long)first * R::kBytes, n[t]);
      else slot[t] = -1;
    }
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    if (slot[t] < 0) continue;  // whole quads
    const unsigned s = scale_of<F>(quad_max(e[t].most()));
    float x[8];
    e[t].up(x);
    // 2^(127 - s); exact, and so is the product (a subnormal product is far below half of the smallest code)
    const float inverse = as_f32(s == 255 ? 0u : s == 254 ? 0x400000u : (254u - s) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inverse;
    typename L::type c = F::down(x);
    if (s == 255) c = typename L::type{};
    const unsigned page = a.page_tokens.divide((unsigned)slot[t]), token = (unsigned)slot[t] - page * a.page_tokens.d;
    char *to = codes + page * a.code_page + token * a.code_token + head[t] * a.code_head +
               (block[t] * PCCL_CACHE_BLOCK + q * kPerLane) * F::kBits / 8;
    if (n[t] == 8) {
      *(typename L::any *)to = c;
    } else {
      const int bytes = (n[t] * F::kBits + 7) / 8;
#pragma unroll
      for (int i = 0; i < F::kBits; ++i) {
        unsigned w;
        if constexpr (F::kBits == 8) w = c[i / 4];
        else w = c;
        if (i < bytes) to[i] = (char)(w >> (8 * (i % 4)));
      }
    }
    if (q == 0) scales[page * a.scale_page + token * a.scale_token + head[t] * a.scale_head + block[t]] = (char)s;
  }
}

struct ReadArgs : CacheArgs {
  char *outs[PCCL_CACHE_MAX_TENSORS];
  long out_token, out_head;  // bytes
  long out_rows, max_len, table_stride;
  const int *page_table, *lengths;
  const long *row_start;
  long token0;        // the launch's first token of every sequence
  unsigned n_blocks;  // of the launch, per sequence
  int seq0;
  long n_pages;
};

template <int DT, int FMT, int TIMES>
__global__ void __launch_bounds__(kBlock) cache_read_kernel(const ReadArgs a) {
  typedef RowType<DT> R;
  typedef CacheFormat<FMT> F;
  typedef LaneCodes<F::kBits> L;
  const long seq = a.seq0 + (long)blockIdx.y;
  const char *codes = a.codes[blockIdx.z], *scales = a.scales[blockIdx.z];
  char *out = a.outs[blockIdx.z];
  const int q = (int)threadIdx.x % kQuad;
  long length = a.lengths[seq];
  if (length > a.max_len) length = a.max_len;
  const unsigned base = blockIdx.x * TIMES * kBlocksAtOnce;
  if (a.token0 + (long)a.by_heads.divide(a.blocks.divide(base)) >= length) return;  // the workgroup's first token is behind the end
  const long first_row = a.row_start ? a.row_start[seq] : seq * a.max_len;
  const int *table = a.page_table + seq * a.table_stride;
  typename L::type c[TIMES];
  unsigned s[TIMES];
  char *to[TIMES];
  int n[TIMES];
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    const unsigned u = base + t * kBlocksAtOnce + threadIdx.x / kQuad;
    n[t] = 0;
    if (u >= a.n_blocks) continue;
    const unsigned row = a.blocks.divide(u), token_of = a.by_heads.divide(row);
    const unsigned block = u - row * a.blocks.d, head = row - token_of * a.by_heads.d;
    const long pos = a.token0 + token_of, out_row = first_row + pos;
    const unsigned entry = a.page_tokens.divide((unsigned)pos);
    if (pos >= length || (long)entry >= a.table_stride || (unsigned long)out_row >= (unsigned long)a.out_rows) continue;
    const long page = table[entry];
    if ((unsigned long)page >= (unsigned long)a.n_pages) continue;
    const unsigned token = (unsigned)pos - entry * a.page_tokens.d;
    const int first = (int)block * PCCL_CACHE_BLOCK + q * kPerLane;
    n[t] = min(max(a.head_dim - first, 0), kPerLane);
    const char *from = codes + page * a.code_page + token * a.code_token + head * a.code_head + (long)first * F::kBits / 8;
    if (n[t] == 8) {
      c[t] = *(const typename L::any *)from;
    } else {
      const int bytes = (n[t] * F::kBits + 7) / 8;
      unsigned w[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < F::kBits; ++i)
        if (i < bytes) w[i / 4] |= (unsigned)(unsigned char)from[i] << (8 * (i % 4));
      if constexpr (F::kBits == 8) c[t] = u32x2{w[0], w[1]};
      else c[t] = w[0];
    }
    s[t] = (unsigned char)scales[page * a.scale_page + token * a.scale_token + head * a.scale_head + block];
    to[t] = out + out_row * a.out_token + head * a.out_head + (long)first * R::kBytes;
  }
#pragma unroll
  for (int t = 0; t < TIMES; ++t) {
    if (n[t] == 0) continue;
    float x[8];
    // (every product is exact in binary32: a code has at most 7 bits, the smallest is 2^-16 of its scale)
    F::up(c[t], as_f32(s[t] == 255 ? 0x7fc00000u : s[t] == 0 ? 0x400000u : s[t] << 23), x);
    if (n[t] == 8) {
#pragma unroll
      for (int j = 0; j < 8 / R::kPack; ++j) ((typename R::pack_t *)to[t])[j] = R::down(x + j * R::kPack);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n[t]) ((typename R::elem_t *)to[t])[i] = R::down1(x[i]);
    }
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
  a->n_slots = c->n_pages * c->page_tokens;
  a->heads = c->heads;
  a->head_dim = c->head_dim;
  a->blocks.set((unsigned)blocks);
  a->by_heads.set((unsigned)c->heads);
  a->page_tokens.set((unsigned)c->page_tokens);
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

constexpr int kTimes = 4;  // blocks a quad has in flight where there are enough of them

// whether n blocks give every compute unit eight workgroups of kTimes blocks a quad
bool many(long n) { return n >= (long)pccl_host::compute_units() * 8 * kBlocksAtOnce * kTimes; }

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
  a.src_head = src_head_stride * es;
  const long per_token = (long)c->heads * a.blocks.d, most = 0x7fffffffl / per_token;  // block numbers of a launch stay below 2^31
  for (long lo = 0; lo < tokens; lo += most) {
    const long n = std::min(most, tokens - lo);
    for (int k = 0; k < c->n_tensors; ++k) a.srcs[k] = (const char *)srcs[k] + lo * a.src_token;
    a.slots = slots + lo;
    a.n_blocks = (unsigned)(n * per_token);
    with_types(dtype, c->format, [&](auto t, auto f) {
      constexpr int DT = decltype(t)::value, FMT = decltype(f)::value;
      auto grid = [&](unsigned times) { return dim3((a.n_blocks + kBlocksAtOnce * times - 1) / (kBlocksAtOnce * times), c->n_tensors); };
      if (many((long)a.n_blocks * c->n_tensors)) hipLaunchKernelGGL((cache_write_kernel<DT, FMT, kTimes>), grid(kTimes), dim3(kBlock), 0, (hipStream_t)stream, a);
      else hipLaunchKernelGGL((cache_write_kernel<DT, FMT, 1>), grid(1), dim3(kBlock), 0, (hipStream_t)stream, a);
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
  a.out_head = out_head_stride * es;
  a.out_rows = out_rows;
  a.max_len = max_len;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.lengths = lengths;
  a.row_start = row_start;
  a.n_pages = c->n_pages;
  const long per_token = (long)c->heads * a.blocks.d, most = 0x7fffffffl / per_token;
  for (int seq = 0; seq < n_seq; seq += 65535) {
    a.seq0 = seq;
    const int seqs = std::min(65535, n_seq - seq);
    for (long lo = 0; lo < max_len; lo += most) {
      a.token0 = lo;
      a.n_blocks = (unsigned)(std::min(most, max_len - lo) * per_token);
      with_types(dtype, c->format, [&](auto t, auto f) {
        constexpr int DT = decltype(t)::value, FMT = decltype(f)::value;
        auto grid = [&](unsigned times) { return dim3((a.n_blocks + kBlocksAtOnce * times - 1) / (kBlocksAtOnce * times), seqs, c->n_tensors); };
        if (many((long)a.n_blocks * seqs * c->n_tensors)) hipLaunchKernelGGL((cache_read_kernel<DT, FMT, kTimes>), grid(kTimes), dim3(kBlock), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((cache_read_kernel<DT, FMT, 1>), grid(1), dim3(kBlock), 0, (hipStream_t)stream, a);
      });
      rc = launched("cache_read");
      if (rc != PCCL_OK) return rc;
    }
  }
  return PCCL_OK;
}

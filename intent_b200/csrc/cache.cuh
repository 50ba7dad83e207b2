// Rows of a key-value cache in 8 bits: one f32 scale a row, codes that are whole numbers or e4m3.
//
//   int8   scale = max(f32(amax / 127), 2^-126)              code = x / scale, rounded to even
//   e4m3   scale = 2^max(ceil(log2(amax / 448)), -126)       code = x / scale, rounded to even
//
// amax is the largest magnitude of the row.  A row that holds an infinity or a NaN gets the scale
// NaN and codes 0: it reads back as NaN throughout and so spoils what attends to it, as it would in
// 16 bits.  The e4m3 scale is a power of two, so that the quotient is exact and only the code is
// rounded; a power of two would cost a whole-number code up to one of its seven bits, so the int8
// scale is not one, and the code is that of the exact quotient all the same (see int8_code).
#pragma once

#include "heads.cuh"

namespace b200 {
namespace cache {

enum Store : int { kNative = 0, kInt8 = 1, kE4m3 = 2 };

constexpr float kTiny = 1.1754943508222875e-38f;  // 2^-126

// amax as bits: NaN > infinity > every number.  f32(amax / 127) by way of f64: the binary expansion of a whole
// number over 127 repeats after seven digits, so f64 never brings one to halfway between two f32.
__device__ __forceinline__ float int8_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return fmaxf((float)((double)__uint_as_float(amax_bits) * (1.0 / 127.0)), kTiny);
}
// amax = m 2^k with 1 <= m < 2 is at most 448 * 2^(k - 8) if m <= 1.75, else at most 448 * 2^(k - 7).
__device__ __forceinline__ float e4m3_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int k = (int)(amax_bits >> 23) - 127;
  const int e = k - ((amax_bits & 0x7fffffu) > 0x600000u ? 7 : 8);
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

__device__ __forceinline__ uint32_t e4m3_pair(float low, float high) {
  uint16_t packed;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(packed) : "f"(high), "f"(low));
  return packed;
}
__device__ __forceinline__ uint32_t f16x2_of_e4m3(uint32_t pair) {
  uint32_t wide;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(wide) : "h"((uint16_t)pair));
  return wide;
}

// The first bytes of four words.
__device__ __forceinline__ uint32_t first_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// 16 columns of a row and their codes.
//
// int8: the quotient in f64, rounded to a multiple of 2^-30 by one fma and then to a whole number by one
// sum, ties to even both times.  The reciprocal is good to 2^-45 (one Newton step from f32's), so the
// quotient, below 128, to 2^-38: a tie lands on its multiple exactly.  What is no tie is 2^-25 or
// more away from one (twice its distance is a multiple of the scale's last bit, of 24), so it stays on its
// side.  The quotients of 8-bit numbers are so often exact ties that f32 with a second look at the
// doubtful ones cost more: 63 us against 38 for 32768 tokens of 8 heads of 128 columns.
__device__ __forceinline__ uint32_t int8_code(float x, double inverse) {
  const double multiple = fma((double)x, inverse, 6291456.0);                     // 1.5 * 2^22
  return (uint32_t)__double2loint(multiple + (6755399441055744.0 - 6291456.0));   // 1.5 * 2^52
}

__device__ __forceinline__ uint4 encode(const float (&x)[16], int store, float scale) {
  uint32_t words[4];
  if (!(scale < INFINITY)) return make_uint4(0, 0, 0, 0);
  if (store == kInt8) {
    float guess;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(guess) : "f"(scale));
    const double near = guess, inverse = fma(near, fma(-(double)scale, near, 1.0), near);
#pragma unroll
    for (int w = 0; w < 4; ++w)
      words[w] = first_bytes(int8_code(x[4 * w], inverse), int8_code(x[4 * w + 1], inverse), int8_code(x[4 * w + 2], inverse),
                             int8_code(x[4 * w + 3], inverse));
  } else {
    const float inverse = __uint_as_float((254u << 23) - __float_as_uint(scale));   // of a power of two
#pragma unroll
    for (int w = 0; w < 4; ++w)
      words[w] = e4m3_pair(x[4 * w] * inverse, x[4 * w + 1] * inverse) |
                 e4m3_pair(x[4 * w + 2] * inverse, x[4 * w + 3] * inverse) << 16;
  }
  return make_uint4(words[0], words[1], words[2], words[3]);
}
__device__ __forceinline__ void decode(const uint4 &codes, int store, float scale, float (&x)[16]) {
  const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (store == kInt8) {
      // 0x4b000000 + u is 2^23 + u in f32; u = code + 128 (the sign bit flipped)
      const uint32_t biased = words[w] ^ 0x80808080u;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[4 * w + i] = (__uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 | i)) - 8388736.0f) * scale;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t pair = f16x2_of_e4m3((words[w] >> (16 * i)) & 0xffffu);
        const float2 wide = __half22float2(*reinterpret_cast<const __half2 *>(&pair));
        x[4 * w + 2 * i] = wide.x * scale;
        x[4 * w + 2 * i + 1] = wide.y * scale;
      }
    }
  }
}

// Page and place of a slot; slots of ordinary caches fit 32 bits, where a division costs a quarter.
__device__ __forceinline__ void locate(int64_t slot, int page_size, int64_t &page, int &offset) {
  if ((uint64_t)slot >> 32) {
    page = slot / page_size;
    offset = (int)(slot - page * page_size);
  } else {
    const uint32_t p = (uint32_t)slot / (uint32_t)page_size;
    page = p;
    offset = (int)((uint32_t)slot - p * (uint32_t)page_size);
  }
}

// ---- host ----------------------------------------------------------------------
struct Cache {
  heads::View4 k, v;
  heads::View3 k_scale, v_scale;
};

// What every entry wants of a cache: pages x heads x page_size x columns, 16-bit rows or codes with scales.
inline int check(const char *what, const Cache &c, int32_t dtype, int32_t store, int64_t most_columns) {
  using namespace heads;
  if (store != B200_F16 && store != B200_BF16 && store != B200_I8 && store != B200_E4M3)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: unknown cache element type %d", what, store);
  const bool native = store == B200_F16 || store == B200_BF16;
  if (native && store != dtype)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: a 16-bit cache holds the rows' own type", what);
  if (!sane(c.k) || !sane(c.v)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
  if (c.k.d0 != c.v.d0 || c.k.d1 != c.v.d1 || c.k.d2 != c.v.d2 || c.k.d3 != c.v.d3)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the key and value caches differ in shape", what);
  if (c.k.d3 < 16 || c.k.d3 > most_columns || c.k.d3 % 16)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: head_dim %lld is not a multiple of 16 in [16, %lld]", what,
                (long long)c.k.d3, (long long)most_columns);
  if (c.k.d0 >= (int64_t(1) << 31) || c.k.d2 >= (int64_t(1) << 31) || c.k.d1 > 65536)
    return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: 2^31 pages or slots of a page, or more than 65536 heads", what);
  const bool any = c.k.d0 && c.k.d1 && c.k.d2;
  if (any && (!c.k.data || !c.v.data)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (any && (!vector_rows(c.k, element_size(store)) || !vector_rows(c.v, element_size(store))))
    return fail(B200_ERR_UNSUPPORTED_LAYOUT,
                "%s: cache rows need a unit inner stride, a 16-byte aligned base and outer strides of whole 16-byte steps", what);
  if (native) return B200_OK;
  const View3 *const scales[] = {&c.k_scale, &c.v_scale};
  for (const View3 *s : scales) {
    if (!sane(*s)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: negative or huge extent or stride", what);
    if (s->d0 != c.k.d0 || s->d1 != c.k.d1 || s->d2 != c.k.d2 || (any && !s->data))
      return fail(B200_ERR_INVALID_ARGUMENT, "%s: an 8-bit cache needs scales of shape (pages, heads, page_size)", what);
    if (!aligned4(s->data)) return fail(B200_ERR_UNSUPPORTED_LAYOUT, "%s: scales are 4-byte aligned", what);
  }
  return B200_OK;
}

}  // namespace cache
}  // namespace b200

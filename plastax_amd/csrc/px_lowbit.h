// px_lowbit.h -- pieces shared by the kernels of level pairs in few bits: the
// two block formats, the element types and the fragments of the matrix
// instructions.
//
// A block is 32 consecutive values of a line under one scale 2^(s - 127), s
// one byte. In 4 bits (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6, sign in bit 3) two
// values share a byte, the earlier one low; in 8 bits (e4m3: 4 exponent bits
// of bias 7, 3 behind the point, no infinities, 0x7f / 0xff NaN) each has one.
// The scale is the least power of two under which the block's largest value
// is not above 6 or 448.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/plastax_hip.h"

namespace px {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ bf16x8 as_bf16x8(uint4 v) { return __builtin_bit_cast(bf16x8, v); }

__device__ __forceinline__ i32x8 as_i32x8(bf16x8 v) {  // (4-bit operands take the first half)
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const i32x4 w = __builtin_bit_cast(i32x4, v);
  return i32x8{w[0], w[1], w[2], w[3], 0, 0, 0, 0};
}

// Element types of activations and gradients: float, __bf16, _Float16.
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);  // to the nearest, ties to even
}

// Eight consecutive values as they are in memory, and as a load that needs
// no more than the values' own alignment (the memory pipeline takes 16 bytes
// from any address: rows of an odd length need no loads of single values).
template <typename T>
struct Unit {
  typedef T type __attribute__((ext_vector_type(8)));
  typedef T load __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
// p[i * stride], i < n; zeros from there on.
// PASS: as in store8, of what a pass reads once.
template <bool PASS = false, typename T>
__device__ __forceinline__ typename Unit<T>::type load_unit(const T* p, int64_t stride, int n) {
  if (stride == 1 && n >= 8) {
    if (PASS) return __builtin_nontemporal_load(reinterpret_cast<const typename Unit<T>::load*>(p));
    return *reinterpret_cast<const typename Unit<T>::load*>(p);
  }
  typename Unit<T>::type r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = i < n ? p[i * stride] : from_f32<T>(0.0f);
  return r;
}
// The same as float32.
template <bool PASS = false, typename T>
__device__ __forceinline__ void load8(const T* p, int64_t stride, int n, float v[8]) {
  const typename Unit<T>::type r = load_unit<PASS>(p, stride, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32(r[i]);
}

// PASS: the results of a pass over a large array, read by nothing in it: 16
// bytes a lane go past the caches' replacement (of float32, whose two stores
// would each leave half of every line, only whole lines may).
template <bool PASS = false, typename T>
__device__ __forceinline__ void store8(T* p, int n, const float v[8]) {
  if (n >= 8) {
    typename Unit<T>::load r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = from_f32<T>(v[i]);
    if (PASS && sizeof(T) == 2)
      __builtin_nontemporal_store(r, reinterpret_cast<typename Unit<T>::load*>(p));
    else
      *reinterpret_cast<typename Unit<T>::load*>(p) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = from_f32<T>(v[i]);
}

// Four consecutive results of a row, `left` of them inside it.
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, f32x4 v) {
  typedef T t4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (left >= 4) {
    t4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = from_f32<T>(v[i]);
    *reinterpret_cast<t4*>(p) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = from_f32<T>(v[i]);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kInfBits = 0x7F800000u;

// The exponent e of a block whose largest |value| has these bits (finite):
// amax <= (1 + mantissa / 2^23) 2^top 2^e, e >= least. Subnormal amax: the
// exponent field is 0, and least stands above what it gives.
__device__ __forceinline__ int block_exponent(uint32_t amax, uint32_t mantissa, int top, int least) {
  const int e = static_cast<int>(amax >> 23) - 127 - top + ((amax & 0x7FFFFFu) > mantissa ? 1 : 0);
  return e > least ? e : least;
}
__device__ __forceinline__ int exponent4(uint32_t amax) { return block_exponent(amax, 0x400000u, 2, -125); }
__device__ __forceinline__ int exponent8(uint32_t amax) { return block_exponent(amax, 0x600000u, 8, -117); }

// 2^e, e in [-126, 127].
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// What a scale byte stands for; 255 is a block of NaN.
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7FC00000u : s << 23);
}

// 8 values under the scale 2^e as 4-bit codes, to the nearest, ties to the
// even code (the conversion instruction divides by its scale operand).
__device__ __forceinline__ uint32_t codes4(const float v[8], float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return c;
}

// 8 values times inv = 2^-e as e4m3 codes; one that is not finite is some NaN.
__device__ __forceinline__ uint2 codes8(const float v[8], float inv) {
  int a = 0, b = 0;
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, a, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, a, true);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, b, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, b, true);
  return make_uint2(static_cast<uint32_t>(a), static_cast<uint32_t>(b));
}
// The codes of values that are not finite: 0xff for a negative infinity, 0x7f
// for the others.
__device__ __forceinline__ uint2 mark8(uint2 c, const float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (abs_bits(v[i]) >= kInfBits) {
      const uint32_t code = __float_as_uint(v[i]) == (0x80000000u | kInfBits) ? 0xFFu : 0x7Fu;
      uint32_t& w = i < 4 ? c.x : c.y;
      w = (w & ~(0xFFu << (i % 4 * 8))) | code << (i % 4 * 8);
    }
  return c;
}
// The largest of m and 8 |values| as bits, of all of them or of the finite ones.
template <bool FINITE>
__device__ __forceinline__ uint32_t largest8(uint32_t m, const float v[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = abs_bits(v[i]);
    m = a > m && (!FINITE || a < kInfBits) ? a : m;
  }
  return m;
}

// The float32 values of 8 codes under a scale (exact: 2 or 4 significant
// bits times a power of two, normal by the formats' least exponents).
__device__ __forceinline__ void values4(uint32_t c, float scale, float v[8]) {
  f32x2 p;
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0), v[0] = p[0], v[1] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1), v[2] = p[0], v[3] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2), v[4] = p[0], v[5] = p[1];
  p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3), v[6] = p[0], v[7] = p[1];
}
__device__ __forceinline__ void values8(uint2 c, float scale, float v[8]) {
  f32x2 p;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, false), v[0] = p[0] * scale, v[1] = p[1] * scale;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.x, true), v[2] = p[0] * scale, v[3] = p[1] * scale;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, false), v[4] = p[0] * scale, v[5] = p[1] * scale;
  p = __builtin_amdgcn_cvt_pk_f32_fp8(c.y, true), v[6] = p[0] * scale, v[7] = p[1] * scale;
}

// The same as bf16, exact for the same reason (bf16 has float32's exponents).
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xFFFF0000u);
}
__device__ __forceinline__ uint4 bf16_of4(uint32_t c, float scale) {
  uint4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3));
  return r;
}
// The first `left` of 8 codes of 8 bits, zeros in place of the others: what is
// behind a line's end may be NaN, which no other operand's zero takes out of a sum.
__device__ __forceinline__ uint2 first_codes8(uint2 c, int64_t left) {
  if (left >= 8) return c;
  const uint64_t keep = left > 0 ? (uint64_t{1} << (8 * left)) - 1 : 0;
  return make_uint2(c.x & static_cast<uint32_t>(keep), c.y & static_cast<uint32_t>(keep >> 32));
}
__device__ __forceinline__ uint4 bf16_of8(uint2 c, float scale) {
  float v[8];
  values8(c, scale, v);
  return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}

// bf16 of two values, to the nearest, and its halves as float32.
__device__ __forceinline__ uint32_t round_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
__device__ __forceinline__ float low_bf16(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_bf16(uint32_t p) { return __uint_as_float(p & 0xFFFF0000u); }
// The high halves of two values: bf16 by cutting off.
__device__ __forceinline__ uint32_t cut_bf16(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// 8 values as sums of P bf16 pieces, exactly. P = 1: bf16. P = 2: float16's 11
// significant bits, the first 8 cut off. P = 3: float32, v = p0 + 2^-7 p1 +
// 2^-16 p2: p0 the first 8 bits (a multiple of 2^-133, bf16's least step), p1
// 2^7 times what is left of v, rounded to the nearest 8 bits, and p2 2^9 times
// what is then left, which is 8 bits at most. Scaled so, the pieces of the
// least values keep all bits (p2's steps stand for 2^-149, float32's own), and
// none is larger than v, so their sums stay finite where those of |v| do. An
// infinity or a NaN is its own first piece and its others are zero.
constexpr float kPiece1 = 0x1p-7f, kPiece2 = 0x1p-9f;  // p1's unit in p0's, p2's in p1's
template <int P>
__device__ __forceinline__ void pieces8(const float v[8], uint4 out[P]) {
  uint32_t r[P][4];
  float rest[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[0][i] = cut_bf16(v[2 * i], v[2 * i + 1]);
    rest[2 * i] = v[2 * i] - low_bf16(r[0][i]), rest[2 * i + 1] = v[2 * i + 1] - high_bf16(r[0][i]);
  }
  // (The rest of a value that is not finite is NaN, and stays so in a sum; the
  // others' rests are far from float32's largest.)
  const float sum = ((rest[0] + rest[1]) + (rest[2] + rest[3])) + ((rest[4] + rest[5]) + (rest[6] + rest[7]));
  if (P > 1 && sum != sum) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (abs_bits(v[i]) >= kInfBits) rest[i] = 0.0f;
      if (abs_bits(v[i]) > kInfBits) r[0][i / 2] |= i % 2 ? 0x00400000u : 0x00000040u;  // (a NaN stays one)
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = rest[2 * i], b = rest[2 * i + 1];
    if (P == 2) r[P - 1][i] = cut_bf16(a, b);
    if (P == 3) {
      a *= 1.0f / kPiece1, b *= 1.0f / kPiece1;
      const uint32_t p = round_bf16(a, b);
      r[P - 2][i] = p;
      r[P - 1][i] = cut_bf16((a - low_bf16(p)) * (1.0f / kPiece2), (b - high_bf16(p)) * (1.0f / kPiece2));
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) out[p] = make_uint4(r[p][0], r[p][1], r[p][2], r[p][3]);
}
template <typename T>
struct Pieces {
  static constexpr int n = 3, sums = 3;  // (of different units, so with sums of their own)
};
template <>
struct Pieces<__bf16> {
  static constexpr int n = 1, sums = 1;
};
template <>
struct Pieces<_Float16> {
  static constexpr int n = 2, sums = 1;
};
template <typename V>
__device__ __forceinline__ V join_sums(const V (&s)[1]) {
  return s[0];
}
template <typename V>
__device__ __forceinline__ V join_sums(const V (&s)[3]) {
  return s[0] + kPiece1 * (s[1] + kPiece2 * s[2]);
}

}  // namespace px

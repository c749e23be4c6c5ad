// The arithmetic of the 8-bit codes that tokens (rows that share one scale) and the group norm's input are kept in.
//
// With `top` the largest magnitude that shares a scale, a value's code is 127 |x| / top, rounded to the nearest whole
// number, halves up, with the sign of x: -127 .. 127.  The scale, which turns codes back into values, is top / 127 in
// 32 bits.  A top below 2^-100 counts as zero (scale 0, codes 0); a NaN or an infinity makes the scale NaN and every
// code 0, so that all that shares it comes back as NaN.
//
// The codes are exactly that: no rounding of the arithmetic moves one across a half.  127 |x| / top can only lie exactly
// on a half or at least 1 / (254 X) of its own size from it, X being the significand of x as a whole number: 2^-19 for
// fp16, 2^-16 for bf16, 2^-32 for fp32.  So the factor 127 / top is taken larger by a share below that distance and above the
// errors of the factor, the product and the sum: a half is then always rounded up, and nothing below it is.  16-bit types
// compute in fp32 (factor larger by 2^-21, errors below 2^-22), fp32 values in fp64 (2^-45, 2^-50).
#pragma once

#include "device_utils.h"

namespace actnn {

constexpr float kTopSmallest = 0x1p-100f;
constexpr float kScaleLargest = 0x1.0204060000000p+121f;     // 127 times it is the largest below infinity

struct TokenScale {
  float scale;                          // what a code is multiplied by
  uint32_t keep;                        // all ones, or 0 where every code is 0
};
ACTNN_DEV TokenScale token_scale(float top) {
  TokenScale s;
  s.keep = top >= kTopSmallest && top <= 3.402823466e38f ? ~0u : 0u;
  s.scale = s.keep ? __builtin_fminf(top / 127.0f, kScaleLargest) : top < kTopSmallest ? 0.0f : __builtin_nanf("");
  return s;
}

// (an int conversion of a value that no int holds is one instruction that clamps, and `keep` drops what it gave)
template <typename T> struct Coder {
  float factor;
  Coder() = default;
  ACTNN_DEV explicit Coder(float top) : factor((127.0f / top) * (1.0f + 0x1p-21f)) {}
  ACTNN_DEV int code(float x) const { return (int)__builtin_fmaf(x, factor, __builtin_copysignf(0.5f, x)); }
};
template <> struct Coder<float> {
  double factor;
  Coder() = default;
  ACTNN_DEV explicit Coder(float top) : factor((127.0 / (double)top) * (1.0 + 0x1p-45)) {}
  ACTNN_DEV int code(float x) const { return (int)__builtin_fma((double)x, factor, __builtin_copysign(0.5, (double)x)); }
};
ACTNN_DEV uint32_t pack_codes(int a, int b, int c, int d) {
  return __builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x0c0c0400u) |
         __builtin_amdgcn_perm((uint32_t)d, (uint32_t)c, 0x04000c0cu);
}
// byte I of a word of codes, as a number (one instruction)
template <int I> ACTNN_DEV float code_value(uint32_t word) { return (float)(int8_t)(word >> (8 * I)); }

// Largest magnitudes as the values' bits without the sign: as whole numbers they order like the magnitudes, with
// infinity and then NaN on top, and 16-bit types go two at a time.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T> struct Top {                       // 16-bit types: two running maxima in a word
  uint32_t bits = 0;
  static ACTNN_DEV uint32_t larger(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  }
  ACTNN_DEV void add(const u32x4& v) {
    const uint32_t a = larger(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), b = larger(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu);
    bits = larger(bits, larger(a, b));
  }
  ACTNN_DEV uint32_t one() const { return bits >> 16 > (bits & 0xffffu) ? bits >> 16 : bits & 0xffffu; }
  static ACTNN_DEV float value(uint32_t one);
};
template <> ACTNN_DEV float Top<__half>::value(uint32_t one) { return half_bits_to_float(one); }
template <> ACTNN_DEV float Top<bf16_t>::value(uint32_t one) { return bf16_bits_to_float(one); }
template <> struct Top<float> {
  uint32_t bits = 0;
  static ACTNN_DEV uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
  ACTNN_DEV void add(const u32x4& v) {
    const uint32_t a = larger(v.x & 0x7fffffffu, v.y & 0x7fffffffu), b = larger(v.z & 0x7fffffffu, v.w & 0x7fffffffu);
    bits = larger(bits, larger(a, b));
  }
  ACTNN_DEV uint32_t one() const { return bits; }
  static ACTNN_DEV float value(uint32_t one) { return as_float(one); }
};
ACTNN_DEV uint32_t lanes_largest(uint32_t v) {           // over the wave, whole numbers
  auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  v = up(v, lane_xor<1>(v));
  v = up(v, lane_xor<2>(v));
  v = up(v, lane_xor<4>(v));
  v = up(v, lane_xor<8>(v));
  v = up(v, lane_xor<16>(v));
  return up(v, (uint32_t)__shfl_xor((int)v, 32));
}

// the elements of a 16-byte vector as floats, and their codes
template <typename T> constexpr int kVector = 16 / sizeof(T);
ACTNN_DEV void widen(const float*, const u32x4& v, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = as_float(v[i]);
}
ACTNN_DEV void widen(const __half*, const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = half_bits_to_float(v[i] & 0xffffu);
    f[2 * i + 1] = half_bits_to_float(v[i] >> 16);
  }
}
ACTNN_DEV void widen(const bf16_t*, const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = v[i];
    f[2 * i] = as_float(w << 16);
    f[2 * i + 1] = as_float(w & 0xffff0000u);
  }
}
ACTNN_DEV u32x4 narrow(const float*, const float (&f)[4]) {
  return (u32x4){as_uint(f[0]), as_uint(f[1]), as_uint(f[2]), as_uint(f[3])};
}
template <typename T> ACTNN_DEV u32x4 narrow(const T* p, const float (&f)[8]) { return words_of8(p, f); }

// the packed codes of a vector: one word of four for fp32, two words for 16-bit types
template <typename T> struct CodeWords { typedef u32x2 type; };
template <> struct CodeWords<float> { typedef uint32_t type; };
template <typename T>
ACTNN_DEV typename CodeWords<T>::type codes_of(const Coder<T>& coder, const float (&f)[kVector<T>], uint32_t keep) {
  if constexpr (sizeof(T) == 4) {
    return pack_codes(coder.code(f[0]), coder.code(f[1]), coder.code(f[2]), coder.code(f[3])) & keep;
  } else {
    return (u32x2){pack_codes(coder.code(f[0]), coder.code(f[1]), coder.code(f[2]), coder.code(f[3])) & keep,
                   pack_codes(coder.code(f[4]), coder.code(f[5]), coder.code(f[6]), coder.code(f[7])) & keep};
  }
}
// and back: the codes as numbers
ACTNN_DEV void code_values(uint32_t w, float (&f)[4]) {
  f[0] = code_value<0>(w); f[1] = code_value<1>(w); f[2] = code_value<2>(w); f[3] = code_value<3>(w);
}
ACTNN_DEV void code_values(u32x2 v, float (&f)[8]) {
  const uint32_t a = v.x, b = v.y;
  f[0] = code_value<0>(a); f[1] = code_value<1>(a); f[2] = code_value<2>(a); f[3] = code_value<3>(a);
  f[4] = code_value<0>(b); f[5] = code_value<1>(b); f[6] = code_value<2>(b); f[7] = code_value<3>(b);
}

// Codes 2 J and 2 J + 1 of a word times a scale, in 16 bits: one rounding for fp16 (the codes are made halves by putting them
// behind the exponent of 1024, and a mixed multiply-add rounds their product with the fp32 scale), two for bf16 (to 32 bits
// first).  Two and two and a half instructions a value.
template <typename T, int J> ACTNN_DEV uint32_t code_pair(uint32_t word, float scale);
template <> ACTNN_DEV uint32_t code_pair<bf16_t, 0>(uint32_t w, float s) {
  return pack_bf16x2(code_value<0>(w) * s, code_value<1>(w) * s);
}
template <> ACTNN_DEV uint32_t code_pair<bf16_t, 1>(uint32_t w, float s) {
  return pack_bf16x2(code_value<2>(w) * s, code_value<3>(w) * s);
}
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
template <int J> ACTNN_DEV uint32_t half_code_pair(uint32_t w, float s) {
  const f16x2_t off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  const uint32_t raised = __builtin_amdgcn_perm(w ^ 0x80808080u, 0x64646464u, J == 0 ? 0x00050004u : 0x00070006u);
  const f16x2_t q = __builtin_bit_cast(f16x2_t, raised) + off;
  const f16x2_t v = {(_Float16)__builtin_fmaf((float)q.x, s, 0.0f), (_Float16)__builtin_fmaf((float)q.y, s, 0.0f)};
  return __builtin_bit_cast(uint32_t, v);
}
template <> ACTNN_DEV uint32_t code_pair<__half, 0>(uint32_t w, float s) { return half_code_pair<0>(w, s); }
template <> ACTNN_DEV uint32_t code_pair<__half, 1>(uint32_t w, float s) { return half_code_pair<1>(w, s); }

}  // namespace actnn

// A matrix held in 8 bits: e4m3 codes [rows, Kp], Kp = K rounded up to 128, and one scale byte for
// each block of 128 columns, a power of two (2^(byte - 127)), rows of S = 4 ceil(K / 512) bytes.
//
// Of a block with largest finite magnitude a the exponent is the least whole e >= -126 with
// a <= 448 2^e, and a code is the nearest e4m3 value of x 2^-e (ties to even).  A value that is
// not finite becomes NaN, so that a product shows it.  Powers of two: a code does not depend on
// how a quotient was rounded, e4m3's own exponent makes up for the up to twofold range that a
// free scale would win, and the matrix cores take such scales inside the instruction.
#pragma once

#include "common.hpp"

namespace cobra {

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Scale byte of a block whose largest magnitude has the fp32 bits a: 448 = 1.75 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
  const int e = (int)(a >> 23) - 8 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(e < 1 ? 1 : e);
}
// The scale itself, 1 <= byte < 255.
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// Half of it, for conversions, which take 0 for 2^-127.
__device__ __forceinline__ float half_scale_of(uint32_t byte) { return __uint_as_float((byte << 23) - 0x800000u); }

// What the conversion needs of a 16- or 32-bit activation type.  A magnitude's bits order like the
// magnitudes do, so 16-bit values are compared two at a time; past kInf they are not finite.
template <typename T>
struct Quant;
template <>
struct Quant<f16> {
  static constexpr uint32_t kInf = 0x7c00u;
  static __device__ __forceinline__ float wide(uint32_t mag) { return (float)__builtin_bit_cast(f16, (uint16_t)mag); }
  static __device__ __forceinline__ uint32_t four(uint32_t x, uint32_t y, float s) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, x), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, __builtin_bit_cast(f16x2, y), s, true);
    return __builtin_bit_cast(uint32_t, r);
  }
};
template <>
struct Quant<bf16> {
  static constexpr uint32_t kInf = 0x7f80u;
  static __device__ __forceinline__ float wide(uint32_t mag) { return __uint_as_float(mag << 16); }
  static __device__ __forceinline__ uint32_t four(uint32_t x, uint32_t y, float s) {
    s16x2 r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, x), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2, y), s, true);
    return __builtin_bit_cast(uint32_t, r);
  }
};

// The larger magnitude of each half of w (N words of two 16-bit values), over all words.
template <int N>
__device__ __forceinline__ uint32_t largest16(const uint32_t (&w)[N]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}
// The words with everything that is not finite made NaN (e4m3's conversion would take an infinity
// for its largest code), and the largest finite magnitude.
template <typename T, int N>
__device__ __forceinline__ uint32_t finite16(uint32_t (&w)[N]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    if (lo >= Quant<T>::kInf) w[i] |= 0x7fffu;
    else m = max(m, lo);
    if (hi >= Quant<T>::kInf) w[i] |= 0x7fff0000u;
    else m = max(m, hi);
  }
  return m;
}

// Sixteen bytes at any element's address.
typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));

// Eight values from c on of a row of K >= 8 are loaded as those from min(c, K - 8) on, so that rows of any
// length take the same loads; here the first n > 0 that are not asked for go, zeros follow.
template <int N>
__device__ __forceinline__ void drop_first(uint32_t (&w)[N], int n) {
  constexpr int kPer = 8 / N;  // values of a word
#pragma unroll
  for (int k = N / 2; k >= 1; k /= 2)
    if ((n / kPer) & k) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = i + k < N ? w[i + k] : 0u;
    }
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0u;
  } else if (kPer == 2 && n & 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (w[i] >> 16) | (i + 1 < N ? w[i + 1] << 16 : 0u);
  }
}

}  // namespace cobra

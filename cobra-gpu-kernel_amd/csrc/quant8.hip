// Rows of 16- or 32-bit values into 8-bit blocks (quant8.hpp): one pass, each value read once.
//
// 16 lanes have a block of 128 columns, 8 each; their largest magnitude meets over four lane
// exchanges and the codes are converted from the loaded words, two at a time, the scale inside the
// conversion.  A wave has 512 columns of a row at a time, so that its scales are one word, or several rows
// of few columns.
// Bound by memory for many rows, by the launch for few.
#include "kernels.hpp"
#include "quant8.hpp"

namespace cobra {

namespace {

// Eight values of a lane as loaded.
template <typename T>
struct Eight {
  uint32_t w[sizeof(T) * 2];
};

// Eight columns of a row of K for column c, to be settled; SHORT: K < 8.
template <typename T, bool SHORT>
__device__ __forceinline__ Eight<T> load8_of(const T* row, int c, int K) {
  Eight<T> r{};
  if constexpr (SHORT) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (c + i < K) {
        if constexpr (sizeof(T) == 2)
          r.w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[c + i] << (16 * (i & 1));
        else
          r.w[i] = reinterpret_cast<const uint32_t*>(row)[c + i];
      }
  } else {
    const T* p = row + min(c, K - 8);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
      const Words q = reinterpret_cast<const Words*>(p)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[4 * i + e] = q[e];
    }
  }
  return r;
}

// Largest of a's 16-lane row, in every lane of it.
__device__ __forceinline__ uint32_t max16(uint32_t a) {
  float v = __uint_as_float(a);  // magnitudes' bits as fp32 magnitudes, none of them NaN
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  v = fmaxf(v, dpp_f32<0x140>(v));
  return __float_as_uint(v);
}

// The fp32 bits of the largest finite magnitude; what is not finite becomes NaN.
template <typename T>
__device__ __forceinline__ uint32_t largest_of(Eight<T>& x) {
  if constexpr (sizeof(T) == 2) {
    uint32_t m = largest16(x.w);
    if (__any(m >= Quant<T>::kInf)) m = finite16<T>(x.w);
    return __float_as_uint(Quant<T>::wide(m));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t a = x.w[i] & 0x7fffffffu;
      if (a >= 0x7f800000u) x.w[i] |= 0x7fffffffu;
      else m = max(m, a);
    }
    return m;
  }
}

template <typename T>
__device__ __forceinline__ uint2 codes_of(const Eight<T>& x, float s) {
  if constexpr (sizeof(T) == 2) {
    return make_uint2(Quant<T>::four(x.w[0], x.w[1], s), Quant<T>::four(x.w[2], x.w[3], s));
  } else {
    uint32_t r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s16x2 p = {0, 0};
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, __uint_as_float(x.w[4 * i]), __uint_as_float(x.w[4 * i + 1]), s,
                                                   false);
      p = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(p, __uint_as_float(x.w[4 * i + 2]), __uint_as_float(x.w[4 * i + 3]),
                                                   s, true);
      r[i] = __builtin_bit_cast(uint32_t, p);
    }
    return make_uint2(r[0], r[1]);
  }
}

// U units a wave, all of their loads asked for before the first is used.  A unit is 512 columns of a row,
// or with few columns R rows of 512 / R: 60 MB in rows of 128 take 16.4 us with four rows a unit and 30.6
// with one, in rows of 200 columns 18.4 and 21.4 with two and one.  Rows of every length take the same
// loads, at any element's address: 60 MB in rows of 8190 take 16.2 us, of 8191 18.5 (a value at a time
// 35.8), of 512 15.8, of 50 25.1 (157).
template <typename T, bool SHORT, int U, int R>
__global__ __launch_bounds__(256) void quantize8_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                        uint32_t* __restrict__ scale, int64_t rows, int64_t K,
                                                        uint32_t per_row, uint32_t units) {
  constexpr int kLanes = 64 / R;  // of a row
  const uint32_t lane = threadIdx.x & 63, sub = lane / kLanes;
  const uint32_t wave = __builtin_amdgcn_readfirstlane((blockIdx.x * 256 + threadIdx.x) >> 6);
  const uint32_t u0 = wave * U;
  const int kp = (int)((K + 127) & ~int64_t(127));
  auto row_of = [&](uint32_t u) { return R > 1 ? (int64_t)u * R + sub : (int64_t)(u / per_row); };
  auto col_of = [&](uint32_t u) { return (int)((R > 1 ? 0 : u % per_row) * 512 + (lane % kLanes) * 8); };
  Eight<T> v[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = u0 + i;
    if (u < units && (R == 1 || row_of(u) < rows)) v[i] = load8_of<T, SHORT>(x + row_of(u) * K, col_of(u), (int)K);
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const uint32_t u = u0 + i;
    if (u >= units) return;
    const int64_t row = row_of(u);
    const int c = col_of(u);
    const bool there = c < kp && (R == 1 || row < rows);
    if (R > 1 && row >= rows) v[i] = Eight<T>{};
    if (!SHORT && c + 8 > (int)K) drop_first(v[i].w, c + 8 - (int)K);
    const uint32_t mine = scale_byte(max16(largest_of(v[i])));
    const uint32_t byte = there ? mine : 127u;
    const uint2 q = codes_of(v[i], scale_of(byte));
    if (there) *reinterpret_cast<uint2*>(codes + row * kp + c) = q;
    // A row's word: its blocks' bytes, 127 past them.
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)byte, 16 * j);
      if (R == 1) word |= b << (8 * j);
      else if ((uint32_t)(16 * j / kLanes) == sub) word |= b << (8 * (j % (4 / R)));
    }
    if (R == 2) word |= 0x7f7f0000u;
    if (R == 4) word |= 0x7f7f7f00u;
    if (lane % kLanes == 0 && (R == 1 || row < rows)) scale[R == 1 ? u : row] = word;
  }
}

template <typename T, bool SHORT, int R>
hipError_t launch(const Quantize8Args& a, hipStream_t stream) {
  const int64_t per_row = (a.K + 511) / 512, units = R > 1 ? (a.M + R - 1) / R : a.M * per_row;
  if (units > 0x7fffffff || a.K > 0x7fffff00) return hipErrorInvalidValue;
  // Four units a wave once every CU has its eight workgroups with one: until then more waves
  // shorten the call, from there on more loads in flight for each do.
  const bool many = units > 4 * 8 * (int64_t)compute_units();
  const int64_t groups = many ? (units + 15) / 16 : (units + 3) / 4;
  auto* kernel = many ? quantize8_kernel<T, SHORT, 4, R> : quantize8_kernel<T, SHORT, 1, R>;
  return launch_status(kernel, dim3((unsigned)groups), dim3(256), stream, static_cast<const T*>(a.x),
                       static_cast<uint8_t*>(a.codes), static_cast<uint32_t*>(a.scale), a.M, a.K, (uint32_t)per_row,
                       (uint32_t)units);
}

template <typename T>
hipError_t launch_rows(const Quantize8Args& a, hipStream_t stream) {
  if (a.K < 8) return launch<T, true, 4>(a, stream);
  return a.K <= 128 ? launch<T, false, 4>(a, stream) : a.K <= 256 ? launch<T, false, 2>(a, stream)
                                                                  : launch<T, false, 1>(a, stream);
}

}  // namespace

hipError_t run_quantize8(const Quantize8Args& a, hipStream_t stream) {
  switch (a.dtype) {
    case kF16: return launch_rows<f16>(a, stream);
    case kBF16: return launch_rows<bf16>(a, stream);
    case kF32: return launch_rows<float>(a, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace cobra

// C[M,N] = A[M,K] . W[N,K]^T (+ bias, GELU, row masks, + resid) with both matrices in 8 bits and a
// power-of-two scale for each row and block of 128 columns (quant8.hpp):
//   c = sum_j 2^(ea[m,j] + ew[n,j]) sum_{k in block j} a[m,k] w[n,k]
// Two kinds of matrix instructions.
// * Exact: codes become bf16 in registers, with their scale inside the conversion (4 significant bits
//   and a power of two), and v_mfma_*_bf16 adds their products in fp32.  Each operand is widened with half of its
//   scale, since a block's largest value may round to 2^128, which bf16 has not; sums are multiplied by 4.
//   Nothing is rounded but blocks under 2^-115 (scale bytes 1 to 3), whose least values become whole
//   multiples of 2^-132, bf16's least step twice.
// * Scaled: v_mfma_scale_f32_32x32x64_f8f6f4 takes the codes as they are and one scale byte for each
//   row and 32 columns of an operand, at twice the rate.  All lanes that hold parts of a row's
//   block give the block's byte, so it does not matter which columns the instruction counts to which
//   lane.  But it adds eight products at a time and cuts each where it falls under 2^-13 of
//   the largest one's exponent (measured, as for the instructions without scales; the sums of eight
//   meet in fp32): 4e-5 to 6e-5 of a result in the root mean square, and where large products cancel
//   what they leave may be gone.  Only bf16 results take this kind: their own rounding is 1.6e-3 in the
//   root mean square, and half a step of one as large as the largest product, 2^-8, covers the 7 2^-13 of
//   it that an eight can lose.  An fp16's rounding is 2e-4, an fp32's 3e-8: the exact kind, for any
//   number of rows.
//
// Two kernels.  Up to 16 rows of A the weights' bytes are all that counts: linear8_few_kernel
// (exact) has 16 or more rows of W a workgroup, split along K over its waves, and takes 16-bit
// activations as they are, quantising them in the registers that the product reads.  More rows go
// through tiles in LDS.
#include <type_traits>

#include "kernels.hpp"
#include "lds_dma.hpp"
#include "quant8.hpp"

namespace cobra {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 join8(const i32x4& a, const i32x4& b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Eight codes times a scale, exactly.
__device__ __forceinline__ bf16x8 widen(uint32_t x, uint32_t y, float scale) {
  struct {
    bf16x2 p[4];
  } q;
  q.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, false);
  q.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, true);
  q.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, false);
  q.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, scale, true);
  return __builtin_bit_cast(bf16x8, q);
}
__device__ __forceinline__ f32x16 mfma8(const i32x8& a, const i32x8& b, const f32x16& c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// What products of operands with half of their scales are short of.
constexpr float kUnhalve = 4.f;

struct Args {
  const void* a;
  const uint8_t *a_scale, *w, *w_scale;
  const float* bias;
  const void* resid;
  const uint8_t* row_mask;
  void* c;
  int64_t M;
  int N, K;      // K: columns of 16-bit activations
  int kp, s;     // columns of codes, bytes of a row of scales
  int resid_dtype, c_dtype, epi;
};

// Element i of a matrix of one of the three types.
__device__ __forceinline__ float get(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  if (dtype == kF16) return (float)static_cast<const f16*>(p)[i];
  return (float)static_cast<const bf16*>(p)[i];
}
__device__ __forceinline__ void put(void* p, int dtype, int64_t i, float v) {
  if (dtype == kF32) static_cast<float*>(p)[i] = v;
  else if (dtype == kF16) static_cast<f16*>(p)[i] = (f16)v;
  else static_cast<bf16*>(p)[i] = (bf16)v;
}
// Four elements at any element's address.
typedef float f32x4e __attribute__((ext_vector_type(4), aligned(4)));
typedef f16 f16x4e __attribute__((ext_vector_type(4), aligned(2)));
typedef bf16 bf16x4e __attribute__((ext_vector_type(4), aligned(2)));

// Four consecutive elements from i on.
__device__ __forceinline__ f32x4 get4(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return *reinterpret_cast<const f32x4e*>(static_cast<const float*>(p) + i);
  f32x4 r;
  if (dtype == kF16) {
    const f16x4 h = *reinterpret_cast<const f16x4e*>(static_cast<const f16*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (float)h[e];
  } else {
    const bf16x4 h = *reinterpret_cast<const bf16x4e*>(static_cast<const bf16*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (float)h[e];
  }
  return r;
}
__device__ __forceinline__ void put4(void* p, int dtype, int64_t i, const f32x4& v) {
  if (dtype == kF32) {
    *reinterpret_cast<f32x4e*>(static_cast<float*>(p) + i) = v;
  } else if (dtype == kF16) {
    f16x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (f16)v[e];
    *reinterpret_cast<f16x4e*>(static_cast<f16*>(p) + i) = h;
  } else {
    bf16x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (bf16)v[e];
    *reinterpret_cast<bf16x4e*>(static_cast<bf16*>(p) + i) = h;
  }
}

// -- few rows --------------------------------------------------------------------------

// A lane's 32 columns of a block of one row of activations: codes and the block's scale.  16-bit values
// are quantised here: a row's block lies in the four lanes l, l + 16, l + 32, l + 48.  ODD: K >= 8 is no
// multiple of 8 (one row of 1023, 1024 rows of W: 3.8 to 4.5 us, quantised first 6.0 to 7.7).
template <typename TA, bool ODD>
struct RowBlock {
  uint32_t w[16];
  __device__ __forceinline__ void load(const Args& a, int64_t m, bool there, int j, int g) {
    const TA* p = static_cast<const TA*>(a.a) + m * a.K;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = 128 * j + 64 * h + 16 * g;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there && c + 8 * q < a.K) {
          if constexpr (ODD) {
            const Words x = *reinterpret_cast<const Words*>(p + min(c + 8 * q, a.K - 8));
            v = make_uint4(x[0], x[1], x[2], x[3]);
          } else {
            v = *reinterpret_cast<const uint4*>(p + c + 8 * q);
          }
        }
        w[8 * h + 4 * q] = v.x;
        w[8 * h + 4 * q + 1] = v.y;
        w[8 * h + 4 * q + 2] = v.z;
        w[8 * h + 4 * q + 3] = v.w;
      }
    }
    if constexpr (ODD) {
      if (128 * j + 128 > a.K) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int past = 128 * j + 64 * (k >> 1) + 16 * g + 8 * (k & 1) + 8 - a.K;
          uint32_t x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = w[4 * k + e];
          if (past > 0) drop_first(x, past);
#pragma unroll
          for (int e = 0; e < 4; ++e) w[4 * k + e] = x[e];
        }
      }
    }
  }
  __device__ __forceinline__ i32x8 codes(uint32_t& byte) {
    uint32_t m = largest16(w);
    if (__any(m >= Quant<TA>::kInf)) m = finite16<TA>(w);
    float v = Quant<TA>::wide(m);
    const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = max_xor32(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
    byte = scale_byte(__float_as_uint(v));
    const float scale = scale_of(byte);
    i32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (int)Quant<TA>::four(w[2 * i], w[2 * i + 1], scale);
    return r;
  }
};
template <>
struct RowBlock<uint8_t, false> {
  i32x4 lo, hi;
  uint32_t b;
  __device__ __forceinline__ void load(const Args& a, int64_t m, bool there, int j, int g) {
    lo = i32x4{0, 0, 0, 0};
    hi = lo;
    b = 127;
    if (there) {
      const uint8_t* p = static_cast<const uint8_t*>(a.a) + m * a.kp + 128 * j + 16 * g;
      lo = *reinterpret_cast<const i32x4*>(p);
      hi = *reinterpret_cast<const i32x4*>(p + 64);
      b = a.a_scale[m * a.s + j];
    }
  }
  __device__ __forceinline__ i32x8 codes(uint32_t& byte) {
    byte = b;
    return join8(lo, hi);
  }
};

// A workgroup has NT sets of 16 rows of W, its eight waves every eighth block of K each.
//
// Bound by memory behind a launch's and a first load's latency: 8192 x 4096 weights take 10.8 us with
// one row (9.9 as codes), 3.1 TB/s in all, where the bytes alone are 6.6 us at a copy's rate; 12.4 with 16
// rows.  32 rows of W a workgroup where that still gives every CU one, 16 otherwise: each workgroup reads and
// quantises all of A (16 rows, 8192 x 4096: 12.4 us against 16.2 with 16; 4096 x 8192: 16.0 against
// 20.9 with 32).  Several blocks' loads asked for together gained nothing (12.4 to 14.9 us, 16.0 to 16.8),
// nor did 16 waves (12.6, 16.3).  From 17 rows on quantising once and a tile kernel are faster: 32 rows
// 13 us against 16.8, 64 rows 15 against 28.
template <typename TA, bool ODD, int NT>
__global__ __launch_bounds__(512) void linear8_few_kernel(Args a) {
  constexpr int kWaves = 8;
  __shared__ f32x4 part[kWaves][NT][64];
  const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 16 * NT;
  const int blocks = a.kp >> 7;
  const uint8_t *w[NT], *ws[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {  // rows past N give columns that are never stored
    const int64_t n = min(n0 + 16 * t + r, a.N - 1);
    w[t] = a.w + n * a.kp + 16 * g;
    ws[t] = a.w_scale + n * a.s;
  }
  f32x4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int j = wave; j < blocks; j += kWaves) {
    i32x8 c[NT];
    uint32_t wb[NT];
    RowBlock<TA, ODD> x;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      c[t] = join8(*reinterpret_cast<const i32x4*>(w[t] + 128 * j), *reinterpret_cast<const i32x4*>(w[t] + 128 * j + 64));
      wb[t] = ws[t][j];
    }
    x.load(a, r, r < a.M, j, g);
    uint32_t row_byte;
    const i32x8 q = x.codes(row_byte);
    const float row_scale = half_scale_of(row_byte);
    bf16x8 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = widen(q[2 * k], q[2 * k + 1], row_scale);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float scale = half_scale_of(wb[t]);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[t] = mfma16(widen(c[t][2 * k], c[t][2 * k + 1], scale), y[k], acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  // A thread has four columns of a row: the waves' shares in their order.
  for (int q = threadIdx.x; q < NT * 64; q += kWaves * 64) {
    const int tile = q >> 6, l = q & 63;
    const int m = l & 15, n = n0 + 16 * tile + 4 * (l >> 4);
    if (m >= a.M || n >= a.N) continue;
    f32x4 v = part[0][tile][l];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) v += part[k][tile][l];
    const bool padded = (a.epi & (kEpiMaskBranch | kEpiMaskResid)) && a.row_mask[m] == 0;
    const bool four = n + 4 <= a.N;
    const int64_t at = (int64_t)m * a.N + n;
    f32x4 b = {0.f, 0.f, 0.f, 0.f}, e = b;
    if (four) {
      if (a.bias) b = *reinterpret_cast<const f32x4*>(a.bias + n);
      if (a.resid) e = get4(a.resid, a.resid_dtype, at);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) {
          if (a.bias) b[i] = a.bias[n + i];
          if (a.resid) e[i] = get(a.resid, a.resid_dtype, at + i);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = fmaf(v[i], kUnhalve, b[i]);
      if (a.epi & kEpiGelu) v[i] = gelu_erf(v[i]);
      if (padded && (a.epi & kEpiMaskBranch)) v[i] = 0.f;
      v[i] += e[i];
      if (padded && (a.epi & kEpiMaskResid)) v[i] *= 0.f;
    }
    if (four) {
      put4(a.c, a.c_dtype, at, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) put(a.c, a.c_dtype, at + i, v[i]);
    }
  }
}

// -- many rows -------------------------------------------------------------------------

// 4 bytes per lane from a per-lane address to lds + 4 * lane (lds_dma.hpp: dma16_untracked).
__device__ __forceinline__ void dma4_untracked(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(src) : "memory");
}

// A tile of BM x BN by WM x WN waves; a k-tile is one block of 128 columns.  A stage of LDS holds
// the rows' codes (A's, then W's), 128 bytes each with 16-byte chunks swizzled by row as in the
// 16-bit kernel, and behind them the rows' words of four scale bytes.  KS groups of such waves have a
// k-tile each at a time, with stages of their own, and are added at the end.
//
// Large tiles are bound by the matrix cores (8192^3 2635 TFLOP/s of 4600 that the instruction reaches by
// itself, with the clock that such a load leaves), small ones by how much a CU has in flight: a CU alone
// takes in some 21 GB/s from memory, so few rows want as many workgroups as there are CUs, and two groups
// of waves in each.  64 rows, 4096 x 4096 weights take 8.4 us in tiles of 64 x 32 and two groups, 9.3 with
// one, 11.7 in 64 x 64, 11.0 there with two groups; 64 rows, 8192 x 4096 12.1, 12.6, 15.9 and 16.2.
template <int BM, int BN, int WM, int WN, int ST, int KS>
struct Tile {
  static constexpr int NW = WM * WN, NT = NW * KS * 64;  // waves of a group, threads
  static constexpr int WTM = BM / WM, WTN = BN / WN, TM = WTM / 32, TN = WTN / 32;
  static constexpr int ROWS = BM + BN;
  static constexpr int SCALES = (ROWS + 63) / 64;  // transfers of 64 rows' scale words
  static constexpr int PART = ROWS * 128 + SCALES * 256, STAGE = PART * KS;
  static constexpr int LPT = ROWS / 8 / NW;     // transfers of 8 rows' codes a wave and k-tile; one more of scales
  static constexpr int EPW = WN * 32, LDC = EPW + 4;
  static constexpr int EPI_LDS = BM * LDC * 4;
  static constexpr int LDS = ST * STAGE > EPI_LDS ? ST * STAGE : EPI_LDS;
  static_assert(WTM % 32 == 0 && WTN % 32 == 0 && BM % 64 == 0 && BN % 32 == 0, "wave tile");
  static_assert(ROWS / 8 % NW == 0, "every wave issues the same number of transfers");
  static_assert(LDS <= 163840, "LDS budget");
  static_assert(TN <= 4, "slices of the epilogue");
};

__device__ __forceinline__ int chunk_swz(int row) { return (row >> 1) & 7; }

template <int BM, int BN, int WM, int WN, int ST, int KS, bool EXACT>
__device__ __forceinline__ void mainloop(const Args& a, int64_t m0, int n0, char* smem,
                                         f32x16 (&acc)[BN / WN / 32][BM / WM / 32]) {
  using T = Tile<BM, BN, WM, WN, ST, KS>;
  constexpr int NW = T::NW, LPT = T::LPT;
  const int tid = threadIdx.x, lane = tid & 63;
  const int group = __builtin_amdgcn_readfirstlane(tid >> 6) / NW, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW;
  const int wm = wave / WN, wn = wave % WN;
  const int li = lane & 31, g = lane >> 5;
  smem += group * T::PART;  // of each stage
  const uint8_t* A = static_cast<const uint8_t*>(a.a) + m0 * a.kp;
  const uint8_t* W = a.w + (int64_t)n0 * a.kp;
  // Rows past M or N are the last one: their products are never stored.
  unsigned src_off[LPT];
#pragma unroll
  for (int i = 0; i < LPT; ++i) {
    const int row = 8 * (wave + i * NW) + (lane >> 3);
    const int chunk = (lane & 7) ^ chunk_swz(row);
    const int64_t at = row < BM ? min(m0 + row, a.M - 1) - m0 : (int64_t)min(n0 + row - BM, a.N - 1) - n0;
    src_off[i] = (unsigned)(at * a.kp + chunk * 16);
  }
  const int srow = min(64 * (wave % T::SCALES) + lane, T::ROWS - 1);
  const uint8_t* scales = srow < BM ? a.a_scale + min(m0 + srow, a.M - 1) * a.s
                                    : a.w_scale + (int64_t)min(n0 + srow - BM, a.N - 1) * a.s;
  const uint32_t lds0 = lds_addr(smem);
  constexpr int kAll = LPT + 1;  // transfers a wave and k-tile
  const int KT = a.kp >> 7, steps = (KT + KS - 1) / KS;
  // Transfer i of this group's k-tile of a step to its stage (where there is none, of the last).
  auto transfer = [&](int step, int i) {
    const uint32_t dst = lds0 + (step % ST) * T::STAGE;
    const int kt = min(step * KS + group, KT - 1);
    if (i < LPT)
      dma16_untracked((8 * (wave + i * NW) < BM ? A : W) + 128 * kt, src_off[i], dst + (wave + i * NW) * 1024);
    else
      dma4_untracked(scales + (kt & ~3), dst + T::ROWS * 128 + (wave % T::SCALES) * 256);
  };

#pragma unroll
  for (int j = 0; j < T::TN; ++j)
#pragma unroll
    for (int i = 0; i < T::TM; ++i) acc[j][i] = zero16();

  const int sw = chunk_swz(li);
  const int arow = wm * T::WTM + li, wrow = BM + wn * T::WTN + li;
#pragma unroll
  for (int s = 0; s < ST; ++s)
    if (s < steps) {
#pragma unroll
      for (int i = 0; i < kAll; ++i) transfer(s, i);
    }

  // Operands of half a k-tile (64 columns), in two sets: a half's products run while the next
  // half's reads and the transfers that refill its stage are in flight, one of each between two
  // products.  In front of them all, a wave's reads kept its matrix core waiting.
  i32x8 af[2][T::TM], wf[2][T::TN];
  int as[T::TM], ws[T::TN], an[T::TM], wnx[T::TN];
  constexpr int kFrags = T::TM + T::TN, kProducts = T::TM * T::TN;
  auto read = [&](const char* st, int kk, int f) {
    const int c0 = ((4 * kk + g) ^ sw) * 16, c1 = ((4 * kk + 2 + g) ^ sw) * 16;
    const char* p = st + (f < T::TN ? wrow + f * 32 : arow + (f - T::TN) * 32) * 128;
    const i32x8 x = join8(*reinterpret_cast<const i32x4*>(p + c0), *reinterpret_cast<const i32x4*>(p + c1));
    if (f < T::TN) wf[kk][f] = x;
    else af[kk][f - T::TN] = x;
  };
  auto read_scales = [&](const char* st) {
    const int* p = reinterpret_cast<const int*>(st + T::ROWS * 128);
#pragma unroll
    for (int j = 0; j < T::TN; ++j) wnx[j] = p[wrow + j * 32];
#pragma unroll
    for (int i = 0; i < T::TM; ++i) an[i] = p[arow + i * 32];
  };
  // Half kk's products; between(x) after product x of kProducts.
  auto products = [&](int kk, auto&& between) {
    if constexpr (EXACT) {
      bf16x8 y[T::TM][4];
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) y[i][k] = widen(af[kk][i][2 * k], af[kk][i][2 * k + 1], half_scale_of(as[i] & 255));
#pragma unroll
      for (int j = 0; j < T::TN; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bf16x8 z = widen(wf[kk][j][2 * k], wf[kk][j][2 * k + 1], half_scale_of(ws[j] & 255));
#pragma unroll
          for (int i = 0; i < T::TM; ++i) acc[j][i] = mfma32x32x16(z, y[i][k], acc[j][i]);
        }
#pragma unroll
        for (int i = 0; i < T::TM; ++i) between(j * T::TM + i);
      }
    } else {
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          acc[j][i] = mfma8(wf[kk][j], af[kk][i], acc[j][i], ws[j], as[i]);
          __builtin_amdgcn_sched_barrier(0);
          between(j * T::TM + i);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  };
  // Wait for the oldest k-tile in flight, of which there are n.
  auto wait_oldest = [&](int n) {
    if (ST >= 4 && n >= 4) wait_vmcnt<(ST >= 4 ? 3 : 0) * kAll>();
    else if (ST >= 3 && n >= 3) wait_vmcnt<(ST >= 3 ? 2 : 0) * kAll>();
    else if (n >= 2) wait_vmcnt<kAll>();
    else wait_vmcnt<0>();
  };
  // One step.  MORE: there is a next one, FILL: and one to refill the stage with.  The barrier
  // stands where a wave has read all of its operands of the step and its own transfers of the
  // next have landed.
  auto take = [&](int at, auto more, auto fill) {
    constexpr bool MORE = decltype(more)::value, FILL = decltype(fill)::value;
    const char* st = smem + (at % ST) * T::STAGE;
    const int kt = at * KS + group;
    if (!MORE && KS > 1 && kt >= KT) return;
#pragma unroll
    for (int j = 0; j < T::TN; ++j) ws[j] = wnx[j] >> (8 * (kt & 3));
#pragma unroll
    for (int i = 0; i < T::TM; ++i) as[i] = an[i] >> (8 * (kt & 3));
    products(0, [&](int x) {
#pragma unroll
      for (int f = x * kFrags / kProducts; f < (x + 1) * kFrags / kProducts; ++f) read(st, 1, f);
    });
    if constexpr (MORE) {
      wait_oldest(FILL ? ST - 1 : min(ST - 1, steps - 1 - at));
      lds_barrier();
    }
    const char* next = smem + ((at + 1) % ST) * T::STAGE;
    if constexpr (MORE) read_scales(next);
    products(1, [&](int x) {
      if constexpr (MORE) {
#pragma unroll
        for (int f = x * kFrags / kProducts; f < (x + 1) * kFrags / kProducts; ++f) read(next, 0, f);
      }
      if constexpr (FILL) {
#pragma unroll
        for (int i = x * kAll / kProducts; i < (x + 1) * kAll / kProducts; ++i) transfer(at + ST, i);
      }
    });
  };
  wait_oldest(min(ST, steps));
  stage_barrier();
#pragma unroll
  for (int f = 0; f < kFrags; ++f) read(smem, 0, f);
  read_scales(smem);
  int at = 0;
  for (; at + ST < steps; ++at) take(at, std::true_type(), std::true_type());
  for (; at + 1 < steps; ++at) take(at, std::true_type(), std::false_type());
  take(at, std::false_type(), std::false_type());
}

// Results whose rounding hides what the scaled instructions cut take them; the others' products are exact.
template <typename TC>
constexpr bool kExactSums = !std::is_same<TC, bf16>::value;

template <int BM, int BN, int WM, int WN, int ST, int KS, int GM, typename TC>
__global__ __launch_bounds__(WM* WN* KS * 64) void linear8_tile_kernel(Args a) {
  using T = Tile<BM, BN, WM, WN, ST, KS>;
  constexpr int NT = T::NT;
  __shared__ __attribute__((aligned(1024))) char smem[T::LDS];
  // Tile order as in the 16-bit kernel: an XCD runs a contiguous range of ids, which walk GM row
  // blocks x all column blocks.
  const int nbn = (a.N + BN - 1) / BN;
  const int nbm = (int)((a.M + BM - 1) / BM);
  const int tile = xcd_remap(blockIdx.x, gridDim.x);
  const int group = tile / (GM * nbn);
  const int first_m = group * GM;
  const int gm = min(nbm - first_m, GM);
  const int in_group = tile - group * GM * nbn;
  const int64_t m0 = (int64_t)(first_m + in_group % gm) * BM;
  const int n0 = (in_group / gm) * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int split = __builtin_amdgcn_readfirstlane(tid >> 6) / T::NW, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % T::NW;
  const int wm = wave / WN, wn = wave % WN;
  const int li = lane & 31, g = lane >> 5;

  f32x16 acc[T::TN][T::TM];
  mainloop<BM, BN, WM, WN, ST, KS, kExactSums<TC>>(a, m0, n0, smem, acc);
  __syncthreads();  // every wave is done with the operand stages

  // In TN slices of 32 columns for each wave column, through LDS as fp32 rows, then written 16
  // bytes a lane with the epilogue's options, at any element's address; the last columns of an N not in
  // groups of that many element by element (with all of them so 8192 x 4096 x 4091 takes
  // 217 us in place of 160, quantising with it).
  float* Cs = reinterpret_cast<float*>(smem);
  constexpr int CPL = 16 / (int)sizeof(TC), LPR = T::EPW / CPL, RPP = NT / LPR, NP = BM > RPP ? BM / RPP : 1;
  static_assert(NT % LPR == 0 && (BM % RPP == 0 || RPP > BM) && 32 % CPL == 0, "epilogue geometry");
  const int cl = (tid % LPR) * CPL;
  const int ccol = (cl / 32) * T::WTN + (cl % 32);
  const bool masks = a.epi & (kEpiMaskBranch | kEpiMaskResid);
  // (A template for each slice: as a loop, the accumulators' index stayed a variable, and they went to
  // scratch.)
  auto slice = [&](auto jc) {
    constexpr int j = decltype(jc)::value;
    // The groups' shares one after the other.
#pragma unroll
    for (int k = KS - 1; k >= 0; --k) {
      if (k < KS - 1) __syncthreads();
      if (KS == 1 || split == k) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < T::TM; ++i) {
            f32x4* at = reinterpret_cast<f32x4*>(Cs + (wm * T::WTM + i * 32 + li) * T::LDC + wn * 32 + 8 * q + 4 * g);
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[j][i][4 * q + e];
            if (k < KS - 1) v += *at;
            *at = v;
          }
      }
    }
    const int n = n0 + ccol + j * 32;
    const int live = a.N - n;  // columns that are there
    f32x4 bv[CPL / 4];
#pragma unroll
    for (int h = 0; h < CPL / 4; ++h) {
      bv[h] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (a.bias && live >= CPL) bv[h] = *reinterpret_cast<const f32x4*>(a.bias + n + 4 * h);
    }
    if (a.bias && live < CPL) {
#pragma unroll
      for (int e = 0; e < CPL; ++e)
        if (e < live) bv[e >> 2][e & 3] = a.bias[n + e];
    }
    // A row of the slice: its LDS place, product, bias and GELU.
    auto value = [&](int p, int h) {
      f32x4 v = *reinterpret_cast<const f32x4*>(Cs + (tid / LPR + p * RPP) * T::LDC + cl + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = kExactSums<TC> ? fmaf(v[e], kUnhalve, bv[h][e]) : v[e] + bv[h][e];
      if (a.epi & kEpiGelu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_erf(v[e]);
      }
      return v;
    };
    auto store = [&](int64_t m, const f32x4 (&v)[CPL / 4]) {
      TC* at = static_cast<TC*>(a.c) + m * a.N + n;
      if (live < CPL) {
#pragma unroll
        for (int e = 0; e < CPL; ++e)
          if (e < live) at[e] = (TC)v[e >> 2][e & 3];
      } else if constexpr (sizeof(TC) == 4) {
        *reinterpret_cast<f32x4e*>(at) = v[0];
      } else {
        typename Op16<TC>::V8 hv;
#pragma unroll
        for (int e = 0; e < 8; ++e) hv[e] = (TC)v[e >> 2][e & 3];
        *reinterpret_cast<Words*>(at) = __builtin_bit_cast(Words, hv);
      }
    };
    // This thread's rows: first, first + RPP, ..
    const int64_t first = RPP <= BM || tid / LPR < BM ? m0 + tid / LPR : a.M;
    // Loads share a counter with the stores: one between two passes would wait for the stores of
    // the pass before it.  So there are none in the loop without residual and masks (which is no
    // longer than it is because a tile runs it once, its instructions coming from memory), and with
    // them all of a slice's are asked for before its first store.
    if (!a.resid && !masks) {
      __syncthreads();
      if (live > 0) {
#pragma unroll 2
        for (int p = 0; p < NP; ++p) {
          if (first + p * RPP >= a.M) break;
          f32x4 v[CPL / 4];
#pragma unroll
          for (int h = 0; h < CPL / 4; ++h) v[h] = value(p, h);
          store(first + p * RPP, v);
        }
      }
    } else {
      f32x4 rv[NP][CPL / 4];
      uint32_t padded = 0;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int64_t m = min(first + p * RPP, a.M - 1);
        if (masks && a.row_mask[m] == 0) padded |= 1u << p;
#pragma unroll
        for (int h = 0; h < CPL / 4; ++h) {
          rv[p][h] = f32x4{0.f, 0.f, 0.f, 0.f};
          if (a.resid && live >= CPL) rv[p][h] = get4(a.resid, a.resid_dtype, m * a.N + n + 4 * h);
        }
        if (a.resid && live < CPL) {
#pragma unroll
          for (int e = 0; e < CPL; ++e)
            if (e < live) rv[p][e >> 2][e & 3] = get(a.resid, a.resid_dtype, m * a.N + n + e);
        }
      }
      __syncthreads();
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        if (live > 0 && first + p * RPP < a.M) {
          f32x4 v[CPL / 4];
#pragma unroll
          for (int h = 0; h < CPL / 4; ++h) {
            v[h] = value(p, h);
            if ((padded >> p & 1) && (a.epi & kEpiMaskBranch)) v[h] = f32x4{0.f, 0.f, 0.f, 0.f};
            v[h] += rv[p][h];
            if ((padded >> p & 1) && (a.epi & kEpiMaskResid)) v[h] *= 0.f;
          }
          store(first + p * RPP, v);
        }
      }
    }
    if (j + 1 < T::TN) __syncthreads();
  };
  slice(std::integral_constant<int, 0>());
  if constexpr (T::TN > 1) slice(std::integral_constant<int, 1>());
  if constexpr (T::TN > 2) slice(std::integral_constant<int, 2>());
  if constexpr (T::TN > 3) slice(std::integral_constant<int, 3>());
}

template <int BM, int BN, int WM, int WN, int ST, int KS, int GM, typename TC>
hipError_t launch_tile(const Args& a, hipStream_t stream) {
  const int64_t tiles = ((a.M + BM - 1) / BM) * (int64_t)((a.N + BN - 1) / BN);
  if (tiles > 0x7fffff) return hipErrorInvalidValue;
  return launch_status(linear8_tile_kernel<BM, BN, WM, WN, ST, KS, GM, TC>, dim3((unsigned)tiles),
                       dim3(WM * WN * KS * 64), stream, a);
}

// Tile choice: the candidate with the least estimated time, as for the 16-bit kernel.  n workgroups
// fall to each CU, per_cu at a time; a group of r takes `fixed` (launch, first loads, epilogue) plus
// per k-tile the larger of `step` (one workgroup's chain) and r x `busy` (its share of the CU).  Fits
// (us) to timings of every candidate over M 64 .. 16384, N and K 1000 .. 8192, for the scaled
// kind and the exact one: 8192 x 4096 x 4096 takes 114.8 us in 256 x 256 tiles (2394 TFLOP/s) and 146 in
// 128 x 128, 8192^3 417 (2635 TFLOP/s; a library product of e4m3 2605 to 2675 on the same cards) and 539,
// 512 x 4096 x 4096 44.6, 26.6, 16.4 and 19.7 in the four, 128 x 4096 x 4096 37.8, 19.5, 14.8 and 10.6.
// Exact, fp32 results: 8192 x 4096 x 4096 221 us in 256 x 256 and 241 in 128 x 128, 8192^3 790
// (1391 TFLOP/s; a library product in bf16 1308 to 1339) and 881.  Exact, fp16 results, in the tiles chosen: 8192^3
// 763, 8192 x 4096 x 4096 200 (116 scaled), 512 x 4096 x 4096 24.8 (16.1), 64 x 4096 x 4096 10.6 (7.8).
struct TileCand {
  int bm, bn, per_cu;
  double fixed, step, busy;
};
constexpr int kTiles = 5;
constexpr TileCand kScaled[kTiles] = {{256, 256, 1, 11.0, 1.00, 1.45}, {128, 128, 2, 4.4, 0.47, 0.50},
                                      {128, 64, 2, 4.1, 0.36, 0.28},   {64, 64, 2, 3.5, 0.22, 0.21},
                                      {64, 32, 1, 2.9, 0.20, 0.23}};
constexpr TileCand kExact[kTiles] = {{256, 256, 1, 21.0, 1.80, 2.75}, {128, 128, 2, 8.7, 0.67, 0.80},
                                     {128, 64, 2, 6.0, 0.58, 0.51},   {64, 64, 2, 4.8, 0.37, 0.39},
                                     {64, 32, 1, 3.6, 0.21, 0.235}};

int pick_tile(const TileCand (&tiles)[kTiles], const Args& a) {
  const int64_t cus = compute_units();
  const double kt = a.kp / 128;
  int best = 0;
  double best_t = 1e300;
  for (int i = 0; i < kTiles; ++i) {
    const TileCand& c = tiles[i];
    const int64_t all = ((a.M + c.bm - 1) / c.bm) * (int64_t)((a.N + c.bn - 1) / c.bn);
    const int64_t n = (all + cus - 1) / cus, rest = n % c.per_cu;
    auto group = [&](double r) { return c.fixed + kt * (r * c.busy > c.step ? r * c.busy : c.step); };
    const double t = (double)(n / c.per_cu) * group(c.per_cu) + (rest ? group((double)rest) : 0.0);
    if (t < best_t) {
      best_t = t;
      best = i;
    }
  }
  return best;
}

template <typename TC>
hipError_t dispatch_tile(const Args& a, hipStream_t stream) {
  switch (pick_tile(kExactSums<TC> ? kExact : kScaled, a)) {
    case 0: return launch_tile<256, 256, 4, 2, 2, 1, 4, TC>(a, stream);
    case 1: return launch_tile<128, 128, 2, 2, 2, 1, 8, TC>(a, stream);
    case 2: return launch_tile<128, 64, 2, 2, 3, 1, 8, TC>(a, stream);
    case 3: return launch_tile<64, 64, 2, 2, 4, 1, 8, TC>(a, stream);
    default: return launch_tile<64, 32, 2, 1, 4, 2, 8, TC>(a, stream);
  }
}

template <int NT, typename TA, bool ODD>
hipError_t launch_few(const Args& a, hipStream_t stream) {
  return launch_status(linear8_few_kernel<TA, ODD, NT>, dim3((unsigned)((a.N + 16 * NT - 1) / (16 * NT))), dim3(512),
                       stream, a);
}
template <typename TA, bool ODD>
hipError_t dispatch_few(const Args& a, hipStream_t stream) {
  const bool wide = (a.N + 31) / 32 >= compute_units();
  return wide ? launch_few<2, TA, ODD>(a, stream) : launch_few<1, TA, ODD>(a, stream);
}

constexpr int64_t kFewRows = 16;

// Few rows of 16-bit activations that the product itself quantises.
bool quantised_inside(int64_t M, int64_t K, int a_dtype) { return M <= kFewRows && K >= 8 && a_dtype != kE4M3; }

}  // namespace

int64_t linear8_workspace_bytes(int64_t M, int64_t K, int a_dtype) {
  if (a_dtype == kE4M3 || quantised_inside(M, K, a_dtype)) return 0;
  const int64_t kp = (K + 127) & ~int64_t(127), s = (K + 511) / 512 * 4;
  return M * (kp + s);
}

hipError_t run_linear8(const Linear8Args& c, int64_t workspace_bytes, hipStream_t stream) {
  const int64_t kp = (c.K + 127) & ~int64_t(127), s = (c.K + 511) / 512 * 4;
  // Offsets inside a tile's rows are 32 bits wide.
  if (c.M <= 0 || c.N <= 0 || c.N > 0x7fffff0 || kp > 0x7fffff || c.M > 0x7fffffff) return hipErrorInvalidValue;
  Args a{c.a, c.a_scale, c.w, c.w_scale, c.bias, c.resid, c.row_mask, c.c, c.M, (int)c.N, (int)c.K, (int)kp, (int)s,
         c.resid_dtype, c.c_dtype, c.epi};
  const bool codes = c.a_dtype == kE4M3;
  if (quantised_inside(c.M, c.K, c.a_dtype)) {
    if (c.K % 8)
      return c.a_dtype == kF16 ? dispatch_few<f16, true>(a, stream) : dispatch_few<bf16, true>(a, stream);
    return c.a_dtype == kF16 ? dispatch_few<f16, false>(a, stream) : dispatch_few<bf16, false>(a, stream);
  }
  if (!codes) {
    if (!c.workspace || workspace_bytes < c.M * (kp + s)) return hipErrorInvalidValue;
    uint8_t* scale = static_cast<uint8_t*>(c.workspace) + c.M * kp;
    const Quantize8Args q{c.a, c.workspace, scale, c.M, c.K, c.a_dtype};
    const hipError_t e = run_quantize8(q, stream);
    if (e != hipSuccess) return e;
    a.a = c.workspace;
    a.a_scale = scale;
  }
  if (c.M <= kFewRows) return dispatch_few<uint8_t, false>(a, stream);
  switch (c.c_dtype) {
    case kF16: return dispatch_tile<f16>(a, stream);
    case kBF16: return dispatch_tile<bf16>(a, stream);
    case kF32: return dispatch_tile<float>(a, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace cobra

// Block tables, slot maps and the write of new keys and values for a cache held in 8 bits.
//
// A layer's cache is a pool of blocks of bs tokens (bs = 16, 32, 64 or 128):
//   k [num_blocks, kv_heads, bs, hdp],  v [num_blocks, kv_heads, hdp, bs]   codes, 1 byte
//   k_scale, v_scale [num_blocks, kv_heads]                                 fp32
// with hdp = cache_width(head_dim) and the columns past head_dim zero.  V is kept with its
// tokens innermost: the attention's P.V product wants consecutive keys of one dimension in a
// lane, and reads them from memory as they lie.  A code c stands for c * scale.  Scales are
// powers of two, so that dividing by one is exact: a code depends on the value and the scale's
// exponent alone, never on how a quotient was rounded, and a block whose scale grows loses
// only the bits that no longer fit (e4m3: none above its subnormals).
#include "common.hpp"
#include "kernels.hpp"

namespace cobra {

namespace {

constexpr int kInLds = 1024;  // requests whose prefix sums the table kernels keep in LDS

__device__ __forceinline__ int64_t wave_incl(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Inclusive prefix sums of two values over the workgroup's NT threads; their totals in sx, sy.
template <int NT>
__device__ __forceinline__ void block_incl(int64_t& x, int64_t& y, int64_t (*red)[2], int64_t* sx, int64_t* sy) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = wave_incl(x, lane);
  y = wave_incl(y, lane);
  __syncthreads();  // red may still be read from the call before
  if (lane == 63) {
    red[wave][0] = x;
    red[wave][1] = y;
  }
  __syncthreads();
  int64_t bx = 0, by = 0, ax = 0, ay = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) {
      bx += red[w][0];
      by += red[w][1];
    }
    ax += red[w][0];
    ay += red[w][1];
  }
  x += bx;
  y += by;
  *sx = ax;
  *sy = ay;
}

__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int shift) {
  return (tokens + (int64_t(1) << shift) - 1) >> shift;
}

// The first i in [0, n) with v[i] > x (v does not decrease, v[n - 1] > x).
__device__ __forceinline__ int first_above(const int32_t* v, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// The slots of tokens first, first + step, .. and the table entries of new blocks first,
// first + step, .. of a reserve whose sums are final: ends[b] = new tokens, incl[b] = new blocks
// of requests 0 .. b, had[b] = tokens of request b before it, count = the free blocks before it.
__device__ __forceinline__ void reserve_fill(const CacheReserveArgs& a, const int32_t* ends, const int32_t* incl,
                                             const int32_t* lens, int count, int64_t first, int64_t step) {
  const int used = ends[a.batch - 1], blocks = incl[a.batch - 1];
#pragma unroll 4
  for (int64_t t = first; t < a.tokens; t += step) {
    int64_t slot = -1;
    if (t < used) {
      const int b = first_above(ends, a.batch, (int)t);
      const int begin = b ? ends[b - 1] : 0, before = b ? incl[b - 1] : 0;
      const int64_t held = (int64_t)lens[b] - (ends[b] - begin);
      const int64_t pos = held + (t - begin), had = blocks_of(held, a.shift), page = pos >> a.shift;
      const int32_t id = page < had ? a.table[b * a.width + page] : a.free_list[count - 1 - (before + (int)(page - had))];
      slot = ((int64_t)id << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    a.slots[t] = slot;
  }
  for (int64_t k = first; k < blocks; k += step) {
    const int b = first_above(incl, a.batch, (int)k);
    const int64_t held = (int64_t)lens[b] - (ends[b] - (b ? ends[b - 1] : 0));
    a.table[b * a.width + blocks_of(held, a.shift) + (k - (b ? incl[b - 1] : 0))] = a.free_list[count - 1 - k];
  }
}

// need_b = ceil((L + n) / bs) - ceil(L / bs) blocks for request b, handed out from the top of
// the stack of free blocks in the order of requests; all requests get theirs or none does.
// One workgroup: the sums are over a few hundred requests, and a barrier is cheaper than a
// second launch.  It also writes slots and table entries where `fill` says so.  Bound by
// latency: 3.7 us for 64 requests of up to 5 tokens, 4.2 for the sums of 200 requests.
template <int NT>
__global__ __launch_bounds__(NT) void cache_reserve_kernel(CacheReserveArgs a, int fill) {
  __shared__ int64_t red[NT / 64][2];
  __shared__ int32_t s_ends[kInLds], s_incl[kInLds], s_lens[kInLds];
  __shared__ int bad;
  const int tid = threadIdx.x;
  const bool near = a.batch <= kInLds;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int count = *a.free_count;
  int64_t toks = 0, need_all = 0;
  for (int b0 = 0; b0 < a.batch; b0 += NT) {
    const int b = b0 + tid;
    int64_t n = 0, need = 0, len = 0;
    if (b < a.batch) {
      len = a.lens[b];
      n = a.new_lens[b];
      if (len < 0 || n < 0 || len + n > 0x7fffffff || blocks_of(len + n, a.shift) > a.width) {
        bad = 1;
        n = 0;
      } else {
        need = blocks_of(len + n, a.shift) - blocks_of(len, a.shift);
      }
    }
    int64_t ts, ns, ti = n, ni = need;
    block_incl<NT>(ti, ni, red, &ts, &ns);
    if (b < a.batch) {
      a.cu[b + 1] = (int32_t)(ti + toks);
      a.incl[b] = (int32_t)(ni + need_all);
      if (near) {
        s_ends[b] = (int32_t)(ti + toks);
        s_incl[b] = (int32_t)(ni + need_all);
        s_lens[b] = (int32_t)(len + n);
      }
    }
    toks += ts;
    need_all += ns;
  }
  __syncthreads();
  int missing = 0;
  if (bad || toks > a.tokens || count < 0 || count > a.num_free)
    missing = -1;
  else if (need_all > count)
    missing = (int)(need_all - count);
  for (int b = tid; b < a.batch; b += NT) {
    if (missing) {
      a.cu[b + 1] = 0;
      a.incl[b] = 0;
      if (near) s_ends[b] = s_incl[b] = 0;
    } else if (near) {
      a.lens[b] = s_lens[b];
    } else {
      a.lens[b] += a.new_lens[b];
    }
  }
  if (tid == 0) {
    a.cu[0] = 0;
    *a.missing = missing;
    a.incl[a.batch] = count;  // for the fill
    if (!missing) *a.free_count = count - (int)need_all;
  }
  if (fill) {
    __syncthreads();
    if (near)
      reserve_fill(a, s_ends, s_incl, s_lens, count, tid, NT);
    else
      reserve_fill(a, a.cu + 1, a.incl, a.lens, count, tid, NT);
  }
}

// The fill over the whole chip, where there are many tokens: a thread for each of 300000 (4.7
// us; 7.5 with four tokens a thread).
__global__ __launch_bounds__(256) void cache_reserve_fill_kernel(CacheReserveArgs a) {
  __shared__ int32_t s_ends[kInLds], s_incl[kInLds], s_lens[kInLds];
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const int count = a.incl[a.batch];
  if (a.batch <= kInLds) {
    for (int b = threadIdx.x; b < a.batch; b += 256) {
      s_ends[b] = a.cu[b + 1];
      s_incl[b] = a.incl[b];
      s_lens[b] = a.lens[b];
    }
    __syncthreads();
    reserve_fill(a, s_ends, s_incl, s_lens, count, first, step);
  } else {
    reserve_fill(a, a.cu + 1, a.incl, a.lens, count, first, step);
  }
}

// The blocks first, first + step, .. that a trim gives back, to their places below `top`.
__device__ __forceinline__ void trim_fill(const CacheTrimArgs& a, const int32_t* incl, int64_t top, int64_t first,
                                          int64_t step) {
  const int all = incl[a.batch - 1];
#pragma unroll 4
  for (int64_t k = first; k < all; k += step) {
    const int b = first_above(incl, a.batch, (int)k);
    const int64_t keep = a.keep_lens[b] < 0 ? 0 : a.keep_lens[b];
    a.free_list[top - 1 - k] = a.table[b * a.width + blocks_of(keep, a.shift) + (k - (b ? incl[b - 1] : 0))];
  }
}

// Requests cut to min(L, max(keep, 0)) tokens; the k-th block given back (requests in order,
// a request's blocks in order) goes k places below the new top of the stack, which undoes a
// reserve exactly.  Bound by latency (64 requests: 2.8 us; 200, with the fill below: 3.2 + 3.6).
template <int NT>
__global__ __launch_bounds__(NT) void cache_trim_kernel(CacheTrimArgs a, int fill) {
  __shared__ int64_t red[NT / 64][2];
  __shared__ int32_t s_incl[kInLds];
  __shared__ int bad;
  const int tid = threadIdx.x;
  const bool near = a.batch <= kInLds;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int count = *a.free_count;
  int64_t all = 0;
  for (int b0 = 0; b0 < a.batch; b0 += NT) {
    const int b = b0 + tid;
    int64_t back = 0, none = 0;
    if (b < a.batch) {
      const int64_t len = a.lens[b];
      const int64_t keep = a.keep_lens[b] < 0 ? 0 : a.keep_lens[b];
      if (len < 0 || blocks_of(len, a.shift) > a.width)
        bad = 1;
      else if (keep < len)
        back = blocks_of(len, a.shift) - blocks_of(keep, a.shift);
    }
    int64_t s, z;
    block_incl<NT>(back, none, red, &s, &z);
    const int64_t i = back + all;
    if (b < a.batch) {
      a.incl[b] = (int32_t)(i > 0x7fffffff ? 0x7fffffff : i);
      if (near) s_incl[b] = (int32_t)(i > 0x7fffffff ? 0x7fffffff : i);
    }
    all += s;
  }
  __syncthreads();
  const bool refused = bad || count < 0 || all + count > a.num_free;
  if (tid == 0) *a.refused = refused ? 1 : 0;
  if (refused) {
    for (int b = tid; b < a.batch; b += NT) a.incl[b] = 0;  // for the fill
    return;
  }
  if (fill) trim_fill(a, near ? s_incl : a.incl, count + all, tid, NT);
  for (int b = tid; b < a.batch; b += NT) {
    const int keep = a.keep_lens[b] < 0 ? 0 : a.keep_lens[b];
    if (keep < a.lens[b]) a.lens[b] = keep;
  }
  if (tid == 0) *a.free_count = count + (int)all;
}

__global__ __launch_bounds__(256) void cache_trim_fill_kernel(CacheTrimArgs a) {
  __shared__ int32_t s_incl[kInLds];
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const int64_t top = *a.free_count;
  if (a.batch <= kInLds) {
    for (int b = threadIdx.x; b < a.batch; b += 256) s_incl[b] = a.incl[b];
    __syncthreads();
    trim_fill(a, s_incl, top, first, step);
  } else {
    trim_fill(a, a.incl, top, first, step);
  }
}

// -- append ---------------------------------------------------------------------------

constexpr int kMaxBlock = 128;
constexpr int kScaleMin = -40, kScaleMax = 40;  // exponents of the scales

// The scale's exponent: the least e in range with amax <= qmax 2^e (the range holds what fp16
// activations can reach with room to spare; beyond it values saturate or round to zero).
template <int CACHE>
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.f)) return kScaleMin;
  // amax = m 2^x with 1 <= m < 2; qmax = 1.75 2^8 (e4m3) or 1.984375 2^6 (int8)
  int x;
  const float m = 2.f * frexpf(amax, &x);
  --x;
  int e = CACHE == kCacheE4M3 ? x - 8 + (m > 1.75f ? 1 : 0) : x - 6 + (m > 1.984375f ? 1 : 0);
  e = e < kScaleMin ? kScaleMin : e;
  return e > kScaleMax ? kScaleMax : e;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Nearest codes (ties to even) of two values, clamped to the code's range; NaN becomes 0 so
// that the cache holds finite values only.
template <int CACHE>
__device__ __forceinline__ uint32_t quant2(float x, float y) {
  constexpr float qmax = CACHE == kCacheE4M3 ? 448.f : 127.f;
  x = x == x ? fminf(fmaxf(x, -qmax), qmax) : 0.f;
  y = y == y ? fminf(fmaxf(y, -qmax), qmax) : 0.f;
  if constexpr (CACHE == kCacheE4M3) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xffffu;
  } else {
    const int i = (int)rintf(x), j = (int)rintf(y);
    return ((uint32_t)i & 0xffu) | (((uint32_t)j & 0xffu) << 8);
  }
}

// quant2 of four values that are finite and inside the code's range.
template <int CACHE>
__device__ __forceinline__ uint32_t quant4(float x, float y, float z, float w) {
  if constexpr (CACHE == kCacheE4M3) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z, w, __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false), true);
  } else {
    // Next to 1.5 x 2^23 a step is 1 and a sum's low byte the rounded integer's.
    constexpr float at = 12582912.f;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y + at), __float_as_uint(x + at), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(w + at), __float_as_uint(z + at), 0x04000c0cu);
    return lo | hi;
  }
}

// What quant2 does with a value before it rounds.
template <int CACHE>
__device__ __forceinline__ float inside(float x) {
  constexpr float qmax = CACHE == kCacheE4M3 ? 448.f : 127.f;
  return x == x ? fminf(fmaxf(x, -qmax), qmax) : 0.f;
}

// Magnitudes of 16-bit floating point numbers are ordered as their bits are; from kNoNumber on
// they are infinities and NaN.
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Magnitude;
template <>
struct Magnitude<f16> {
  static constexpr int kNoNumber = 0x7c00;
};
template <>
struct Magnitude<bf16> {
  static constexpr int kNoNumber = 0x7f80;
};

// The value of code i (0 .. 3) of a word.
template <int CACHE, int I>
__device__ __forceinline__ float code_value(uint32_t w) {
  if constexpr (CACHE == kCacheE4M3)
    return __builtin_amdgcn_cvt_f32_fp8(w, I);
  else
    return (float)(int8_t)(w >> (8 * I));
}

// The codes of a word under a scale grown by 1 / ratio.
template <int CACHE>
__device__ __forceinline__ uint32_t regrade(uint32_t w, float ratio) {
  const uint32_t lo = quant2<CACHE>(code_value<CACHE, 0>(w) * ratio, code_value<CACHE, 1>(w) * ratio);
  const uint32_t hi = quant2<CACHE>(code_value<CACHE, 2>(w) * ratio, code_value<CACHE, 3>(w) * ratio);
  return lo | (hi << 16);
}

__device__ __forceinline__ float finite_abs(float x) {
  const float y = fabsf(x);
  return y < __builtin_huge_valf() ? y : 0.f;  // NaN compares false
}

// Largest value over the workgroup's NT threads.
template <int NT>
__device__ __forceinline__ float group_max(float v, float* red) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  v = fmaxf(v, dpp_f32<0x140>(v));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v = fmaxf(v, red[w]);
    __syncthreads();
  }
  return v;
}

// One workgroup writes what a call brings to the keys (blockIdx.z 0) or values (1) of one
// (block, head).  It belongs to the block's first token in the call (tokens of a block stand
// next to each other in the call).  A workgroup looks for first ones among `window` (<= 63)
// tokens, one a lane.  Where a run writes offset 0 the block starts anew: its scale comes from
// this call's tokens alone.
//
// The values are read twice, for the largest and for the codes; the second time they come from
// the caches (kept in registers in between they cost the occupancy that hides the first: 14000
// tokens of 8 x 128 took twice as long).  K's rows are written eight codes to a store.  V's rows
// run along tokens: a thread takes 4 tokens x 8 dimensions and writes eight words of 4 codes,
// neighbouring lanes neighbouring words of a row.
//
// Bound by latency at one token a request (64 of 8 x 64: 4.8 us).  With whole prompts by the vector
// ALU, active in 62 % of cycles, and by each block's wait for its largest value: 14000 tokens of
// 8 x 128 take 27.3 us, 58 MB read, 29 written, 3.2 TB/s where a large copy makes 5.1 (30.7 us and
// 78 % before magnitudes went two at a time as integers, values unclamped where nothing can need
// it, and codes of four tokens were joined by the conversion itself).
template <typename T, int CACHE, int NT>
__global__ __launch_bounds__(NT) void cache_append_kernel(CacheAppendArgs a, int window, int share) {
  typedef typename Op16<T>::V8 V8;
  __shared__ int src[kMaxBlock];  // token of each offset of the block, -1: none
  __shared__ float red[NT / 64];
  __shared__ int range[2];
  const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.y;
  const bool values = blockIdx.z != 0;
  const int bs = 1 << a.shift, hd = a.head_dim, hdp = a.width, pieces = hd >> 3, wide = hdp >> 3;
  const int64_t slots_end = a.num_blocks << a.shift;
  const int windows = gridDim.x / share;  // ids apart by it share one: neighbours, on different XCDs, all have work
  const int64_t w0 = (int64_t)(blockIdx.x % windows) * window;
  const T* x0 = static_cast<const T*>(a.qkv) + (int64_t)(a.heads + (values ? a.kv_heads : 0) + head) * hd;
  uint8_t* codes = static_cast<uint8_t*>(values ? a.v : a.k);
  float* scales = values ? a.v_scale : a.k_scale;
  // Lane i has the slot of token w0 - 1 + i.
  int64_t slot = -1;
  {
    const int64_t t = w0 - 1 + lane;
    if (t >= 0 && t < a.tokens) slot = a.slots[t];
  }
  const int64_t before = __shfl_up(slot, 1);
  uint64_t firsts = __ballot(lane >= 1 && lane <= window && slot >= 0 && slot < slots_end &&
                             (before < 0 || (before >> a.shift) != (slot >> a.shift)));
  for (int turn = blockIdx.x / windows; firsts; firsts &= firsts - 1) {
    if (turn-- > 0) continue;
    turn = share - 1;
    const int f = __builtin_ctzll(firsts);
    const int64_t t0 = w0 - 1 + f, blk = __shfl(slot, f) >> a.shift;
    const int64_t bh = blk * a.kv_heads + head;
    const float had = fminf(fmaxf(scales[bh], pow2(kScaleMin)), pow2(kScaleMax));
    // The run of tokens that go to this block; of two for one slot the later one stays.
    __syncthreads();
    for (int o = tid; o < bs; o += NT) src[o] = -1;
    __syncthreads();
    if (tid < 64) {
      int lo = bs, hi = -1;
      for (int64_t c = t0;; c += 64) {
        const int64_t t = c + lane;
        const int64_t s = t < a.tokens ? a.slots[t] : -1;
        const uint64_t other = __ballot(s < 0 || (s >> a.shift) != blk);
        if (lane < (other ? __builtin_ctzll(other) : 64)) {
          const int off = (int)(s & (bs - 1));
          atomicMax(&src[off], (int)t);
          lo = min(lo, off);
          hi = max(hi, off);
        }
        if (other) break;
      }
#pragma unroll
      for (int x = 32; x; x >>= 1) {
        lo = min(lo, __shfl_xor(lo, x));
        hi = max(hi, __shfl_xor(hi, x));
      }
      if (lane == 0) {
        range[0] = lo;
        range[1] = hi;
      }
    }
    __syncthreads();
    const int lo = range[0], hi = range[1];
    // Item i: piece p of offset `off` (keys), or piece p of quad q's four offsets (values).
    const int q0 = lo >> 2, quads = (hi >> 2) + 1 - q0;
    const int items = values ? quads * pieces : (hi + 1 - lo) * pieces;
    // Where there is no token the lowest offset's is read (not the run's first, which a later one
    // for its slot may have replaced): loads without a branch between them are in flight together.
    const int some = src[lo];
    auto read = [&](int token, int p) {
      return *reinterpret_cast<const V8*>(x0 + (token < 0 ? some : token) * a.ld + 8 * p);
    };
    // For the largest the order does not matter: keys and values alike in rows, and magnitudes two
    // at a time as integers.  Where one is no number the finite ones' largest is looked for anew.
    const int all = (hi + 1 - lo) * pieces;
    u16x2 top = {0, 0};
#pragma unroll 4
    for (int i = tid; i < all; i += NT) {
      const int r = i / pieces;
      struct {
        u16x2 w[4];
      } x = __builtin_bit_cast(decltype(x), read(src[lo + r], i - r * pieces));
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, x.w[e] & (uint16_t)0x7fff);
    }
    const int bits = (int)group_max<NT>((float)(top[0] > top[1] ? top[0] : top[1]), red);
    const bool numbers = bits < Magnitude<T>::kNoNumber;
    float amax = (float)__builtin_bit_cast(T, (uint16_t)bits);
    if (!numbers) {
      amax = 0.f;
      for (int i = tid; i < all; i += NT) {
        const int r = i / pieces;
        const V8 x = read(src[lo + r], i - r * pieces);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, finite_abs((float)x[e]));
      }
      amax = group_max<NT>(amax, red);
    }
    float scale = pow2(scale_exponent<CACHE>(amax)), ratio = 1.f;
    bool grow = false;
    if (lo > 0) {
      grow = scale > had;
      ratio = grow ? had / scale : 1.f;
      scale = fmaxf(scale, had);
    }
    if (tid == 0) scales[bh] = scale;  // every thread has read the old one: there was a barrier since
    const float inv = 1.f / scale;
    // Nothing to clamp: every value is a number, and within the scale's range (all but bf16's largest).
    const bool plain = numbers && amax <= (CACHE == kCacheE4M3 ? 448.f : 127.f) * scale;
    auto scaled = [&](float (&f)[8], const V8& x) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)x[e] * inv;
      if (!plain) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = inside<CACHE>(f[e]);
      }
    };
    uint8_t* to = codes + bh * bs * hdp;
    if (!values) {
      auto put = [&](int off, int p, const V8& x) {
        float f[8];
        scaled(f, x);
        uint2 w;
        w.x = quant4<CACHE>(f[0], f[1], f[2], f[3]);
        w.y = quant4<CACHE>(f[4], f[5], f[6], f[7]);
        *reinterpret_cast<uint2*>(to + off * hdp + 8 * p) = w;
      };
#pragma unroll 4
      for (int i = tid; i < items; i += NT) {
        const int r = i / pieces, p = i - r * pieces;
        const V8 x = read(src[lo + r], p);
        if (src[lo + r] >= 0) put(lo + r, p, x);
      }
      const int tail = wide - pieces;  // zeros up to the row's width
      if (tail > 0)
        for (int i = tid; i < (hi + 1 - lo) * tail; i += NT) {
          const int r = i / tail, p = pieces + (i - r * tail);
          if (src[lo + r] >= 0) *reinterpret_cast<uint2*>(to + (lo + r) * hdp + 8 * p) = uint2{0u, 0u};
        }
      if (grow)  // tokens of a run may leave offsets out: they are not the call's
        for (int i = tid; i < lo * wide; i += NT) {
          uint2* w = reinterpret_cast<uint2*>(to + (int64_t)i * 8);
          uint2 c = *w;
          c.x = regrade<CACHE>(c.x, ratio);
          c.y = regrade<CACHE>(c.y, ratio);
          *w = c;
        }
    } else {
      // Eight rows' words of quad q: new codes where there are tokens, old ones rounded again
      // below lo, others left.
      auto put = [&](int q, int p, const V8 (&x)[4]) {
        uint32_t w[8], mask = 0, old = 0;
        float f[4][8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          scaled(f[j], x[j]);
          if (src[4 * q + j] >= 0)
            mask |= 0xffu << (8 * j);
          else if (grow && 4 * q + j < lo)
            old |= 0xffu << (8 * j);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = quant4<CACHE>(f[0][e], f[1][e], f[2][e], f[3][e]);
        uint8_t* at = to + (int64_t)p * 8 * bs + 4 * q;
        if (mask == 0xffffffffu) {
#pragma unroll
          for (int e = 0; e < 8; ++e) *reinterpret_cast<uint32_t*>(at + e * bs) = w[e];
        } else if (old) {
          uint32_t was[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) was[e] = *reinterpret_cast<const uint32_t*>(at + e * bs);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<uint32_t*>(at + e * bs) =
                (w[e] & mask) | (regrade<CACHE>(was[e], ratio) & old) | (was[e] & ~(mask | old));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (mask >> (8 * j) & 1u) {
#pragma unroll
              for (int e = 0; e < 8; ++e) at[e * bs + j] = (uint8_t)(w[e] >> (8 * j));
            }
        }
      };
      V8 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = zero8_of<T>();
#pragma unroll 2
      for (int i = tid; i < items; i += NT) {
        const int p = i / quads, q = q0 + (i - p * quads);
        V8 y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[j] = read(src[4 * q + j], p);
        }
        put(q, p, y);
      }
      const int tail = wide - pieces;
      for (int i = tid; i < quads * tail; i += NT) {
        const int p = i / quads;
        put(q0 + (i - p * quads), pieces + p, x);
      }
      if (grow)  // the quads below the first one written
        for (int i = tid; i < q0 * wide; i += NT) {
          const int p = i / q0;
          put(i - p * q0, p, x);
        }
    }
  }
}

template <typename T, int CACHE>
hipError_t launch_append(const CacheAppendArgs& a, hipStream_t stream) {
  // Few tokens: a workgroup for each (64 requests of one token, 8 x 64: 6 to 8 us, in windows of 63
  // 75; 1024 of them 22 and 84).  Many: they are taken for prompts, whose blocks begin every bs
  // tokens (8 prompts of 1500 to 2048 tokens, 8 x 64: 18 us in windows, 74 with a workgroup for each
  // token).  So many requests of one token each are not: 2048 of 8 x 64 take 89 us, a workgroup for each
  // token would take 39; of 5 tokens each 53 and 63.
  // One and a half times as many workgroups for a window as it has blocks, as some end inside one:
  // 7 prompts of up to 700 tokens, 8 x 64, take 7.7, 7.9 and 9.8 us in blocks of 16, 32 and 64, with one
  // workgroup for a window 17.6, 13.0 and 12.7; the 8 prompts of 8 x 128 28.5, 25.7 and 28.5 for 27.9,
  // 29.0 and 33.1.  (A block of 128 has one both ways.)
  const bool few = a.tokens * a.kv_heads <= 8192;
  const int window = few ? 1 : 63, share = few ? 1 : (96 + (1 << a.shift) - 1) >> a.shift;
  // A wave for up to 8192 values, the 8 prompts' blocks of 64 x 128: 28.5 us, 31.8 with four waves (7
  // prompts of up to 700 tokens 13.7 and 10.1); of 16 x 128 28.5 and 63, of 128 x 64 21.1 and 21.3.
  const bool wave = few || (a.head_dim << a.shift) <= 8192;
  const int64_t groups = (a.tokens + window - 1) / window * share;
  if (groups * (wave ? 64 : 256) > 0xffffffff) return hipErrorInvalidValue;  // threads are counted in 32 bits
  const dim3 grid((unsigned)groups, (unsigned)a.kv_heads, 2);
  return wave ? launch_status(cache_append_kernel<T, CACHE, 64>, grid, dim3(64), stream, a, window, share)
              : launch_status(cache_append_kernel<T, CACHE, 256>, grid, dim3(256), stream, a, window, share);
}

}  // namespace

int cache_width(int64_t head_dim) {
  if (head_dim <= 0 || head_dim > 256 || head_dim % 8) return -1;
  for (int w : {32, 64, 96, 128, 192, 256})
    if (head_dim <= w) return w;
  return -1;
}

int cache_shift(int64_t block) {
  return block == 16 ? 4 : block == 32 ? 5 : block == 64 ? 6 : block == 128 ? 7 : -1;
}

hipError_t run_cache_reserve(const CacheReserveArgs& a, hipStream_t stream) {
  if (a.batch <= 0 || a.width < 0 || a.tokens < 0 || a.tokens > 0x7fffffff || a.num_free < 0) return hipErrorInvalidValue;
  // One workgroup fills 1024 slots at a time; past a few rounds of it a second launch over
  // the whole chip is faster.
  const bool one = a.tokens <= 8192;
  const hipError_t e =
      a.batch <= 256 && a.tokens <= 1024
          ? launch_status(cache_reserve_kernel<256>, dim3(1), dim3(256), stream, a, 1)
          : launch_status(cache_reserve_kernel<1024>, dim3(1), dim3(1024), stream, a, one ? 1 : 0);
  if (one || e != hipSuccess) return e;
  const int64_t g = (a.tokens + 255) / 256;  // up to 2048, a full chip of them
  return launch_status(cache_reserve_fill_kernel, dim3((unsigned)(g < 2048 ? g : 2048)), dim3(256), stream, a);
}

hipError_t run_cache_trim(const CacheTrimArgs& a, hipStream_t stream) {
  if (a.batch <= 0 || a.width < 0 || a.num_free < 0) return hipErrorInvalidValue;
  // How many blocks come back is not known here, only that it is at most the table's size.
  const bool one = a.batch * a.width <= 16384;
  const hipError_t e = a.batch <= 256 && one
                           ? launch_status(cache_trim_kernel<256>, dim3(1), dim3(256), stream, a, 1)
                           : launch_status(cache_trim_kernel<1024>, dim3(1), dim3(1024), stream, a, one ? 1 : 0);
  if (one || e != hipSuccess) return e;
  return launch_status(cache_trim_fill_kernel, dim3(64), dim3(256), stream, a);
}

hipError_t run_cache_append(const CacheAppendArgs& a, hipStream_t stream) {
  if (a.tokens <= 0 || a.tokens > 0x7fffffff || a.kv_heads > 65535) return hipErrorInvalidValue;
  if (a.dtype == kF16)
    return a.cache == kCacheE4M3 ? launch_append<f16, kCacheE4M3>(a, stream) : launch_append<f16, kCacheI8>(a, stream);
  return a.cache == kCacheE4M3 ? launch_append<bf16, kCacheE4M3>(a, stream) : launch_append<bf16, kCacheI8>(a, stream);
}

}  // namespace cobra

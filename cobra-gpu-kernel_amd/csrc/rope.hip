// Norms of queries and keys for each head and their rotation by position, in one pass over packed
// q | k | v rows, in place; and the positions of new tokens of cached requests.
//
// A head's vector x of D: y = x / sqrt(sum x^2 / D + eps) * w (fp32; without weights y = x), then of its
// first R columns each pair turns by the token's position times the pair's frequency f_i:
//   (y_a, y_b) -> (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = p f_i,
// pairs (i, i + R / 2) or (2 i, 2 i + 1), i < R / 2.  The angle is formed in turns and in 64 bits and
// brought to half a turn before it is rounded to 32: in 32 bits a position of 100000 would be off by
// 0.006 already.  One rounding, of the result.
//
// Bound by memory for many tokens (every query and key read and written once), by the launch for few.
// A token's R / 2 sines and cosines are formed once, in LDS, for all of its heads.  A lane has two
// pieces of V columns, chosen so that a pair's partners are both its own: V columns from i and V from
// i + R / 2, or two neighbouring pieces.  Heads that 2 columns do not divide (the whole, its pitch or
// half of what turns) have a wave each and their partners from memory.
#include "common.hpp"
#include "kernels.hpp"
#include "lds_dma.hpp"

namespace cobra {

namespace {

constexpr int kMaxDim = 256;
constexpr int kTurns = 512, kSome = 8;  // angles and tokens of a workgroup, at most

struct Args {
  void* qkv;
  const int32_t* positions;
  const float *inv_freq, *q_weight, *k_weight;
  int64_t tokens, ld, seq_len;
  int heads, all;       // query heads; query and key heads
  int dim, pitch, half; // columns of a head, from a head to the next, and half of those that turn
  int lanes;            // of a head
  float eps;
};

// V consecutive values as loaded.
template <typename T, int V>
struct __attribute__((aligned(V * 2))) Piece {
  T e[V];
};

// Sum over a head's lanes: aligned groups of `lanes`, a power of two up to 64, all of them active.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  if (lanes >= 2) v += dpp_f32<0xB1>(v);
  if (lanes >= 4) v += dpp_f32<0x4E>(v);
  if (lanes >= 8) v += dpp_f32<0x141>(v);
  if (lanes >= 16) v += dpp_f32<0x140>(v);
  if (lanes >= 32) v = sum_xor16(v);
  if (lanes >= 64) v = sum_xor32(v);
  return v;
}

__device__ __forceinline__ int position_of(const Args& a, int64_t t) {
  return a.positions ? a.positions[t] : a.seq_len ? (int)(t % a.seq_len) : 0;
}
// (cos, sin) of a position times frequency i.
__device__ __forceinline__ float2 turn_of(const Args& a, int pos, int i) {
  const double x = (double)pos * ((double)a.inv_freq[i] * 0.15915494309189535);  // 1 / 2 pi
  float s, c;
  sincospif(2.f * (float)(x - __builtin_rint(x)), &s, &c);
  return make_float2(c, s);
}
__device__ __forceinline__ void rotate(float& u, float& v, const float2& r) {
  const float x = u;
  u = x * r.x - v * r.y;
  v = v * r.x + x * r.y;
}
__device__ __forceinline__ float norm_of(const Args& a, float sum) { return 1.0f / sqrtf(sum / (float)a.dim + a.eps); }

// A workgroup has `some` tokens; a thread every 256th piece pair of their heads, always the same place
// in the head, so that it holds that place's weights.  U pairs' loads are asked for before the turns are
// formed, and always the next U before the last ones are finished.  16384 tokens of 32 + 8 heads of 128
// (335 MB): 80 to 90 us from memory, 3.7 to 4.2 TB/s against a large copy's 5.1; with a token a workgroup 162
// (its angles and barriers), with two 117, four 90, eight 85; without the loads ahead 98 where this takes 90;
// four pairs at a time no faster (registers for three waves of a SIMD either way); stores past the
// caches 97 to 101.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(Args a, int some) {
  constexpr int U = 2;
  __shared__ float2 turn[kTurns];
  __shared__ int place[kSome];
  const int tid = threadIdx.x;
  const int p = tid & (a.lanes - 1), per = 256 / a.lanes;
  const bool pair = !INTER && p * V < a.half;  // this lane's pieces are partners
  const int c0 = pair ? p * V : 2 * p * V, c1 = pair ? a.half + p * V : c0 + V;
  const bool on0 = c0 < a.dim, on1 = c1 < a.dim;
  const int64_t t0 = (int64_t)blockIdx.x * some;
  const int count = (int)min((int64_t)some, a.tokens - t0);
  const uint32_t work = (uint32_t)count * a.all;  // heads of these tokens
  T* base = static_cast<T*>(a.qkv) + t0 * a.ld;
  Piece<T, V> b0[U][2], b1[U][2];
  auto ask = [&](Piece<T, V> (&x)[U][2], uint32_t first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t w = first + u * per;
      x[u][0] = x[u][1] = Piece<T, V>{};
      if (w < work) {
        const uint32_t t = w / a.all;
        const T* at = base + t * a.ld + (int64_t)(w - t * a.all) * a.pitch;
        if (on0) x[u][0] = *reinterpret_cast<const Piece<T, V>*>(at + c0);
        if (on1) x[u][1] = *reinterpret_cast<const Piece<T, V>*>(at + c1);
      }
    }
  };
  const uint32_t mine = tid / a.lanes;
  // The positions first: loads come back in order, and the angles need nothing else.
  const int at = tid < count ? position_of(a, t0 + tid) : 0;
  ask(b0, mine);
  if (tid < count) place[tid] = at;
  float wq[2][V], wk[2][V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    wq[0][e] = a.q_weight && on0 ? a.q_weight[c0 + e] : 1.f;
    wq[1][e] = a.q_weight && on1 ? a.q_weight[c1 + e] : 1.f;
    wk[0][e] = a.q_weight && on0 ? a.k_weight[c0 + e] : 1.f;
    wk[1][e] = a.q_weight && on1 ? a.k_weight[c1 + e] : 1.f;
  }
  lds_barrier();
  for (int i = tid; i < count * a.half; i += 256) {
    const int t = i / a.half, k = i - t * a.half;
    turn[i] = turn_of(a, place[t], k);
  }
  lds_barrier();
  auto finish = [&](const Piece<T, V> (&x)[U][2], uint32_t first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t w = first + u * per;
      if (w >= work) break;
      const uint32_t t = w / a.all, h = w - t * a.all;
      float y0[V], y1[V], ss = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        y0[e] = (float)x[u][0].e[e];
        y1[e] = (float)x[u][1].e[e];
        ss = fmaf(y0[e], y0[e], fmaf(y1[e], y1[e], ss));
      }
      if (a.q_weight) {
        const float inv = norm_of(a, lanes_sum(ss, a.lanes));
        const bool query = h < (uint32_t)a.heads;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y0[e] *= inv * (query ? wq[0][e] : wk[0][e]);
          y1[e] *= inv * (query ? wq[1][e] : wk[1][e]);
        }
      }
      const float2* r = turn + t * a.half;
      if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          if (c0 + e < 2 * a.half) rotate(y0[e], y0[e + 1], r[(c0 + e) >> 1]);
          if (c1 + e < 2 * a.half) rotate(y1[e], y1[e + 1], r[(c1 + e) >> 1]);
        }
      } else if (pair) {
#pragma unroll
        for (int e = 0; e < V; ++e) rotate(y0[e], y1[e], r[c0 + e]);
      }
      if (place[t] < 0) continue;
      Piece<T, V> z0, z1;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        z0.e[e] = (T)y0[e];
        z1.e[e] = (T)y1[e];
      }
      T* at = base + t * a.ld + (int64_t)h * a.pitch;
      if (on0) *reinterpret_cast<Piece<T, V>*>(at + c0) = z0;
      if (on1) *reinterpret_cast<Piece<T, V>*>(at + c1) = z1;
    }
  };
  for (uint32_t first = mine; first < work; first += 2 * U * per) {
    ask(b1, first + U * per);
    finish(b0, first);
    ask(b0, first + 2 * U * per);
    finish(b1, first + U * per);
  }
}

// Any geometry: a wave has a head, a lane its columns lane, lane + 64, ..; all of a head's loads come
// before its stores.
template <typename T>
__global__ __launch_bounds__(256) void qk_norm_rope_any_kernel(Args a, int inter) {
  constexpr int kPer = kMaxDim / 64;
  __shared__ float2 turn[kMaxDim / 2];
  const int lane = threadIdx.x & 63;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int pos = position_of(a, t);
    if (pos < 0) continue;
    __syncthreads();
    for (int i = threadIdx.x; i < a.half; i += 256) turn[i] = turn_of(a, pos, i);
    __syncthreads();
    T* row = static_cast<T*>(a.qkv) + t * a.ld;
    for (int h = threadIdx.x >> 6; h < a.all; h += 4) {
      T* x = row + (int64_t)h * a.pitch;
      float y[kPer], z[kPer], ss = 0.f;  // a column and its partner
      int at[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = lane + 64 * e;
        at[e] = i >= 2 * a.half ? i : inter ? i ^ 1 : i < a.half ? i + a.half : i - a.half;
        y[e] = i < a.dim ? (float)x[i] : 0.f;
        z[e] = i < a.dim ? (float)x[at[e]] : 0.f;
        ss = fmaf(y[e], y[e], ss);
      }
      const float* w = h < a.heads ? a.q_weight : a.k_weight;
      if (w) {
        const float inv = norm_of(a, group_sum<64>(ss));
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (lane + 64 * e < a.dim) {
            y[e] *= inv * w[lane + 64 * e];
            z[e] *= inv * w[at[e]];
          }
      }
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        const int i = lane + 64 * e;
        if (i < 2 * a.half) {
          const float2 r = turn[inter ? i >> 1 : i < a.half ? i : i - a.half];
          y[e] = y[e] * r.x + (at[e] > i ? -z[e] : z[e]) * r.y;
        }
        if (i < a.dim) x[i] = (T)y[e];
      }
    }
  }
}

template <typename T>
hipError_t any(const Args& a, int inter, hipStream_t stream) {
  const dim3 groups((unsigned)(a.tokens < (1 << 20) ? a.tokens : 1 << 20));
  return launch_status(qk_norm_rope_any_kernel<T>, groups, dim3(256), stream, a, inter);
}

template <typename T, int V, bool INTER>
hipError_t launch(Args a, hipStream_t stream) {
  a.lanes = 1;
  while (a.lanes * 2 * V < a.dim) a.lanes *= 2;
  // As many tokens a workgroup as its threads have ten pairs and two angles each for, fewer where
  // every CU would not have eight workgroups then.
  const int64_t pairs = 10 * 256 / ((int64_t)a.all * a.lanes), angles = a.half ? kTurns / a.half : kSome;
  const int64_t each = a.tokens / (8 * compute_units());
  int64_t some = pairs < angles ? pairs : angles;
  some = some < each ? some : each;
  some = some > kSome ? kSome : some < 1 ? 1 : some;
  const int64_t groups = (a.tokens + some - 1) / some;
  if (groups > 0xffffff) return any<T>(a, INTER, stream);  // (a launch's workgroups; that kernel goes round)
  return launch_status(qk_norm_rope_kernel<T, V, INTER>, dim3((unsigned)groups), dim3(256), stream, a, (int)some);
}

template <typename T>
hipError_t launch_type(const Args& a, int inter, hipStream_t stream) {
  const auto fits = [&](int v) {
    return a.dim % v == 0 && a.pitch % v == 0 && a.ld % v == 0 && (inter || a.half % v == 0) &&
           (reinterpret_cast<uintptr_t>(a.qkv) & (2 * v - 1)) == 0;
  };
  // (In pieces of 2 columns 30 million values of 6 + 6 heads of 40, halves of 10 turned, take 45 us, of
  // 5 + 5 of 168, halves of 42, 41; one by one 135 and 80.)
  if (fits(8)) return inter ? launch<T, 8, true>(a, stream) : launch<T, 8, false>(a, stream);
  if (fits(4)) return inter ? launch<T, 4, true>(a, stream) : launch<T, 4, false>(a, stream);
  if (fits(2)) return inter ? launch<T, 2, true>(a, stream) : launch<T, 2, false>(a, stream);
  return any<T>(a, inter, stream);
}

// Position of each new token: its request's tokens before it, behind those of the prefix; -1 where
// no request has it.  The requests' bounds are searched in LDS where they fit: a search in memory is
// a chain of dependent reads.
constexpr int kBounds = 4096;
template <bool SHARED>
__global__ __launch_bounds__(256) void cache_positions_kernel(const int32_t* __restrict__ cu,
                                                              const int32_t* __restrict__ lens, int32_t* __restrict__ out,
                                                              int64_t tokens, int batch, int prefix) {
  __shared__ int32_t held[SHARED ? kBounds : 1];
  if constexpr (SHARED) {
    for (int i = threadIdx.x; i <= batch; i += 256) held[i] = cu[i];
    __syncthreads();
  }
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= tokens) return;
  auto bound = [&](int i) { return SHARED ? held[i] : cu[i]; };
  int lo = 0, hi = batch;  // the last request with cu[b] <= t is in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (bound(mid) <= t) lo = mid;
    else hi = mid;
  }
  const int64_t first = bound(lo), end = bound(lo + 1);
  int64_t at = -1;
  if (first >= 0 && t >= first && t < end) {
    at = (int64_t)lens[lo] - (end - t);
    if (prefix >= 0 && lo != prefix) at += lens[prefix] > 0 ? lens[prefix] : 0;
    at = at < -1 ? -1 : at > 0x7fffffff ? 0x7fffffff : at;
  }
  out[t] = (int32_t)at;
}

}  // namespace

hipError_t run_qk_norm_rope(const QkNormRopeArgs& c, hipStream_t stream) {
  if (c.head_dim <= 0 || c.head_dim > kMaxDim || c.rot < 0 || c.rot % 2 || c.rot > c.head_dim) return hipErrorInvalidValue;
  const Args a{c.qkv, c.positions, c.inv_freq, c.q_weight, c.k_weight, c.tokens, c.ld, c.seq_len, c.heads, c.heads + c.kv_heads,
               c.head_dim, c.pitch, c.rot / 2, 0, c.eps};
  return c.dtype == kF16 ? launch_type<f16>(a, c.interleaved, stream) : launch_type<bf16>(a, c.interleaved, stream);
}

hipError_t run_cache_positions(const int32_t* cu, const int32_t* lens, int32_t* out, int64_t tokens, int batch,
                               int prefix, hipStream_t stream) {
  const dim3 groups((unsigned)((tokens + 255) / 256));
  return batch < kBounds
             ? launch_status(cache_positions_kernel<true>, groups, dim3(256), stream, cu, lens, out, tokens, batch, prefix)
             : launch_status(cache_positions_kernel<false>, groups, dim3(256), stream, cu, lens, out, tokens, batch, prefix);
}

}  // namespace cobra

// Attention of new tokens over a cache whose requests share a prefix (layout: cache.hip, passes over
// keys: cache_attn.hpp).
//
// Row `prefix` of the tables is a request like any other; a new token of request b sees all of its
// keys and then b's own up to itself (or all of b's), in one softmax:
//   o = (sum_P w v + sum_own w v) / (sum_P w + sum_own w).
// With a table of each request that lists the shared blocks too, the prefix would be read and widened
// once for every request.  Here the rows of all requests pass over it together, as if they were one
// request's: few rows of each become many, which share tiles in LDS.  Both passes are one launch,
// each leaves partial results (O, M, l), and a second launch joins a row's.  The prefix's own new tokens see only itself.
#include "cache_attn.hpp"

namespace cobra {

namespace {

// Both passes by direct loads.
template <typename T, int CACHE, int HDP>
__global__ __launch_bounds__(256) void cache_prefix_decode_kernel(Args own, PrePass pre) {
  if ((int)blockIdx.x < pre.groups)
    decode_rows<kPrefix, T, CACHE, HDP, decode_keys(HDP)>(pre.args, blockIdx.x);
  else
    decode_rows<kOwn, T, CACHE, HDP, decode_keys(HDP)>(own, blockIdx.x - pre.groups);
}

// The request that token t belongs to: the last with cu[b] <= t.
__device__ __forceinline__ int request_at(const Args& a, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (int b0 = 0; b0 < a.batch && a.batch > 1; b0 += 64) {
    const int below = __popcll(__ballot(b0 + lane < a.batch && a.cu[min(b0 + lane, a.batch)] <= t));
    if (below) lo = b0 + below - 1;
    if (below < 64) break;
  }
  return lo;
}

// A row's shares joined, the prefix's splits and then its request's own, always in the same order:
// o = sum 2^(M_s - M) O_s / sum 2^(M_s - M) l_s.  W waves have a row; for the statistics a lane has every
// 64th split, for O a wave takes as many splits at a time as it has lanes for.
//
// Bound by latency, so what does not depend on the request is asked for first: the statistics of
// every split that there may be, and the first kEarly rounds of O.
constexpr int kMaxSplits = 256, kOwnSplits = 64;
template <typename T, int HDP, int W>
__global__ __launch_bounds__(256) void cache_prefix_join_kernel(Args a, PrePass shared, int pre_step, int own_step) {
  constexpr int kLanes = HDP / 4, kAt = 64 / kLanes;  // lanes of a split, splits of a wave
  constexpr int kEarly = W > 1 ? 4 : 8, kStats = W > 1 ? kMaxSplits / 64 : 1;
  __shared__ float factor[4][64 * kStats];
  __shared__ f32x4 sh[W > 1 ? W : 1][kLanes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = W > 1 ? wave : 0;
  const int all = shared.args.splits + a.splits;
  const int sub = lane / kLanes, d = (lane - sub * kLanes) * 4, s0 = part * kAt + sub;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  for (int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave; row < rows;
       row += (int64_t)gridDim.x * (W > 1 ? 1 : 4)) {
    float2 ml[kStats];
#pragma unroll
    for (int k = 0; k < kStats; ++k) {
      ml[k] = make_float2(kNegInf, 0.f);
      if (lane + 64 * k < all) ml[k] = a.part_m[(lane + 64 * k) * rows + row];
    }
    f32x4 early[kEarly];
#pragma unroll
    for (int i = 0; i < kEarly; ++i) {
      const int s = s0 + i * W * kAt;
      if (sub < kAt && s < all) early[i] = *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * HDP + d);
    }
    const int t = (int)(row / a.heads), b = request_at(a, t);
    const Request rq = request_of<kOwn>(a, b), pre = request_of<kPrefix>(a, a.prefix);
    if (t < max(rq.t0, pre.t0) || t >= min(rq.t0 + rq.n, pre.t0 + pre.n)) continue;  // (offsets that fall: no shares)
    const int pre_chunk = chunk_of(shared.args, pre.len, pre_step), own_chunk = chunk_of(a, rq.len, own_step);
    const int pre_n = b == a.prefix ? 0 : (int)(((int64_t)pre.len + pre_chunk - 1) / pre_chunk);
    const int own_n = (int)(((int64_t)rq.len + own_chunk - 1) / own_chunk);
    // Splits that were written: the first pre_n, and own_n from a.base on.
    auto there = [&](int s) { return s < a.base ? s < pre_n : s - a.base < own_n; };
    float m = kNegInf;
#pragma unroll
    for (int k = 0; k < kStats; ++k) {
      if (!there(lane + 64 * k)) ml[k] = make_float2(kNegInf, 0.f);
      m = fmaxf(m, ml[k].x);
    }
#pragma unroll
    for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    float l = 0.f;
#pragma unroll
    for (int k = 0; k < kStats; ++k) {
      const float f = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - m);
      factor[wave][lane + 64 * k] = f;
      l += f * ml[k].y;
    }
    l = group_sum<64>(l);
    __builtin_amdgcn_wave_barrier();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    auto take = [&](int s, const f32x4& x) {
      if (sub < kAt && s < all && there(s)) {
        const float w = factor[wave][s];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(w, x[i], o[i]);
      }
    };
#pragma unroll
    for (int i = 0; i < kEarly; ++i) take(s0 + i * W * kAt, early[i]);
    for (int s = s0 + kEarly * W * kAt; s - sub < all; s += W * kAt) {
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
      if (sub < kAt && s < all) x = *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * HDP + d);
      take(s, x);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kAt; ++k) v += __shfl(o[i], lane % kLanes + k * kLanes);
      o[i] = v;
    }
    if constexpr (W > 1) {
      if (lane < kLanes) sh[part][lane] = o;
      __syncthreads();
      if (part) continue;  // (a workgroup has one row)
#pragma unroll
      for (int w = 1; w < W; ++w)
        if (lane < kLanes) o += sh[w][lane];
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (lane < kLanes && d < a.head_dim) {
      typename Op16<T>::V4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
      *reinterpret_cast<typename Op16<T>::V4*>(static_cast<T*>(a.out) + row * a.head_dim + d) = y;
    }
  }
}

// The same for few splits: a row has as many lanes as its dimensions in fours, which take
// the splits one after the other, so that a wave has 64 / lanes rows and does the divisions and the search
// for the request once for all of them.  Bound by instructions with a row a wave: 44800 rows of 64, 4 splits,
// 15 us in place of 50.  With up to kMoreShares only where a wave has two rows: 8192 of 64 with 9 shares 87 us in
// all in place of 92, 4096 of 128 with 13 8.5 in place of 9.4, but 276 of 256 with 9 6.6 in place of 5.6.
constexpr int kFewShares = 8, kMoreShares = 16;
template <typename T, int HDP, int S>
__global__ __launch_bounds__(256) void cache_prefix_join_rows_kernel(Args a, PrePass shared, int pre_step, int own_step) {
  constexpr int kLanes = HDP / 4, kRows = 64 / kLanes;
  const int lane = threadIdx.x & 63, sub = lane / kLanes, d = (lane - sub * kLanes) * 4;
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rows = (uint32_t)(a.tokens * a.heads), row = wave * kRows + sub;  // (less than 2^31)
  const bool active = sub < kRows && row < rows;
  const int all = shared.args.splits + a.splits;
  float2 ml[S];
  f32x4 x[S];
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < all && active) {
      ml[s] = a.part_m[(int64_t)s * rows + row];
      x[s] = *reinterpret_cast<const f32x4*>(a.part_o + ((int64_t)s * rows + row) * HDP + d);
    }
  const int t = active ? (int)(row / (uint32_t)a.heads) : 0;
  int before = 0;  // requests that begin at t or before it
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int first = b0 + lane < a.batch ? a.cu[b0 + lane] : 0x7fffffff;
    int most = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int n = __popcll(__ballot(first <= __builtin_amdgcn_readlane(t, i * kLanes)));
      if (sub == i) before += n;
      most = max(most, n);
    }
    if (most < 64) break;
  }
  const int b = before > 0 ? before - 1 : 0;
  const Request rq = request_of<kOwn>(a, b), pre = request_of<kPrefix>(a, a.prefix);
  if (!active || t < max(rq.t0, pre.t0) || t >= min(rq.t0 + rq.n, pre.t0 + pre.n)) return;
  const uint32_t pre_chunk = chunk_of(shared.args, pre.len, pre_step), own_chunk = chunk_of(a, rq.len, own_step);
  const int pre_n = b == a.prefix ? 0 : (int)(((uint32_t)pre.len + pre_chunk - 1) / pre_chunk);
  const int own_n = (int)(((uint32_t)rq.len + own_chunk - 1) / own_chunk);
  float m = kNegInf;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool there = s < all && (s < a.base ? s < pre_n : s - a.base < own_n);
    if (!there) {
      ml[s] = make_float2(kNegInf, 0.f);
      x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    m = fmaxf(m, ml[s].x);
  }
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const float w = m == kNegInf ? 0.f : __builtin_amdgcn_exp2f(ml[s].x - m);
    l = fmaf(w, ml[s].y, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(w, x[s][i], o[i]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  if (d < a.head_dim) {
    typename Op16<T>::V4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
    *reinterpret_cast<typename Op16<T>::V4*>(static_cast<T*>(a.out) + (int64_t)row * a.head_dim + d) = y;
  }
}

struct PrefixPlan {
  CachePlan pre, own;
  bool both;  // one pass over the prefix and the request's own keys
};

// More units of rows than CUs take whole rounds, so 1 to 4 splits by cost: a CU's n workgroups pass two at a
// time (up to head_dim 128), one alone in 0.7 of that, over their share of the tiles and two tiles' time to
// start; splits are written and joined, one and a half tiles' time for each 256 units and 64 columns, and as
// much for the pass of its own that each request's keys are then.  Times with 1 to 4 splits:
//   388 units behind 9000 (4 prompts of 300 to 1000 tokens, 16 heads of 64 on 4, fp16)   317 295 266 272
//   680 (8 of them) 566 435 433 446; 388 behind 2000 110 114 117 123
//   324 behind 16000 (16 of 64 to 256 tokens, bf16)                                       408 371 294 320
//   384 behind 12000, 632 behind 8000, 1216 (32 heads of 128 on 8)    453 406 421 411, 548 452 460 471, 809 821 848
//   284 behind 6000 (8 heads of 256 on 2)                                                 495 432 413 431
// (5 to 7 splits gain nothing in any of them.)
int64_t splits_of_many(int64_t units, int64_t keys, int width, bool joined) {
  const int64_t cus = compute_units();
  const double tiles = keys / 64.0, join = 1.5 * (double)units / cus * (width / 64.0);
  int64_t best = 1;
  double best_t = 1e300;
  for (int64_t s = 1; s <= 4; ++s) {
    const int64_t n = (units * s + cus - 1) / cus;
    const double rounds = width > 128 ? (double)n : (double)(n / 2) + 0.7 * (double)(n % 2);
    const double t = rounds * (tiles / (double)s + 2.0) + (s > 1 || joined ? join * (double)(1 + s) : 0.0);
    if (t < best_t) {
      best_t = t;
      best = s;
    }
  }
  return best;
}

// How the prefix's pass is cut: as a call of one request with all of the tokens, but for the splits and
// the kernel.
// Rows pass over the keys by direct loads, in tiles of 16, while that is little work in all (rows x keys x
// head_dim of all kv heads): tiles of 128 take long to start and leave the chip empty.  23 drafts
// of 2 to 6 tokens behind 4001 keys, 6 heads of 256 on 2: 29 us against 39; 64 requests behind 4000, 32
// heads of 128 on 8, 30 and 36, 128 so 47 and 48 (2^31), 64 behind 16000 61 and 57, 128 behind 30000 205 and
// 137; 1024 behind 4000, 8 heads of 64, 92 and 118.  A workgroup a CU then: with two 30, 33, 51, 65, 222
// and 92; two where the splits are of hardly any rows (one request behind 99999, 16 heads of 64 on 2: 16.8 us
// against 19.4).
// In tiles of 128 rows as many splits as give three quarters of the chip's places (two workgroups a CU up
// to head_dim 128) a workgroup, so that the requests' own keys, which are bound by memory, have the rest
// from the start: 128 requests of up to 2000 keys behind 30000, 32 heads of 128 on 8, take 135 to 147 us with
// 384 workgroups, 166 and 152 with 256 and 480; alone the passes take 88 (with 512) and 63.  (Own ones evenly
// between the prefix's: 182 us; behind them in all of these.)  With 256, 320, 384, 448 and 512 (half as many at 256):
//   64 requests of up to 2000 behind 60000, 32 heads of 128 on 8   161 151 135 123 136
//   128 of up to 4000 behind 16000, 32 of 128 on 8                 141 153 165 177 189
//   128 of up to 500 behind 30000, 16 of 64 on 4                    65  68  61  55  53
//   128 of up to 2000 behind 30000, 8 of 128 on 1                   52  55  52  52  54
//   60 of 4 new tokens, up to 2000 behind 30000, 8 of 128 on 2      76  79  71  65  67
//   100 of up to 300 behind 20000, 6 of 256 on 2, int8              80  72  67  69  71
CachePlan pre_plan(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_prefix,
                   const CachePlan& own) {
  CachePlan p = cache_plan(tokens, 1, heads, kv_heads, head_dim, tokens, max_prefix);
  const int width = cache_width(head_dim);
  max_prefix = max_prefix < 1 ? 1 : max_prefix > kMaxKeys ? kMaxKeys : max_prefix;
  const int64_t rows = tokens * (heads / kv_heads);
  if (p.chunked && !own.chunked && rows * kv_heads * width <= ((int64_t)1 << 31) / max_prefix) {
    p.chunked = false;
    p.row_tiles = (rows + 15) / 16;
    p.step = 4 * decode_keys(width);
  }
  const int64_t units = (p.chunked ? (rows + 127) / 128 : p.row_tiles) * kv_heads;
  const int64_t least = p.chunked ? 128 : p.step, room = kMaxParts / (tokens * heads);
  const int64_t target = !p.chunked ? (units <= 4 ? 512 : 256) : width <= 128 ? 384 : 192;
  int64_t splits = p.chunked ? (target + units / 2) / units : (target + units - 1) / units;
  if (p.chunked && units > compute_units())
    splits = splits_of_many(units, max_prefix, width, !own.chunked || own.splits > 1);
  const int64_t most = (max_prefix + least - 1) / least;
  splits = splits < most ? splits : most;
  splits = splits < room ? splits : room;
  splits = splits < kMaxSplits - kOwnSplits ? splits : kMaxSplits - kOwnSplits;
  splits = splits < 1 ? 1 : splits;
  const int64_t even = (max_prefix + splits - 1) / splits;
  p.chunk = (int)((even + p.step - 1) / p.step * p.step);
  p.splits = (int)((max_prefix + p.chunk - 1) / p.chunk);
  return p;
}

// .. and the requests' own keys, in at most kOwnSplits.
CachePlan own_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
                   int64_t max_len) {
  CachePlan p = cache_plan(tokens, batch, heads, kv_heads, head_dim, max_new, max_len);
  if (p.splits > kOwnSplits) {
    const int64_t even = ((max_len > kMaxKeys ? kMaxKeys : max_len) + kOwnSplits - 1) / kOwnSplits;
    p.chunk = (int)((even + p.step - 1) / p.step * p.step);
    p.splits = kOwnSplits;
  }
  return p;
}

PrefixPlan plan_of(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
                   int64_t max_len, int64_t max_prefix) {
  PrefixPlan p;
  p.own = own_plan(tokens, batch, heads, kv_heads, head_dim, max_new, max_len);
  p.pre = pre_plan(tokens, heads, kv_heads, head_dim, max_prefix, p.own);
  // (4 prompts of 300 to 1000 tokens behind 2000, 16 heads of 64 on 4: 110 us in one pass, 114 joined.)
  p.both = p.own.chunked && p.pre.splits == 1 && p.own.splits == 1;
  // (Either pass goes round the row tiles that a launch has no workgroups for.)
  const int64_t tiles = kMaxGrid / (kv_heads * p.pre.splits);
  if (p.pre.row_tiles > tiles) p.pre.row_tiles = tiles > 1 ? tiles : 1;
  return p;
}

template <typename T, int CACHE, int HDP>
hipError_t launch(const Args& a, PrePass shared, const PrefixPlan& p, hipStream_t stream) {
  const dim3 block(256);
  const int64_t own = (int64_t)a.batch * a.kv_heads * p.own.row_tiles * p.own.splits;
  const int64_t pre = (int64_t)a.kv_heads * p.pre.row_tiles * p.pre.splits;
  if (p.both)
    return own > kMaxGrid ? hipErrorInvalidValue
                          : launch_status(cache_chunk_kernel<kBoth, T, CACHE, HDP, 2>, dim3((unsigned)own), block, stream, a, NoPass{});
  if (own > kMaxGrid || pre > kMaxGrid) return hipErrorInvalidValue;
  // Requests of many new tokens are many tokens together.
  auto* kernel = p.own.chunked   ? cache_chunk_kernel<kPrefix, T, CACHE, HDP, 2, true, PrePass>
                 : p.pre.chunked ? cache_chunk_kernel<kPrefix, T, CACHE, HDP, 2, false, PrePass>
                                 : cache_prefix_decode_kernel<T, CACHE, HDP>;
  // Both passes together, or one after the other where they are more workgroups than a launch has.
  const bool together = own + pre <= kMaxGrid;
  shared.groups = (int)pre;
  hipError_t e = launch_status(kernel, dim3((unsigned)(together ? own + pre : pre)), block, stream, a, shared);
  if (e != hipSuccess) return e;
  if (!together) {
    shared.groups = 0;
    e = launch_status(kernel, dim3((unsigned)own), block, stream, a, shared);
    if (e != hipSuccess) return e;
  }
  const int64_t rows = (int64_t)a.tokens * a.heads;
  if (p.pre.splits + p.own.splits > 64)
    return launch_status(cache_prefix_join_kernel<T, HDP, 4>, dim3((unsigned)rows), block, stream, a, shared,
                         p.pre.step, p.own.step);
  constexpr int kRows = 4 * (64 / (HDP / 4));  // of a workgroup, with few shares
  const int shares = p.pre.splits + p.own.splits;
  constexpr int kMost = HDP <= 128 ? kMoreShares : kFewShares;
  if (shares <= kMost && (rows + kRows - 1) / kRows <= kMaxGrid)
    return launch_status(shares <= kFewShares ? cache_prefix_join_rows_kernel<T, HDP, kFewShares>
                                              : cache_prefix_join_rows_kernel<T, HDP, kMost>,
                         dim3((unsigned)((rows + kRows - 1) / kRows)), block, stream, a, shared, p.pre.step, p.own.step);
  const int64_t quads = (rows + 3) / 4;
  return launch_status(cache_prefix_join_kernel<T, HDP, 1>, dim3((unsigned)(quads < kMaxGrid ? quads : kMaxGrid)),
                       block, stream, a, shared, p.pre.step, p.own.step);
}

template <typename T, int CACHE>
hipError_t launch_width(const Args& a, const PrePass& shared, const PrefixPlan& p, int width, hipStream_t stream) {
  switch (width) {
    case 32: return launch<T, CACHE, 32>(a, shared, p, stream);
    case 64: return launch<T, CACHE, 64>(a, shared, p, stream);
    case 96: return launch<T, CACHE, 96>(a, shared, p, stream);
    case 128: return launch<T, CACHE, 128>(a, shared, p, stream);
    case 192: return launch<T, CACHE, 192>(a, shared, p, stream);
    case 256: return launch<T, CACHE, 256>(a, shared, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t cache_prefix_workspace_bytes(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                     int64_t max_new, int64_t max_len, int64_t max_prefix) {
  const PrefixPlan p = plan_of(tokens, batch, heads, kv_heads, head_dim, max_new, max_len, max_prefix);
  if (p.both) return 0;
  return (int64_t)(p.pre.splits + p.own.splits) * tokens * heads * (cache_width(head_dim) * 4 + 8);
}

hipError_t run_cache_prefix(const CachePrefixArgs& c, int64_t workspace_bytes, hipStream_t stream) {
  const CacheAttnArgs& t = c.attn;
  const int width = cache_width(t.head_dim);
  if (!cache_call_ok(t) || c.prefix < 0 || c.prefix >= t.batch) return hipErrorInvalidValue;
  const PrefixPlan p =
      plan_of(t.tokens, t.batch, t.heads, t.kv_heads, t.head_dim, t.max_new, t.max_len, c.max_prefix);
  const int64_t rows = t.tokens * t.heads, parts = (p.pre.splits + p.own.splits) * rows;
  if (!p.both && (!t.part || workspace_bytes < parts * (width * 4 + 8))) return hipErrorInvalidValue;
  Args a = cache_args(t, p.own);
  if (!p.both) {
    a.part_o = t.part;
    a.part_m = reinterpret_cast<float2*>(t.part + parts * width);
  }
  a.prefix = c.prefix;
  a.base = p.pre.splits;
  PrePass shared{a, 0};
  shared.args.causal = 0;
  shared.args.splits = p.pre.splits;
  shared.args.chunk = p.pre.chunk;
  shared.args.row_tiles = (int)p.pre.row_tiles;
  if (t.dtype == kF16)
    return t.cache == kCacheE4M3 ? launch_width<f16, kCacheE4M3>(a, shared, p, width, stream)
                                 : launch_width<f16, kCacheI8>(a, shared, p, width, stream);
  return t.cache == kCacheE4M3 ? launch_width<bf16, kCacheE4M3>(a, shared, p, width, stream)
                               : launch_width<bf16, kCacheI8>(a, shared, p, width, stream);
}

}  // namespace cobra

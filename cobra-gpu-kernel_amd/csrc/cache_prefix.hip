// Attention of new tokens over a cache whose requests share a prefix (layout: cache.hip, passes over
// keys: cache_attn.hpp).
//
// Row `prefix` of the tables is a request like any other; a new token of request b sees all of its
// keys and then b's own up to itself (or all of b's), in one softmax:
//   o = (sum_P w v + sum_own w v) / (sum_P w + sum_own w).
// With a table of each request that lists the shared blocks too, the prefix would be read and widened
// once for every request.  Here the rows of all requests pass over it together, as if they were one
// request's: few rows of each become many, which share tiles in LDS.  Both passes are one launch,
// the prefix's workgroups first, each leaves partial results (O, M, l), and a second launch joins a
// row's.  The prefix's own new tokens see only itself.
#include "cache_attn.hpp"

namespace cobra {

namespace {

// Both passes of a call: the prefix's workgroups, then the requests' own.
struct Both {
  Args pre, own;
  int groups;  // workgroups of the prefix's pass
};

template <typename T, int CACHE, int HDP, bool PRE_CHUNK, bool OWN_CHUNK>
__global__ __launch_bounds__(256, (PRE_CHUNK || OWN_CHUNK) && HDP <= 128 ? 2 : 1) void cache_prefix_kernel(Both c) {
  constexpr bool kChunk = PRE_CHUNK || OWN_CHUNK;
  constexpr int kBytes = kChunk && sizeof(ChunkShared<HDP>) > sizeof(DecodeShared<HDP>) ? (int)sizeof(ChunkShared<HDP>)
                                                                                        : (int)sizeof(DecodeShared<HDP>);
  __shared__ __attribute__((aligned(16))) char smem[kBytes];
  const int id = blockIdx.x;
  if (id < c.groups) {
    if constexpr (PRE_CHUNK)
      chunk_rows<kPrefix, T, CACHE, HDP, 2>(c.pre, id, *reinterpret_cast<ChunkShared<HDP>*>(smem));
    else
      decode_rows<kPrefix, T, CACHE, HDP, decode_keys(HDP)>(c.pre, id, *reinterpret_cast<DecodeShared<HDP>*>(smem));
  } else {
    if constexpr (OWN_CHUNK)
      chunk_rows<kOwn, T, CACHE, HDP, 2>(c.own, id - c.groups, *reinterpret_cast<ChunkShared<HDP>*>(smem));
    else
      decode_rows<kOwn, T, CACHE, HDP, decode_keys(HDP)>(c.own, id - c.groups,
                                                         *reinterpret_cast<DecodeShared<HDP>*>(smem));
  }
}

// A row's shares joined, the prefix's splits and then its request's own, always in the same order:
// o = sum 2^(M_s - M) O_s / sum 2^(M_s - M) l_s.  W waves have a row; a wave takes as many splits at a
// time as it has lanes for.
template <typename T, int HDP, int W>
__global__ __launch_bounds__(256) void cache_prefix_join_kernel(Both c, int pre_step, int own_step) {
  constexpr int kLanes = HDP / 4, kAt = 64 / kLanes;  // lanes of a split, splits of a wave
  __shared__ f32x4 sh[W > 1 ? W : 1][kLanes];
  const Args& a = c.own;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = W > 1 ? wave : 0;
  const int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  if (row >= rows) return;
  const int t = (int)(row / a.heads);
  int lo = 0;  // the last request with cu[b] <= t
  for (int b0 = 0; b0 < a.batch && a.batch > 1; b0 += 64) {
    const int below = __popcll(__ballot(b0 + lane < a.batch && a.cu[min(b0 + lane, a.batch)] <= t));
    if (below) lo = b0 + below - 1;
    if (below < 64) break;
  }
  const Request rq = request_of<kOwn>(a, lo), pre = request_of<kPrefix>(c.pre, a.prefix);
  if (t < rq.t0 || t >= rq.t0 + rq.n) return;
  const int pre_chunk = chunk_of(c.pre, pre.len, pre_step), own_chunk = chunk_of(a, rq.len, own_step);
  const int pre_n = lo == a.prefix ? 0 : (int)(((int64_t)pre.len + pre_chunk - 1) / pre_chunk);
  const int n = pre_n + (int)(((int64_t)rq.len + own_chunk - 1) / own_chunk);
  // Where a row's share s lies.
  auto at = [&](int s) { return (int64_t)(s < pre_n ? s : a.base + s - pre_n) * rows + row; };
  float m = kNegInf;
  for (int s = lane; s < n; s += 64) m = fmaxf(m, a.part_m[at(s)].x);
#pragma unroll
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float base = m == kNegInf ? 0.f : m;
  float l = 0.f;
  for (int s = lane; s < n; s += 64) {
    const float2 ml = a.part_m[at(s)];
    l += __builtin_amdgcn_exp2f(ml.x - base) * ml.y;
  }
  l = group_sum<64>(l);
  const int sub = lane / kLanes, d = (lane - sub * kLanes) * 4;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (sub < kAt) {
#pragma unroll 4
    for (int s = part * kAt + sub; s < n; s += W * kAt) {
      const float f = __builtin_amdgcn_exp2f(a.part_m[at(s)].x - base);
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + at(s) * HDP + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(f, x[i], o[i]);
    }
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
    if (part) return;
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

struct PrefixPlan {
  CachePlan pre, own;
};

PrefixPlan plan_of(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
                   int64_t max_len, int64_t max_prefix) {
  PrefixPlan p;
  // The prefix's pass is a call of one request with all of the tokens.
  p.pre = cache_plan(tokens, 1, heads, kv_heads, head_dim, tokens, max_prefix);
  p.own = cache_plan(tokens, batch, heads, kv_heads, head_dim, max_new, max_len);
  return p;
}

template <typename T, int CACHE, int HDP>
hipError_t launch(const Both& c, const PrefixPlan& p, hipStream_t stream) {
  const int64_t own = (int64_t)c.own.batch * c.own.kv_heads * p.own.row_tiles * p.own.splits;
  const int64_t pre = (int64_t)c.own.kv_heads * p.pre.row_tiles * p.pre.splits;
  if (own + pre > kMaxGrid) return hipErrorInvalidValue;
  Both b = c;
  b.groups = (int)pre;
  const dim3 groups((unsigned)(own + pre)), block(256);
  // Requests of many new tokens are many tokens together.
  auto* kernel = p.own.chunked   ? cache_prefix_kernel<T, CACHE, HDP, true, true>
                 : p.pre.chunked ? cache_prefix_kernel<T, CACHE, HDP, true, false>
                                 : cache_prefix_kernel<T, CACHE, HDP, false, false>;
  const hipError_t e = launch_status(kernel, groups, block, stream, b);
  if (e != hipSuccess) return e;
  const int64_t rows = (int64_t)c.own.tokens * c.own.heads;
  return p.pre.splits + p.own.splits > 16
             ? launch_status(cache_prefix_join_kernel<T, HDP, 4>, dim3((unsigned)rows), block, stream, b, p.pre.step,
                             p.own.step)
             : launch_status(cache_prefix_join_kernel<T, HDP, 1>, dim3((unsigned)((rows + 3) / 4)), block, stream, b,
                             p.pre.step, p.own.step);
}

template <typename T, int CACHE>
hipError_t launch_width(const Both& c, const PrefixPlan& p, int width, hipStream_t stream) {
  switch (width) {
    case 32: return launch<T, CACHE, 32>(c, p, stream);
    case 64: return launch<T, CACHE, 64>(c, p, stream);
    case 96: return launch<T, CACHE, 96>(c, p, stream);
    case 128: return launch<T, CACHE, 128>(c, p, stream);
    case 192: return launch<T, CACHE, 192>(c, p, stream);
    case 256: return launch<T, CACHE, 256>(c, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t cache_prefix_workspace_bytes(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                     int64_t max_new, int64_t max_len, int64_t max_prefix) {
  const PrefixPlan p = plan_of(tokens, batch, heads, kv_heads, head_dim, max_new, max_len, max_prefix);
  return (int64_t)(p.pre.splits + p.own.splits) * tokens * heads * (cache_width(head_dim) * 4 + 8);
}

hipError_t run_cache_prefix(const CachePrefixArgs& c, int64_t workspace_bytes, hipStream_t stream) {
  const CacheAttnArgs& t = c.attn;
  const int width = cache_width(t.head_dim);
  if (!cache_call_ok(t) || c.prefix < 0 || c.prefix >= t.batch) return hipErrorInvalidValue;
  const PrefixPlan p =
      plan_of(t.tokens, t.batch, t.heads, t.kv_heads, t.head_dim, t.max_new, t.max_len, c.max_prefix);
  const int64_t rows = t.tokens * t.heads, parts = (p.pre.splits + p.own.splits) * rows;
  if (!t.part || workspace_bytes < parts * (width * 4 + 8)) return hipErrorInvalidValue;
  Both b{};
  b.own = cache_args(t, p.own);
  b.own.part_o = t.part;
  b.own.part_m = reinterpret_cast<float2*>(t.part + parts * width);
  b.own.prefix = c.prefix;
  b.own.base = p.pre.splits;
  b.pre = b.own;
  b.pre.causal = 0;
  b.pre.splits = p.pre.splits;
  b.pre.chunk = p.pre.chunk;
  b.pre.row_tiles = (int)p.pre.row_tiles;
  if (t.dtype == kF16)
    return t.cache == kCacheE4M3 ? launch_width<f16, kCacheE4M3>(b, p, width, stream)
                                 : launch_width<f16, kCacheI8>(b, p, width, stream);
  return t.cache == kCacheE4M3 ? launch_width<bf16, kCacheE4M3>(b, p, width, stream)
                               : launch_width<bf16, kCacheI8>(b, p, width, stream);
}

}  // namespace cobra

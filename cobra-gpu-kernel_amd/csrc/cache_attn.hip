// Attention of new tokens over a key/value cache held in 8 bits: how a call is cut, and its
// launches (kernels: cache_attn.hpp).
#include "cache_attn.hpp"

namespace cobra {

// How a call is cut.  max_new and max_len are expectations; a call that exceeds them is still
// covered (rows in a loop, longer splits).
CachePlan cache_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
             int64_t max_len) {
  CachePlan p{};
  max_new = max_new < 1 ? 1 : max_new > tokens ? tokens : max_new;
  max_len = max_len < 1 ? 1 : max_len > kMaxKeys ? kMaxKeys : max_len;
  const int64_t group = heads / kv_heads, rows = max_new * group;
  // Past 64 rows a workgroup's keys are worth sharing among four waves' rows: 64 requests of 1000 keys,
  // 32 heads of 128 on 8, take 46 us in tiles of 16 and 64 so at 32 rows, 84 and 68 at 64, 163 and 77
  // at 128; 16 requests of 4000 keys, 6 of 256 on 2, 73 and 57 at 96.  (Requests that leave the chip
  // empty would do with tiles of 16 for longer: one of 4000 keys, 32 of 128 on 8, 18 and 42 us at 128.)
  p.chunked = rows > 64;
  p.row_tiles = p.chunked ? (rows + 127) / 128 : (rows + 15) / 16;
  p.step = p.chunked ? 64 : 4 * decode_keys(cache_width(head_dim));
  // Units of work before the keys are split, and splits up to 512 of them, two for each CU:
  // 64 requests of up to 2048 keys and 8 heads took 16.9 us so and 24.7 in 1024.  A row tile
  // of the chunk kernel is long enough to split its keys only where the chip would be empty.
  const int64_t units = p.chunked ? (tokens * group + 127) / 128 * kv_heads : batch * kv_heads * p.row_tiles;
  const int64_t least = p.chunked ? 1024 : p.step;
  int64_t splits = (512 + units - 1) / units;
  if (p.chunked && units >= 256) splits = 1;
  // Hints that fit leave under 2^17 partial rows (twice 512 units of 16, or 256 of 128 three times).
  // Where max_new is too low for the tokens it is the workspace that has to be bounded.
  const int64_t room = kMaxParts / (tokens * heads);
  splits = splits < room ? splits : room;
  // Every request has its workgroups, those without new tokens too.
  const int64_t places = kMaxGrid / (batch * kv_heads);
  splits = splits < places ? splits : places;
  // Up to 1024 keys one workgroup takes less time than the second launch that joins splits: at 1000
  // 6.6 us against 8.0 for one request of 4 x 32, 10.6 against 14.5 for 64 of 16 x 64 on 4, 12.3 against
  // 15.3 for 16 of 8 x 128 (one of these 10.7 against 10.0), at 300 5.3 to 8.4 against 7.7 to 11.1.
  if (!p.chunked && max_len <= 1024 && cache_width(head_dim) <= 128) splits = 1;
  const int64_t most = (max_len + least - 1) / least;
  splits = splits < most ? splits : most;
  splits = splits < 1 ? 1 : splits;
  const int64_t even = (max_len + splits - 1) / splits;
  p.chunk = (int)((even + p.step - 1) / p.step * p.step);
  p.splits = (int)((max_len + p.chunk - 1) / p.chunk);
  // Workgroups go round the row tiles of their request where these are fewer than it has.
  const int64_t tiles = kMaxGrid / (batch * kv_heads * p.splits);
  if (p.row_tiles > tiles) p.row_tiles = tiles > 1 ? tiles : 1;
  return p;
}

bool cache_call_ok(const CacheAttnArgs& c) {
  return cache_width(c.head_dim) > 0 && c.tokens > 0 && c.tokens <= 0x7fffffff && c.batch > 0 && c.table_width > 0 &&
         c.tokens * c.heads <= 0x7fffff00;  // rows of a kv head are counted in 32 bits
}

namespace {

template <typename T, int CACHE, int HDP>
hipError_t launch(const Args& a, const CachePlan& p, hipStream_t stream) {
  const int64_t grid = (int64_t)a.batch * a.kv_heads * p.row_tiles * p.splits;
  if (grid > kMaxGrid) return hipErrorInvalidValue;
  const dim3 groups((unsigned)grid), block(256);
  const hipError_t e =
      p.chunked ? launch_status(cache_chunk_kernel<kWhole, T, CACHE, HDP, 2>, groups, block, stream, a, NoPass{})
                : launch_status(cache_decode_kernel<T, CACHE, HDP, decode_keys(HDP)>, groups, block, stream, a);
  if (p.splits <= 1 || e != hipSuccess) return e;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  return p.splits > 16 ? launch_status(cache_join_kernel<T, HDP, 4>, dim3((unsigned)rows), block, stream, a, p.step)
                       : launch_status(cache_join_kernel<T, HDP, 1>, dim3((unsigned)((rows + 3) / 4)), block, stream, a,
                                       p.step);
}

template <typename T, int CACHE>
hipError_t launch_width(const Args& a, const CachePlan& p, int width, hipStream_t stream) {
  switch (width) {
    case 32: return launch<T, CACHE, 32>(a, p, stream);
    case 64: return launch<T, CACHE, 64>(a, p, stream);
    case 96: return launch<T, CACHE, 96>(a, p, stream);
    case 128: return launch<T, CACHE, 128>(a, p, stream);
    case 192: return launch<T, CACHE, 192>(a, p, stream);
    case 256: return launch<T, CACHE, 256>(a, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

int64_t cache_attn_workspace_bytes(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t max_new, int64_t max_len) {
  const CachePlan p = cache_plan(tokens, batch, heads, kv_heads, head_dim, max_new, max_len);
  if (p.splits <= 1) return 0;
  return (int64_t)p.splits * tokens * heads * (cache_width(head_dim) * 4 + 8);
}

hipError_t run_cache_attn(const CacheAttnArgs& c, int64_t workspace_bytes, hipStream_t stream) {
  const int width = cache_width(c.head_dim);
  if (!cache_call_ok(c)) return hipErrorInvalidValue;
  const CachePlan p = cache_plan(c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, c.max_new, c.max_len);
  Args a = cache_args(c, p);
  if (p.splits > 1) {
    const int64_t rows = (int64_t)p.splits * c.tokens * c.heads;
    if (!c.part || workspace_bytes < rows * (width * 4 + 8)) return hipErrorInvalidValue;
    a.part_o = c.part;
    a.part_m = reinterpret_cast<float2*>(c.part + rows * width);
  }
  if (c.dtype == kF16)
    return c.cache == kCacheE4M3 ? launch_width<f16, kCacheE4M3>(a, p, width, stream)
                                 : launch_width<f16, kCacheI8>(a, p, width, stream);
  return c.cache == kCacheE4M3 ? launch_width<bf16, kCacheE4M3>(a, p, width, stream)
                               : launch_width<bf16, kCacheI8>(a, p, width, stream);
}

}  // namespace cobra

// Attention of new tokens over a key/value cache held in 8 bits (layout: cache.hip).
//
// For new token i of a request with L keys, n of them new, and a query head of kv head h:
//   o_i = sum_j p_ij v_j,  p_i = softmax_j(scale q_i . k_j),  k_j = sk(j) kc_j,  v_j = sv(j) vc_j
// over j <= L - n + i (causal) or j < L, with codes kc, vc and one scale for each block and head.
//
// In one pass over the keys, with running values for each row (log2 units):
//   u_j = (q . kc_j) sk(j) scale log2(e) + log2 sv(j),   w_j = 2^(u_j - M + 8)
//   O = sum w_j vc_j,   l = sum w_j / sv(j),   o = O / l
// so that V's scales ride in the exponent the softmax computes anyway, and the P.V product
// runs on plain codes.  M is a maximum of u that moves only when a tile has a w near fp16's
// largest number: most tiles need no maximum, no exchange between lanes and no rescaling of O.
// w is rounded to fp16 for the product (11 bits; 2^-22 of the reference's before subnormals)
// whatever the activations' type: codes are exact in fp16.  With fp16 activations the product
// takes what was rounded off as a second term.
// Scores, M, l and O are fp32.  Scales are taken within [2^-40, 2^40], so no w that counts
// underflows and neither sum overflows.
//
// Tiles are 64 keys and 16 rows (v_mfma_f32_16x16x32): S^T = K Q^T, then O^T = V^T P^T.  Row r
// of K's subtile s is key 16 (r / 4) + 4 s + r % 4, which leaves the scores of keys
// 16 g .. 16 g + 15 in lane group g = lane / 16, in order: exactly the keys whose codes that
// group reads of V^T in one 16-byte load.  P goes from the softmax into the product without
// leaving its lane, K and V from memory into the matrix cores without passing LDS, and since a
// block is at least 16 tokens a lane needs one K scale and one V scale for a tile.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"
#include "lds_dma.hpp"

namespace cobra {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr float kBias = 8.f;         // log2 of w where u equals its reference
constexpr float kAccept = 57344.f;   // a lane's sum of w that is taken without a maximum
// Keys of a request that are attended to: what is left to 2^31 covers the rounding up of splits
// and the tiles that loads are ahead.
constexpr int64_t kMaxKeys = 0x7ffff000;
// Workgroups of a launch: of 256 threads, which are counted in 32 bits.
constexpr int64_t kMaxGrid = 0xffffff;
// Rows of a head that all splits of a call leave partial results of (541 MB at head_dim 256).
constexpr int64_t kMaxParts = 1 << 19;

__device__ __forceinline__ f32x4 mfma16(const f16x8& a, const f16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes to the operand type, exactly.
template <int CACHE, typename T>
struct Widen;
template <>
struct Widen<kCacheE4M3, f16> {
  static __device__ __forceinline__ f16x8 of(uint32_t x, uint32_t y) {
    struct {
      f16x2 p[4];
    } q;
    q.p[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false);
    q.p[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true);
    q.p[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, false);
    q.p[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, true);
    return __builtin_bit_cast(f16x8, q);
  }
};
template <>
struct Widen<kCacheE4M3, bf16> {
  static __device__ __forceinline__ bf16x8 of(uint32_t x, uint32_t y) {
    struct {
      bf16x2 p[4];
    } q;
    q.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, false);
    q.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, true);
    q.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, false);
    q.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.f, true);
    return __builtin_bit_cast(bf16x8, q);
  }
};
// int8 to fp16: the byte with its sign flipped, u = c + 128, as the low byte of 0x6400 is the
// number 1024 + u, from which 1152 is taken (both exact).  The subtraction is left to the
// compiler, which keeps the two wait states that a matrix instruction needs after a vector
// one has written its operand; it does not for inline asm.
__device__ __forceinline__ f16x2 i8_pair(uint32_t flipped, uint32_t sel) {
  const uint32_t w = __builtin_amdgcn_perm(0x64646464u, flipped, sel);
  const f16x2 off = {(f16)1152.f, (f16)1152.f};
  return __builtin_bit_cast(f16x2, w) - off;
}
template <>
struct Widen<kCacheI8, f16> {
  static __device__ __forceinline__ f16x8 of(uint32_t x, uint32_t y) {
    struct {
      f16x2 p[4];
    } q;
    x ^= 0x80808080u;
    y ^= 0x80808080u;
    q.p[0] = i8_pair(x, 0x04010400u);
    q.p[1] = i8_pair(x, 0x04030402u);
    q.p[2] = i8_pair(y, 0x04010400u);
    q.p[3] = i8_pair(y, 0x04030402u);
    return __builtin_bit_cast(f16x8, q);
  }
};
template <>
struct Widen<kCacheI8, bf16> {
  static __device__ __forceinline__ bf16x8 of(uint32_t x, uint32_t y) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = (bf16)(float)(int8_t)(x >> (8 * i));
      r[4 + i] = (bf16)(float)(int8_t)(y >> (8 * i));
    }
    return r;
  }
};

// The first n codes of v, zeros after them: memory past a request's end, or of a block that is
// none, may hold NaN codes.
template <typename V>
__device__ __forceinline__ void keep_first(V& v, int n) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
    const int c = n - 4 * i;
    v[i] = c >= 4 ? v[i] : c <= 0 ? 0u : v[i] & (0xffffffffu >> (8 * (4 - c)));
  }
}

struct Args {
  const void* q;
  void* out;
  const int32_t *cu, *lens, *table;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  float* part_o;   // [splits][tokens * heads][hdp], O of each split
  float2* part_m;  // [splits][tokens * heads], (M, l)
  int64_t ldq, table_width, num_blocks;
  int tokens, batch, heads, kv_heads, group, head_dim, shift, causal;
  float c2;        // scale * log2(e)
  int splits;      // grid splits of a request's keys
  int chunk;       // keys of a split, at least (a multiple of the workgroup's step)
  int row_tiles;   // grid tiles of a request's rows
};

// A request as the kernels see it, whatever its lengths say: bounds that keep every access
// inside the tensors.
struct Request {
  int t0, n, len;
};
__device__ __forceinline__ Request request_of(const Args& a, int b) {
  Request r;
  r.t0 = a.cu[b];
  const int t1 = a.cu[b + 1];
  r.n = t1 - r.t0;
  if (r.t0 < 0 || t1 > a.tokens || r.n < 0) r.n = 0;
  const int64_t most = min(a.table_width << a.shift, kMaxKeys);
  const int len = a.lens[b];
  r.len = len < 0 ? 0 : len > most ? (int)most : len;
  return r;
}

// Keys of one split of a request: a.chunk, or more where the grid's splits would not cover it.
__device__ __forceinline__ int chunk_of(const Args& a, int len, int step) {
  const int even = (len + a.splits - 1) / a.splits;
  const int up = (even + step - 1) / step * step;
  return up > a.chunk ? up : a.chunk;
}

// Entries of a request's row of the table, 64 from `first` on a lane each, and the next 64.
// Loads of single entries would be waited for one by one: scalar ones share a counter with
// LDS, vector ones theirs with the tiles in flight.  A tile's blocks never straddle two 64s,
// which begin a whole number of tiles apart.
struct Pages {
  int first, held, ahead, last;
  const int32_t* row;
  __device__ __forceinline__ Pages(const Args& a, int b, int p)
      : first(p), last((int)a.table_width - 1), row(a.table + b * a.table_width) {
    held = entry(p);
    ahead = entry(p + 64);
  }
  __device__ __forceinline__ int entry(int p) const {
    p += threadIdx.x & 63;
    return row[(uint32_t)(p < last ? p : last)];
  }
  __device__ __forceinline__ void reach(const Args& a, int p) {
    if (p - first >= 64) {
      first += 64;
      held = ahead;
      ahead = entry(first + 64);
    }
  }
  __device__ __forceinline__ int any(int p) const {  // p may differ from lane to lane
    return __builtin_amdgcn_ds_bpermute((p - first) * 4, held);
  }
  __device__ __forceinline__ int one(int p) const { return __builtin_amdgcn_readlane(held, p - first); }
};

// Where block id of one kv head lies.  A block's bytes over all heads are under 2^31.
struct Strides {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  uint32_t stride, heads, blocks;
  __device__ __forceinline__ Strides(const Args& a, int h, int plane)
      : k(a.k + (int64_t)h * plane),
        v(a.v + (int64_t)h * plane),
        k_scale(a.k_scale + h),
        v_scale(a.v_scale + h),
        stride((uint32_t)a.kv_heads * (uint32_t)plane),
        heads((uint32_t)a.kv_heads),
        blocks((uint32_t)a.num_blocks) {}
  __device__ __forceinline__ bool there(int id) const { return (uint32_t)id < blocks; }
  __device__ __forceinline__ uint64_t block(int id) const { return (uint64_t)(there(id) ? (uint32_t)id : 0u) * stride; }
  __device__ __forceinline__ uint64_t scale(int id) const { return (uint64_t)(there(id) ? (uint32_t)id : 0u) * heads; }
};

// One wave's state for NR sets of 16 rows and its pass over some tiles of keys.
template <typename T, int CACHE, int HDP, int NR, int KT>
struct Rows {
  typedef typename Op16<T>::V8 V8;
  static constexpr int kSteps = HDP / 32, kWide = HDP / 64, kOdd = kSteps & 1, kDims = HDP / 16;
  static constexpr int kSub = KT / 16, kKeys = KT / 4, kWords = KT / 16, kParts = KT / 32;
  typedef uint32_t VWords __attribute__((ext_vector_type(kWords)));
  // A weight's rounding to fp16 is as large as an fp16 result's own: with one term the results were
  // up to 1.7 times their own rounding off (one key's weight often makes up most of a row), in
  // chunks of prompts 1.08 times.  So with fp16 activations the product takes what was rounded off
  // as a second term: half as many matrix instructions again, and for a pair of weights a multiply-
  // add each and a conversion.  64 requests of 8 x 64 take 0.6 us of 16.9 for it, chunks of 16 x 64
  // 159 us in place of 138, of 32 x 128 1200 in place of 944.  Not with bf16, whose results' own
  // rounding is eight times a weight's (0.00156 from 64 bits with one term, as the plain form's).
  static constexpr bool kTwo = std::is_same<T, f16>::value;
  static constexpr int kTerms = kTwo ? 2 * kParts : kParts;

  V8 q[NR][kSteps];
  f32x4 o[NR][kDims];
  float m[NR], l[NR];  // l: this lane group's share
  int lim[NR];         // keys that this lane's row sees

  __device__ __forceinline__ void init(const Args& a, const Request& rq, int h, int row0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = row0 + 16 * r + n;
      const bool there = row < rq.n * a.group;
      const int tok = there ? row / a.group : 0;
      const int head = h * a.group + (there ? row - tok * a.group : 0);
      const T* p = static_cast<const T*>(a.q) + (int64_t)(rq.t0 + tok) * a.ldq + (int64_t)head * a.head_dim;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = s < 2 * kWide ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 64 * kWide + 8 * g;
        q[r][s] = zero8_of<T>();
        if (there && d < a.head_dim) q[r][s] = *reinterpret_cast<const V8*>(p + d);
      }
      const int seen = a.causal ? rq.len - rq.n + tok + 1 : rq.len;
      lim[r] = there ? (seen < 0 ? 0 : seen) : 0;
      m[r] = kNegInf;
      l[r] = 0.f;
#pragma unroll
      for (int t = 0; t < kDims; ++t) o[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // w = 2^(s skc + shift) of a lane's keys, rounded to fp16 in p, and their sum (not rounded: a
  // key whose V scale is far below the row's largest has a w that fp16 has no bits for, and
  // counts in l all the same).  Of two terms the first is rounded towards zero, by an instruction
  // that takes a pair, so that the rest keeps its sign; the rest, under 2^-10 of w, is rounded to
  // the nearest: 2^-21 of w in all.
  static __device__ __forceinline__ float weigh(const f32x4 (&s)[kSub], float skc, float shift, f16x8 (&p)[kTerms]) {
    float sum = 0.f, minus = -1.f;
    asm("" : "+s"(minus));  // kept a factor: x - w as a multiply-add of an fp16 w is one instruction
#pragma unroll
    for (int e = 0; e < kKeys; e += 2) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], skc, shift));
      const float y = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][(e & 3) + 1], skc, shift));
      f16x2 w = {(f16)x, (f16)y};
      if constexpr (kTwo) {
        w = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
        p[kParts + (e >> 3)][e & 7] = (f16)fmaf((float)w[0], minus, x);
        p[kParts + (e >> 3)][(e & 7) + 1] = (f16)fmaf((float)w[1], minus, y);
      }
      p[e >> 3][e & 7] = w[0];
      p[e >> 3][(e & 7) + 1] = w[1];
      sum += x + y;
    }
    return sum;
  }

  // The queries are waited for here, behind the first tile's loads: waited for in the loop, they
  // would take every later tile's along.
  __device__ __forceinline__ void wait_queries() {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) asm volatile("" : "+v"(q[r][i]));
  }

  // S^T = K Q^T on codes; k(i, j): this lane's K operand of subtile i, step j.
  template <typename K>
  __device__ __forceinline__ void scores(f32x4 (&s)[NR][kSub], K&& k) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < kSub; ++i) s[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Steps outside, so that neighbouring instructions add to different registers.
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        const V8 x = k(i, j);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][i] = mfma16(x, q[r][j], s[r][i]);
      }
  }

  // Scores to weights: this lane's keys begin at key0, its block's scales are sk and sv (of a
  // block outside the pool: bad); slow: not every row sees every key of the tile.  First against
  // the reference that the row has, without a maximum of this tile: right as long as every w
  // stays inside fp16, which a sum at most kAccept of a lane's w shows.
  struct Block {
    float skc, ev, inv;
    __device__ __forceinline__ Block(const Args& a, float sk, float sv) {
      const float svc = fminf(fmaxf(sv, 0x1p-40f), 0x1p40f);
      skc = fminf(fmaxf(sk, 0x1p-40f), 0x1p40f) * a.c2;
      ev = __builtin_amdgcn_logf(svc);
      inv = __builtin_amdgcn_rcpf(svc);  // both exact for powers of two
    }
  };
  __device__ __forceinline__ bool weights(const f32x4 (&s)[NR][kSub], f16x8 (&p)[NR][kTerms], const Block& b,
                                          float (&sum)[NR]) const {
    bool ok = true;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      sum[r] = weigh(s[r], b.skc, b.ev + kBias - m[r], p[r]);
      ok &= sum[r] <= kAccept;  // false for NaN, and where the row has no reference yet
    }
    return ok;
  }
  __device__ __forceinline__ void weights_by_max(f32x4 (&s)[NR][kSub], f16x8 (&p)[NR][kTerms], const Block& b,
                                                 float (&sum)[NR], int key0, bool bad, bool slow) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int seen = bad ? 0 : slow ? lim[r] - key0 : kKeys;  // keys of this lane that count
      float mx = kNegInf;
#pragma unroll
      for (int e = 0; e < kKeys; ++e) {
        const float u = fmaf(s[r][e >> 2][e & 3], b.skc, b.ev);
        s[r][e >> 2][e & 3] = e < seen ? s[r][e >> 2][e & 3] : kNegInf;
        mx = fmaxf(mx, e < seen ? u : kNegInf);
      }
      const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = max_xor32(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
      const float mn = fmaxf(m[r], mx);
      const float alpha = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m[r] - mn);
      m[r] = mn;
      sum[r] = weigh(s[r], b.skc, mn == kNegInf ? kNegInf : b.ev + kBias - mn, p[r]);
      l[r] *= alpha;
#pragma unroll
      for (int t = 0; t < kDims; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[r][t][i] *= alpha;
    }
  }
  __device__ __forceinline__ void softmax(f32x4 (&s)[NR][kSub], f16x8 (&p)[NR][kTerms], const Block& b, int key0,
                                          bool bad, bool slow) {
    float sum[NR];
    if (slow || !__all(weights(s, p, b, sum))) weights_by_max(s, p, b, sum, key0, bad, slow);
#pragma unroll
    for (int r = 0; r < NR; ++r) l[r] = fmaf(sum[r], b.inv, l[r]);
  }

  // O^T += V^T P^T on codes; v(t, i): this lane's V operand of dimensions 16 t .., part i of its keys.
  template <typename V>
  __device__ __forceinline__ void gather(const f16x8 (&p)[NR][kTerms], V&& v) {
#pragma unroll
    for (int i = 0; i < kParts; ++i)
#pragma unroll
      for (int t = 0; t < kDims; ++t) {
        const f16x8 x = v(t, i);
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r][t] = mfma16(x, p[r][i], o[r][t]);
        if constexpr (kTwo) {
#pragma unroll
          for (int r = 0; r < NR; ++r) o[r][t] = mfma16(x, p[r][kParts + i], o[r][t]);
        }
      }
  }

  // Tiles t0, t0 + step, .. below t_end, K and V straight from memory to registers; keys from
  // `full` on are checked against each row's limit.
  __device__ __forceinline__ void pass(const Args& a, const Request& rq, int b, int h, int t0, int t_end, int step,
                                       int full) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15, gk = n >> 2;
    const int bs = 1 << a.shift;
    if (t0 >= t_end) return;

    Pages pages(a, b, (t0 * KT) >> a.shift);
    const Strides st(a, h, bs * HDP);
    u32x4 kw[kSub][kWide > 0 ? kWide : 1];
    u32x2 ko[kSub];
    VWords vw[kDims];
    float sk, sv;
    bool bad = false;
    int idk, idv;  // blocks of the group whose K rows this lane reads, and of its own keys
    auto find = [&](int tile) {
      pages.reach(a, (tile * KT) >> a.shift);
      idk = pages.any((tile * KT + kKeys * gk) >> a.shift);
      idv = pages.any((tile * KT + kKeys * g) >> a.shift);
    };
    auto load_k = [&](int tile) {
      const int off = (tile * KT + kKeys * gk + (n & 3)) & (bs - 1);
      const uint8_t* p = st.k + st.block(idk) + (uint32_t)(off * HDP + 16 * g);
#pragma unroll
      for (int s = 0; s < kSub; ++s) {
#pragma unroll
        for (int j = 0; j < kWide; ++j) kw[s][j] = *reinterpret_cast<const u32x4*>(p + s * 4 * HDP + 64 * j);
        if constexpr (kOdd) ko[s] = *reinterpret_cast<const u32x2*>(p + s * 4 * HDP + 64 * kWide - 8 * g);
      }
    };
    auto load_v = [&](int tile) {
      const int off = (tile * KT + kKeys * g) & (bs - 1);
      const uint8_t* p = st.v + st.block(idv) + (uint32_t)(n * bs + off);
      sk = st.k_scale[st.scale(idv)];
      sv = st.v_scale[st.scale(idv)];
      bad = !st.there(idv);
#pragma unroll
      for (int t = 0; t < kDims; ++t) vw[t] = *reinterpret_cast<const VWords*>(p + (uint32_t)(t * 16 * bs));
    };
    find(t0);
    load_k(t0);
    load_v(t0);
    wait_queries();
    // One tile; `more`: with the loads of the wave's next, the keys' while the softmax runs.  Not
    // a test inside: where the paths met, a wait for one tile's loads would be one for the next's.
    auto one = [&](int tile, auto more) {
      const int key0 = tile * KT + kKeys * g;  // this lane's first key
      f32x4 s[NR][kSub];
      scores(s, [&](int i, int j) {
        if (kOdd && j == kSteps - 1) return Widen<CACHE, T>::of(ko[i][0], ko[i][1]);
        return Widen<CACHE, T>::of(kw[i][j >> 1][2 * (j & 1)], kw[i][j >> 1][2 * (j & 1) + 1]);
      });
      const bool slow = tile * KT + KT > full || __any(bad);
      const int there = bad ? 0 : rq.len - key0;
      const bool bad0 = bad;
      const Block blk(a, sk, sv);
      if constexpr (decltype(more)::value) {
        find(tile + step);
        load_k(tile + step);
      }
      f16x8 p[NR][kTerms];
      softmax(s, p, blk, key0, bad0, slow);
      if (slow) {
#pragma unroll
        for (int t = 0; t < kDims; ++t) keep_first(vw[t], there);
      }
      gather(p, [&](int t, int i) { return Widen<CACHE, f16>::of(vw[t][2 * i], vw[t][2 * i + 1]); });
      if constexpr (decltype(more)::value) load_v(tile + step);
    };
    int tile = t0;
    for (; tile + step < t_end; tile += step) one(tile, std::true_type());
    one(tile, std::false_type());
  }

  __device__ __forceinline__ void total_l() {
#pragma unroll
    for (int r = 0; r < NR; ++r) l[r] = sum_xor32(sum_xor16(l[r]));
  }

  // Row set r to its place: the result, or a split's share of it.
  __device__ __forceinline__ void store(const Args& a, const Request& rq, int h, int row0, int r, int split,
                                        bool whole) const {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int row = row0 + 16 * r + n;
    if (row >= rq.n * a.group) return;
    const int tok = row / a.group;
    const int64_t at = (int64_t)(rq.t0 + tok) * a.heads + h * a.group + (row - tok * a.group);
    if (whole) {
      const float inv = l[r] > 0.f ? 1.f / l[r] : 0.f;
      T* p = static_cast<T*>(a.out) + at * a.head_dim;
#pragma unroll
      for (int t = 0; t < kDims; ++t) {
        const int d = 16 * t + 4 * g;
        if (d < a.head_dim) {
          typename Op16<T>::V4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = (T)(o[r][t][i] * inv);
          *reinterpret_cast<typename Op16<T>::V4*>(p + d) = x;
        }
      }
    } else {
      const int64_t i = (int64_t)split * a.tokens * a.heads + at;
      if (g == 0) a.part_m[i] = make_float2(m[r], l[r]);
      float* p = a.part_o + i * HDP + 4 * g;
#pragma unroll
      for (int t = 0; t < kDims; ++t) *reinterpret_cast<f32x4*>(p + 16 * t) = o[r][t];
    }
  }
};

// Few rows for each kv head: a workgroup has 16 of them and one split of the keys, its waves
// every kWaves-th tile of it; their shares are joined through LDS, the splits' by
// cache_join_kernel.
//
// Bound by memory where the cache is large: 16 requests of 16000 to 32700 keys, 8 heads of 128
// read by 32 (bf16 queries), 804 MB in 135 to 142 us, 5.7 TB/s against a large copy's 5.1 (reads alone are
// faster).  Below that by latency: a wave has one tile's loads in flight and two workgroups
// have a CU (64 requests of up to 2048 keys, 72 MB: 16.9 us; 999 keys of one request: 6.5).
// Eight waves to a workgroup took 24 us for the 64 requests, registers for four waves of a SIMD
// (with scratch) 23, 32 rows a wave 33.6 us for 18 rows where 16 a wave take 26 twice over the
// keys.
template <typename T, int CACHE, int HDP, int KT>
__global__ __launch_bounds__(256) void cache_decode_kernel(Args a) {
  typedef Rows<T, CACHE, HDP, 1, KT> R;
  constexpr int kWaves = 4, kRows = 16;
  __shared__ f32x4 sh_o[kWaves / 2][R::kDims][64];
  __shared__ float sh_m[kWaves / 2][64], sh_l[kWaves / 2][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int id = blockIdx.x;
  const int h = id % a.kv_heads;
  id /= a.kv_heads;
  const int split = id % a.splits;
  id /= a.splits;
  const int b = id % a.batch;
  const Request rq = request_of(a, b);
  const int64_t rows = (int64_t)rq.n * a.group;
  const int chunk = chunk_of(a, rq.len, kWaves * KT);
  if (split > 0 && (int64_t)split * chunk >= rq.len) return;
  for (int64_t row0 = (int64_t)(id / a.batch) * kRows; row0 < rows; row0 += (int64_t)a.row_tiles * kRows) {
    R w;
    w.init(a, rq, h, (int)row0);
    // Keys up to what the tile's last row sees; all of its rows see those below `full`.
    const int64_t end_row = min(row0 + kRows, rows) - 1;
    int end = rq.len, full = rq.len;
    if (a.causal) {
      end = rq.len - rq.n + (int)(end_row / a.group) + 1;
      full = rq.len - rq.n + (int)(row0 / a.group) + 1;
      end = end < 0 ? 0 : end;
    }
    const int64_t k0 = (int64_t)split * chunk;
    const int64_t k1 = min((int64_t)end, k0 + chunk);
    w.pass(a, rq, b, h, (int)(k0 / KT) + wave, (int)((k1 + KT - 1) / KT), kWaves, full);
    w.total_l();
    // The upper half of the waves into the lower, until one is left.
#pragma unroll
    for (int half = kWaves / 2; half; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        sh_m[wave - half][lane] = w.m[0];
        sh_l[wave - half][lane] = w.l[0];
#pragma unroll
        for (int t = 0; t < R::kDims; ++t) sh_o[wave - half][t][lane] = w.o[0][t];
      }
      __syncthreads();
      if (wave < half) {
        const float m2 = sh_m[wave][lane], mn = fmaxf(w.m[0], m2), base = mn == kNegInf ? 0.f : mn;
        const float f1 = __builtin_amdgcn_exp2f(w.m[0] - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
        w.m[0] = mn;
        w.l[0] = w.l[0] * f1 + sh_l[wave][lane] * f2;
#pragma unroll
        for (int t = 0; t < R::kDims; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) w.o[0][t][i] = w.o[0][t][i] * f1 + sh_o[wave][t][lane][i] * f2;
      }
    }
    if (wave == 0) w.store(a, rq, h, (int)row0, 0, split, chunk >= rq.len);
  }
}

// The splits of a row joined: o = sum 2^(M_s - M) O_s / sum 2^(M_s - M) l_s, always in the same
// order.  W waves have a row; a wave takes as many splits at a time as it has lanes for.
// Bound by latency: 4.2 to 4.8 us for a few splits of 134 rows of 256, 5.4 to 6.1 us for 196
// splits of 16 rows of 64.  With one wave the first kEarly rounds are asked for before it is
// known how many splits the row's request has (5.1 us otherwise for the first); four waves
// gained nothing from it (6.3 us for the second), sixteen waves lost (7.6).
template <typename T, int HDP, int W>
__global__ __launch_bounds__(256) void cache_join_kernel(Args a, int step) {
  constexpr int kLanes = HDP / 4, kAt = 64 / kLanes;  // lanes of a split, splits of a wave
  constexpr int kEarly = W > 1 ? 0 : 4;
  __shared__ f32x4 sh[W > 1 ? W : 1][kLanes];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = W > 1 ? wave : 0;
  const int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  if (row >= rows) return;
  const int sub = lane / kLanes, d = (lane - sub * kLanes) * 4, s0 = part * kAt + sub;
  float em[kEarly + 1];
  f32x4 early[kEarly + 1];
#pragma unroll
  for (int i = 0; i < kEarly; ++i) {
    const int s = s0 + i * W * kAt;
    if (sub < kAt && s < a.splits) {
      em[i] = a.part_m[s * rows + row].x;
      early[i] = *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * HDP + d);
    }
  }
  const int t = (int)(row / a.heads);
  int lo = 0;  // the last request with cu[b] <= t
  for (int b0 = 0; b0 < a.batch && a.batch > 1; b0 += 64) {
    const int below = __popcll(__ballot(b0 + lane < a.batch && a.cu[min(b0 + lane, a.batch)] <= t));
    if (below) lo = b0 + below - 1;
    if (below < 64) break;
  }
  const Request rq = request_of(a, lo);
  if (t < rq.t0 || t >= rq.t0 + rq.n) return;
  const int chunk = chunk_of(a, rq.len, step);
  if (chunk >= rq.len) return;  // written by the workgroup that had all of it
  const int n = (int)(((int64_t)rq.len + chunk - 1) / chunk);
  float m = kNegInf;
  for (int s = lane; s < n; s += 64) m = fmaxf(m, a.part_m[s * rows + row].x);
#pragma unroll
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  const float base = m == kNegInf ? 0.f : m;
  float l = 0.f;
  for (int s = lane; s < n; s += 64) {
    const float2 ml = a.part_m[s * rows + row];
    l += __builtin_amdgcn_exp2f(ml.x - base) * ml.y;
  }
  l = group_sum<64>(l);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto take = [&](float ms, const f32x4& x) {
    const float f = __builtin_amdgcn_exp2f(ms - base);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(f, x[i], o[i]);
  };
  if (sub < kAt) {
#pragma unroll
    for (int i = 0; i < kEarly; ++i)
      if (s0 + i * W * kAt < n) take(em[i], early[i]);
#pragma unroll 4
    for (int s = s0 + kEarly * W * kAt; s < n; s += W * kAt)
      take(a.part_m[s * rows + row].x, *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * HDP + d));
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

// Many rows for each kv head: a wave has NR sets of 16 and passes over all of their keys.  Tiles
// of 64 keys go through LDS as codes, once for the four waves: each wave taking them from the
// caches by itself asked 7 TB/s of L2 and waited for half of its time.  Each wave widens what
// it reads: held in 16 bits, widened once, a tile takes twice the LDS reads, which cost more
// (1187 us against 1132).  Codes lie in 16-byte pieces, XOR-swizzled by row so that the eight
// lanes which LDS serves at a time meet eight different places of 128 bytes.  Two stages: a
// tile is in registers while the one before it is in LDS and the one before that in use.
// Sets of 32 rows a wave, so that each widened code feeds two matrix instructions; two
// workgroups to a CU up to head_dim 128.
//
// Bound by the alternation of products and softmax, which hardly overlap: for each of a lane's scores
// an fma, an exponential, a conversion and an addition beside the matrix instructions.  2 requests of
// 2000 new tokens behind 8000 to 14000, 32 heads of 128 on 8 (bf16): 942 us, 0.97 PFLOP/s, the vector
// ALU active in 64 % of cycles, the matrix cores in 40 %.  With few requests by the longest one's tiles:
// 5 of 301 to 1024 new tokens, 16 heads of 64 on 4 (fp16), 159 us, CUs busy for two thirds of it (the
// vector ALU for 67 %, the matrix cores for 32 % of that) while one request's 105 tiles follow each other.
template <typename T, int CACHE, int HDP, int NR>
__global__ __launch_bounds__(256, HDP <= 128 ? 2 : 1) void cache_chunk_kernel(Args a) {
  constexpr int kWaves = 4, kRows = kWaves * NR * 16, KT = 64;
  typedef Rows<T, CACHE, HDP, NR, KT> R;
  constexpr int kC = HDP / 16, kPer = (HDP + 63) / 64;  // 16 codes each: of a K row; a thread's of K, of V
  constexpr bool kAll = HDP % 64 == 0;
  // At head_dim 128 int8's widening leaves no registers for a product's codes at once.
  constexpr bool kBatch = CACHE == kCacheE4M3 || HDP != 128;
  __shared__ u32x4 sh_k[2][KT * kC], sh_v[2][HDP * 4];
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto swz = [](int row) { return kC == 8 || kC == 16 ? row & 7 : kC == 4 || kC == 12 ? (row >> 1) & 3 : (row >> 2) & 1; };
  auto swz_v = [](int d) { return (d >> 1) & 3; };
  // The longest request first (where a wave can rank them), of a request the row tiles with the
  // most keys first: workgroups start in order of their ids, and what starts last should be
  // short.  Neighbours, which go to XCDs round-robin, take different kv heads.
  int id = blockIdx.x;
  const int h = id % a.kv_heads;
  id /= a.kv_heads;
  const int tile0 = a.row_tiles - 1 - id % a.row_tiles;
  id /= a.row_tiles;
  const int split = id % a.splits;
  int b = id / a.splits;
  if (a.batch <= 64) {
    const int len = lane < a.batch ? a.lens[lane] : -1;
    int rank = 0;
    for (int k = 0; k < a.batch; ++k) {
      const int other = __builtin_amdgcn_readlane(len, k);
      rank += other > len || (other == len && k < lane);
    }
    b = __builtin_ctzll(__ballot(lane < a.batch && rank == b));
  }
  const Request rq = request_of(a, b);
  const int64_t rows = (int64_t)rq.n * a.group;
  const int chunk = chunk_of(a, rq.len, KT);
  if (split > 0 && (int64_t)split * chunk >= rq.len) return;
  const int first = split * (chunk / KT);
  const int bs = 1 << a.shift;
  const Strides st(a, h, bs * HDP);
  Pages pages(a, b, (first * KT) >> a.shift);

  // What this thread brings of a tile: of K 16-code pieces lane, lane + 64, .. of the keys of
  // group `wave`, of V pieces tid, tid + 256, .. (four to a dimension).
  u32x4 rk[kPer], rv[kPer];
  // Blocks of a tile's four groups of 16 keys.  With blocks of 64 tokens and more they are one,
  // and everything that depends on it is the same for all lanes.
  const bool one = a.shift >= 6;
  struct Ids {
    int i0, i1, i2, i3;
    __device__ __forceinline__ int of(int i) const {
      const int even = i & 2 ? +i2 : +i0, odd = i & 2 ? +i3 : +i1;
      return i & 1 ? odd : even;
    }
  };
  auto load_ids = [&](int tile) {
    pages.reach(a, (tile * KT) >> a.shift);
    Ids x;
    x.i0 = pages.one((tile * KT) >> a.shift);
    if (!one) {
      x.i1 = pages.one((tile * KT + 16) >> a.shift);
      x.i2 = pages.one((tile * KT + 32) >> a.shift);
      x.i3 = pages.one((tile * KT + 48) >> a.shift);
    }
    return x;
  };
  const uint32_t k_off = lane * 16, v_off = (tid >> 2) * bs;
  auto load_k = [&](int tile, const Ids& ids) {
    const int id = one ? ids.i0 : ids.of(wave);
    const uint8_t* pk = st.k + st.block(id) + (uint32_t)(((tile * KT + 16 * wave) & (bs - 1)) * HDP);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (kAll || lane + 64 * i < HDP) rk[i] = *reinterpret_cast<const u32x4*>(pk + (k_off + 1024u * i));
  };
  int there = 64;  // tokens of the V piece that are the request's
  float sk = 1.f, sv = 1.f;
  bool bad = false;
  auto load_v = [&](int tile, const Ids& ids) {
    there = rq.len - tile * KT - 16 * (tid & 3);
    if (one) {
      const uint8_t* pv = st.v + st.block(ids.i0) + (uint32_t)((tile * KT) & (bs - 1));
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (kAll || (tid >> 2) + 64 * i < HDP) rv[i] = *reinterpret_cast<const u32x4*>(pv + (v_off + (tid & 3) * 16 + 64u * i * bs));
      if (!st.there(ids.i0)) there = 0;
    } else {
      const int id = ids.of(tid & 3);
      const uint8_t* pv = st.v + st.block(id) + (uint32_t)((tile * KT + 16 * (tid & 3)) & (bs - 1));
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (kAll || (tid >> 2) + 64 * i < HDP) rv[i] = *reinterpret_cast<const u32x4*>(pv + (v_off + 64u * i * bs));
      if (!st.there(id)) there = 0;
    }
  };
  auto load_scales = [&](const Ids& ids) {
    const int id = one ? ids.i0 : ids.of(g);
    sk = st.k_scale[st.scale(id)];
    sv = st.v_scale[st.scale(id)];
    bad = !st.there(id);
  };
  auto put_k = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = lane + 64 * i, key = c / kC, row = 16 * (key >> 2) + 4 * wave + (key & 3);
      if (kAll || c < HDP) sh_k[stage][row * kC + ((c % kC) ^ swz(row))] = rk[i];
    }
  };
  auto put_v = [&](int stage) {
    if (__any(there < 16)) {
      asm volatile("");  // a branch, not 20 instructions for every tile
#pragma unroll
      for (int i = 0; i < kPer; ++i) keep_first(rv[i], there);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = (tid >> 2) + 64 * i;
      if (kAll || d < HDP) sh_v[stage][d * 4 + ((tid & 3) ^ swz_v(d))] = rv[i];
    }
  };

  for (int64_t at = (int64_t)tile0 * kRows; at < rows; at += (int64_t)a.row_tiles * kRows) {
    if (at != (int64_t)tile0 * kRows) pages = Pages(a, b, (first * KT) >> a.shift);
    const int64_t row0 = at + wave * NR * 16;
    R w;
    w.init(a, rq, h, (int)row0);
    wait_vmcnt<0>();  // the queries: waited for in the loop, they would take every tile's loads along
    // Tiles that any of the workgroup's rows see; keys that all of this wave's do.
    int full = rq.len, most = rq.len;
    if (a.causal) {
      full = rq.len - rq.n + (int)(row0 / a.group) + 1;
      most = rq.len - rq.n + (int)((min(at + kRows, rows) - 1) / a.group) + 1;
    }
    most = most > 0 ? (most + KT - 1) / KT : 0;
    if (most > first + chunk / KT) most = first + chunk / KT;
    __syncthreads();
    Ids ids, next;  // of the tiles two ahead and one ahead
    int begin = first;
    asm volatile("" : "+s"(begin));  // nothing of a first tile's addresses is kept for the next round of rows
    if (begin < most) {
      ids = load_ids(begin);
      load_k(begin, ids);
      load_v(begin, ids);
      load_scales(ids);
      put_k(begin & 1);
      put_v(begin & 1);
      next = load_ids(begin + 1);
      load_k(begin + 1, next);
      load_v(begin + 1, next);
      ids = load_ids(begin + 2);
    }
    for (int tile = first; tile < most; ++tile) {
      lds_barrier();  // this tile's stage is written, the other one read
      const int key0 = tile * KT + 16 * g;
      const bool bad0 = bad, slow = tile * KT + KT > full || __any(bad);
      const u32x4 *pk = sh_k[tile & 1] + n * kC, *pv = sh_v[tile & 1] + n * 4 + (g ^ swz_v(n));
      // All of a product's codes are asked for before its first instruction, V's before the
      // softmax where there are registers: one wait for LDS, or none, in place of one for each.
      u32x4 kw[4][R::kWide > 0 ? R::kWide : 1];
      u32x2 ko[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < R::kWide; ++j) kw[i][j] = pk[i * 16 * kC + ((4 * j + g) ^ swz(n))];
        if constexpr (R::kOdd)
          ko[i] = reinterpret_cast<const u32x2*>(pk + i * 16 * kC + ((4 * R::kWide + (g >> 1)) ^ swz(n)))[g & 1];
      }
      if constexpr (kBatch) __builtin_amdgcn_sched_barrier(0);
      f32x4 s[NR][4];
      w.scores(s, [&](int i, int j) {
        if (R::kOdd && j == R::kSteps - 1) return Widen<CACHE, T>::of(ko[i][0], ko[i][1]);
        return Widen<CACHE, T>::of(kw[i][j >> 1][2 * (j & 1)], kw[i][j >> 1][2 * (j & 1) + 1]);
      });
      u32x4 vw[R::kDims];
      auto ask_v = [&]() {
#pragma unroll
        for (int t = 0; t < R::kDims; ++t) vw[t] = pv[t * 64];
        if constexpr (kBatch) __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr (HDP < 96) ask_v();
      f16x8 p[NR][R::kTerms];
      w.softmax(s, p, typename R::Block(a, sk, sv), key0, bad0, slow);
      if constexpr (HDP >= 96) ask_v();
      w.gather(p, [&](int t, int i) { return Widen<CACHE, f16>::of(vw[t][2 * i], vw[t][2 * i + 1]); });
      if (tile + 1 < most) {
        put_k((tile + 1) & 1);
        put_v((tile + 1) & 1);
        load_scales(next);
        load_k(tile + 2, ids);
        load_v(tile + 2, ids);
        next = ids;
        ids = load_ids(tile + 3);
      }
    }
    if (row0 < rows) {
      w.total_l();
#pragma unroll
      for (int r = 0; r < NR; ++r) w.store(a, rq, h, (int)row0, r, split, chunk >= rq.len);
    }
  }
}

struct Plan {
  bool chunked;
  int step;  // keys that a workgroup takes at a time
  int splits, chunk;
  int64_t row_tiles;
};

// Keys of a tile: at head_dim over 128 two waves of a SIMD have no registers for 64.
constexpr int decode_keys(int width) { return width <= 128 ? 64 : 32; }

// How a call is cut.  max_new and max_len are expectations; a call that exceeds them is still
// covered (rows in a loop, longer splits).
Plan plan_of(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
             int64_t max_len) {
  Plan p{};
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

template <typename T, int CACHE, int HDP>
hipError_t launch(const Args& a, const Plan& p, hipStream_t stream) {
  const int64_t grid = (int64_t)a.batch * a.kv_heads * p.row_tiles * p.splits;
  if (grid > kMaxGrid) return hipErrorInvalidValue;
  const dim3 groups((unsigned)grid), block(256);
  const hipError_t e =
      p.chunked ? launch_status(cache_chunk_kernel<T, CACHE, HDP, 2>, groups, block, stream, a)
                : launch_status(cache_decode_kernel<T, CACHE, HDP, decode_keys(HDP)>, groups, block, stream, a);
  if (p.splits <= 1 || e != hipSuccess) return e;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  return p.splits > 16 ? launch_status(cache_join_kernel<T, HDP, 4>, dim3((unsigned)rows), block, stream, a, p.step)
                       : launch_status(cache_join_kernel<T, HDP, 1>, dim3((unsigned)((rows + 3) / 4)), block, stream, a,
                                       p.step);
}

template <typename T, int CACHE>
hipError_t launch_width(const Args& a, const Plan& p, int width, hipStream_t stream) {
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
  const Plan p = plan_of(tokens, batch, heads, kv_heads, head_dim, max_new, max_len);
  if (p.splits <= 1) return 0;
  return (int64_t)p.splits * tokens * heads * (cache_width(head_dim) * 4 + 8);
}

hipError_t run_cache_attn(const CacheAttnArgs& c, int64_t workspace_bytes, hipStream_t stream) {
  const int width = cache_width(c.head_dim);
  if (width < 0 || c.tokens <= 0 || c.tokens > 0x7fffffff || c.batch <= 0 || c.table_width <= 0 ||
      c.tokens * c.heads > 0x7fffff00)  // rows of a kv head are counted in 32 bits
    return hipErrorInvalidValue;
  const Plan p = plan_of(c.tokens, c.batch, c.heads, c.kv_heads, c.head_dim, c.max_new, c.max_len);
  Args a{};
  a.q = c.q;
  a.out = c.out;
  a.cu = c.cu;
  a.lens = c.lens;
  a.table = c.table;
  a.k = static_cast<const uint8_t*>(c.k);
  a.v = static_cast<const uint8_t*>(c.v);
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  a.ldq = c.ldq;
  a.table_width = c.table_width;
  a.num_blocks = c.num_blocks;
  a.tokens = (int)c.tokens;
  a.batch = c.batch;
  a.heads = c.heads;
  a.kv_heads = c.kv_heads;
  a.group = c.heads / c.kv_heads;
  a.head_dim = c.head_dim;
  a.shift = c.shift;
  a.causal = c.causal;
  a.c2 = c.scale * 1.4426950408889634f;
  a.splits = p.splits;
  a.chunk = p.chunk;
  a.row_tiles = (int)p.row_tiles;
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

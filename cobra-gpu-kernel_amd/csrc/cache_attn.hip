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
// whatever the activations' type: codes are exact in fp16.
// Scores, M, l and O are fp32.  Scales are taken within [2^-40, 2^40], so no w that counts
// underflows and neither sum overflows.
//
// Tiles are 64 keys and 16 rows (v_mfma_f32_16x16x32): S^T = K Q^T, then O^T = V^T P^T.  Row r
// of K's subtile s is key 16 (r / 4) + 4 s + r % 4, which leaves the scores of keys
// 16 g .. 16 g + 15 in lane group g = lane / 16, in order: exactly the keys whose codes that
// group reads of V^T in one 16-byte load.  P goes from the softmax into the product without
// leaving its lane, K and V from memory into the matrix cores without passing LDS, and since a
// block is at least 16 tokens a lane needs one K scale and one V scale for a tile.
#include "common.hpp"
#include "kernels.hpp"
#include "lds_dma.hpp"

namespace cobra {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr float kBias = 8.f;         // log2 of w where u equals its reference
constexpr float kAccept = 57344.f;   // a lane's sum of w that is taken without a maximum

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
  const int64_t most = min(a.table_width << a.shift, (int64_t)0x7fffff00);
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

// One wave's state for NR sets of 16 rows and its pass over some tiles of keys.
template <typename T, int CACHE, int HDP, int NR, int KT>
struct Rows {
  typedef typename Op16<T>::V8 V8;
  static constexpr int kSteps = HDP / 32, kWide = HDP / 64, kOdd = kSteps & 1, kDims = HDP / 16;
  static constexpr int kSub = KT / 16, kKeys = KT / 4, kWords = KT / 16, kParts = KT / 32;
  typedef uint32_t VWords __attribute__((ext_vector_type(kWords)));

  V8 q[NR][kSteps];
  f32x4 o[NR][kDims];
  float m[NR], l[NR];  // l: this lane group's share
  int lim[NR];         // keys that this lane's row sees

  __device__ __forceinline__ void init(const Args& a, const Request& rq, int h, int64_t row0) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int64_t row = row0 + 16 * r + n;
      const bool there = row < (int64_t)rq.n * a.group;
      const int tok = there ? (int)(row / a.group) : 0;
      const int head = h * a.group + (there ? (int)(row - (int64_t)tok * a.group) : 0);
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
  // counts in l all the same).
  static __device__ __forceinline__ float weigh(const f32x4 (&s)[kSub], float skc, float shift, f16x8 (&p)[kParts]) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < kKeys; e += 2) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], skc, shift));
      const float y = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][(e & 3) + 1], skc, shift));
      p[e >> 3][e & 7] = (f16)x;
      p[e >> 3][(e & 7) + 1] = (f16)y;
      sum += x + y;
    }
    return sum;
  }

  // S^T = K Q^T on codes; wide(i, j) and odd(i): this lane's K codes of subtile i.
  template <typename W, typename O>
  __device__ __forceinline__ void scores(f32x4 (&s)[NR][kSub], W&& wide, O&& odd) {
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int i = 0; i < kSub; ++i) s[r][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
#pragma unroll
      for (int j = 0; j < kWide; ++j) {
        const u32x4 k = wide(i, j);
        const V8 lo = Widen<CACHE, T>::of(k.x, k.y), hi = Widen<CACHE, T>::of(k.z, k.w);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][i] = mfma16(lo, q[r][2 * j], s[r][i]);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][i] = mfma16(hi, q[r][2 * j + 1], s[r][i]);
      }
      if constexpr (kOdd) {
        const u32x2 k = odd(i);
        const V8 lo = Widen<CACHE, T>::of(k.x, k.y);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][i] = mfma16(lo, q[r][kSteps - 1], s[r][i]);
      }
    }
  }

  // Scores to weights: this lane's keys begin at key0, its block's scales are sk and sv (of a
  // block outside the pool: bad); slow: not every row sees every key of the tile.
  __device__ __forceinline__ void softmax(const Args& a, f32x4 (&s)[NR][kSub], f16x8 (&p)[NR][kParts], float sk,
                                          float sv, int key0, bool bad, bool slow) {
    const float skc = fminf(fmaxf(sk, 0x1p-40f), 0x1p40f) * a.c2, svc = fminf(fmaxf(sv, 0x1p-40f), 0x1p40f);
    const float ev = __builtin_amdgcn_logf(svc), inv = 1.f / svc;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      // Against the reference that the row has, without a maximum of this tile: right as long
      // as every w stays inside fp16, which a sum at most kAccept of a lane's w shows.
      float shift = ev + kBias - m[r], sum;
      bool ok = false;
      if (!slow) {
        sum = weigh(s[r], skc, shift, p[r]);
        ok = sum <= kAccept;  // false for NaN, and where the row has no reference yet
      }
      if (!__all(ok)) {
        const int seen = bad ? 0 : slow ? lim[r] - key0 : kKeys;  // keys of this lane that count
        float mx = kNegInf;
#pragma unroll
        for (int e = 0; e < kKeys; ++e) {
          const float u = fmaf(s[r][e >> 2][e & 3], skc, ev);
          s[r][e >> 2][e & 3] = e < seen ? s[r][e >> 2][e & 3] : kNegInf;
          mx = fmaxf(mx, e < seen ? u : kNegInf);
        }
        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = max_xor32(fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])));
        const float mn = fmaxf(m[r], mx);
        const float alpha = mn == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m[r] - mn);
        m[r] = mn;
        shift = mn == kNegInf ? kNegInf : ev + kBias - mn;
        sum = weigh(s[r], skc, shift, p[r]);
        l[r] *= alpha;
#pragma unroll
        for (int t = 0; t < kDims; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[r][t][i] *= alpha;
      }
      l[r] = fmaf(sum, inv, l[r]);
    }
  }

  // O^T += V^T P^T on codes; codes(t): this lane's keys of dimension 16 t + n, of which the
  // first `there` count where cut (memory past a request's end, or of a block that is none,
  // may hold NaN codes).
  template <typename V>
  __device__ __forceinline__ void gather(const f16x8 (&p)[NR][kParts], V&& codes, bool cut, int there) {
    if (cut) {
#pragma unroll
      for (int t = 0; t < kDims; ++t) {
        VWords v = codes(t);
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const int c = there - 4 * i;
          v[i] = c >= 4 ? v[i] : c <= 0 ? 0u : v[i] & (0xffffffffu >> (8 * (4 - c)));
        }
        add(t, v, p);
      }
    } else {
#pragma unroll
      for (int t = 0; t < kDims; ++t) add(t, codes(t), p);
    }
  }
  __device__ __forceinline__ void add(int t, const VWords& v, const f16x8 (&p)[NR][kParts]) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const f16x8 w = Widen<CACHE, f16>::of(v[2 * i], v[2 * i + 1]);
#pragma unroll
      for (int r = 0; r < NR; ++r) o[r][t] = mfma16(w, p[r][i], o[r][t]);
    }
  }

  // Tiles t0, t0 + step, .. below t_end, K and V straight from memory to registers; keys from
  // `full` on are checked against each row's limit.
  __device__ __forceinline__ void pass(const Args& a, const Request& rq, int b, int h, int t0, int t_end, int step,
                                       int full) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15, gk = n >> 2;
    const int32_t* table = a.table + b * a.table_width;
    const int bs = 1 << a.shift, last_page = (int)a.table_width - 1;
    const int64_t plane = (int64_t)bs * HDP;
    if (t0 >= t_end) return;

    // Block ids of a tile: of the group whose K rows this lane reads, and of its own V keys.
    auto page = [&](int tile, int grp) {
      const int p = (tile * KT + kKeys * grp) >> a.shift;
      return table[p < last_page ? p : last_page];
    };
    u32x4 kw[kSub][kWide > 0 ? kWide : 1];
    u32x2 ko[kSub];
    VWords vw[kDims];
    float sk, sv;
    int idk = page(t0, gk), idv = page(t0, g);
    bool bad_next = false;
    auto clamp_id = [&](int id) { return (unsigned)id < (unsigned)a.num_blocks ? id : 0; };
    auto load_k = [&](int tile) {
      const int64_t at = ((int64_t)clamp_id(idk) * a.kv_heads + h) * plane;
      const int off = (tile * KT + kKeys * gk + (n & 3)) & (bs - 1);
      const uint8_t* p = a.k + at + (int64_t)off * HDP;
#pragma unroll
      for (int s = 0; s < kSub; ++s) {
#pragma unroll
        for (int j = 0; j < kWide; ++j) kw[s][j] = *reinterpret_cast<const u32x4*>(p + s * 4 * HDP + 64 * j + 16 * g);
        if constexpr (kOdd) ko[s] = *reinterpret_cast<const u32x2*>(p + s * 4 * HDP + 64 * kWide + 8 * g);
      }
    };
    auto load_v = [&](int tile) {
      const int64_t bh = (int64_t)clamp_id(idv) * a.kv_heads + h;
      const int off = (tile * KT + kKeys * g) & (bs - 1);
      const uint8_t* p = a.v + bh * plane + (int64_t)n * bs + off;
#pragma unroll
      for (int t = 0; t < kDims; ++t) vw[t] = *reinterpret_cast<const VWords*>(p + (int64_t)t * 16 * bs);
    };
    auto load_scales = [&]() {
      const int64_t bh = (int64_t)clamp_id(idv) * a.kv_heads + h;
      sk = a.k_scale[bh];
      sv = a.v_scale[bh];
      bad_next = (unsigned)idv >= (unsigned)a.num_blocks;
    };
    load_k(t0);
    load_scales();
    load_v(t0);
    int idk2 = 0, idv2 = 0;
    if (t0 + step < t_end) {
      idk2 = page(t0 + step, gk);
      idv2 = page(t0 + step, g);
    }
    for (int tile = t0; tile < t_end; tile += step) {
      const bool more = tile + step < t_end;
      const int key0 = tile * KT + kKeys * g;  // this lane's first key
      f32x4 s[NR][kSub];
      scores(s, [&](int i, int j) { return kw[i][j]; }, [&](int i) { return ko[i]; });
      const bool bad = bad_next;
      const float sk0 = sk, sv0 = sv;
      // The next tile's keys and scales while this one's softmax runs.
      if (more) {
        idk = idk2;
        idv = idv2;
        load_k(tile + step);
        load_scales();
        if (tile + 2 * step < t_end) {
          idk2 = page(tile + 2 * step, gk);
          idv2 = page(tile + 2 * step, g);
        }
      }
      const bool slow = tile * KT + KT > full || __any(bad);
      f16x8 p[NR][kParts];
      softmax(a, s, p, sk0, sv0, key0, bad, slow);
      gather(p, [&](int t) { return vw[t]; }, slow, bad ? 0 : rq.len - key0);
      if (more) load_v(tile + step);
    }
  }

  __device__ __forceinline__ void total_l() {
#pragma unroll
    for (int r = 0; r < NR; ++r) l[r] = sum_xor32(sum_xor16(l[r]));
  }

  // Row set r to its place: the result, or a split's share of it.
  __device__ __forceinline__ void store(const Args& a, const Request& rq, int h, int64_t row0, int r, int split,
                                        bool whole) const {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15;
    const int64_t row = row0 + 16 * r + n;
    if (row >= (int64_t)rq.n * a.group) return;
    const int tok = (int)(row / a.group);
    const int64_t at = (int64_t)(rq.t0 + tok) * a.heads + h * a.group + (row - (int64_t)tok * a.group);
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
template <typename T, int CACHE, int HDP, int NR, int KT, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void cache_decode_kernel(Args a) {
  typedef Rows<T, CACHE, HDP, NR, KT> R;
  constexpr int kRows = 16 * NR;
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
    w.init(a, rq, h, row0);
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
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int half = kWaves / 2; half; half >>= 1) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
          sh_m[wave - half][lane] = w.m[r];
          sh_l[wave - half][lane] = w.l[r];
#pragma unroll
          for (int t = 0; t < R::kDims; ++t) sh_o[wave - half][t][lane] = w.o[r][t];
        }
        __syncthreads();
        if (wave < half) {
          const float m2 = sh_m[wave][lane], mn = fmaxf(w.m[r], m2), base = mn == kNegInf ? 0.f : mn;
          const float f1 = __builtin_amdgcn_exp2f(w.m[r] - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
          w.m[r] = mn;
          w.l[r] = w.l[r] * f1 + sh_l[wave][lane] * f2;
#pragma unroll
          for (int t = 0; t < R::kDims; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) w.o[r][t][i] = w.o[r][t][i] * f1 + sh_o[wave][t][lane][i] * f2;
        }
      }
      if (wave == 0) w.store(a, rq, h, row0, r, split, chunk >= rq.len);
    }
  }
}

// The splits of a row joined: o = sum 2^(M_s - M) O_s / sum 2^(M_s - M) l_s, always in the same
// order.  W waves have a row; a wave takes as many splits at a time as it has lanes for.
template <typename T, int HDP, int W>
__global__ __launch_bounds__(256) void cache_join_kernel(Args a, int step) {
  constexpr int kLanes = HDP / 4, kAt = 64 / kLanes;  // lanes of a split, splits of a wave
  __shared__ f32x4 sh[W > 1 ? W : 1][kLanes];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = W > 1 ? wave : 0;
  const int64_t row = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  if (row >= rows) return;
  const int t = (int)(row / a.heads);
  int lo = 0, hi = a.batch;  // the last request with cu[b] <= t
  while (lo + 1 < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.cu[mid] <= t)
      lo = mid;
    else
      hi = mid;
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
  const int sub = lane / kLanes, d = (lane - sub * kLanes) * 4;
  if (sub < kAt) {
#pragma unroll 4
    for (int s = part * kAt + sub; s < n; s += W * kAt) {
      const float f = __builtin_amdgcn_exp2f(a.part_m[s * rows + row].x - base);
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * HDP + d);
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

// Many rows for each kv head: a wave has NR sets of 16 and passes over all of their keys.  Tiles
// of 64 keys go through LDS, whence all four waves read their codes (each taking them from the
// caches by itself asked 7 TB/s of L2 and waited for half of its time): 16-byte chunks in the
// order in which a wave reads them, XOR-swizzled by row so that eight lanes in a row meet eight
// different ones of 128 bytes' places.  Two stages: a tile is in registers while the one before
// it is in LDS and the one before that in use.
template <typename T, int CACHE, int HDP, int NR>
__global__ __launch_bounds__(256, HDP <= 128 ? 2 : 1) void cache_chunk_kernel(Args a) {
  constexpr int kWaves = 4, kRows = kWaves * NR * 16, KT = 64;
  typedef Rows<T, CACHE, HDP, NR, KT> R;
  constexpr int kC = HDP / 16, kPer = (HDP + 63) / 64;  // chunks of a K row; a thread's of K, of V
  __shared__ u32x4 sh_k[2][KT * kC], sh_v[2][HDP * 4];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, n = lane & 15;
  auto swz = [](int row) {
    return kC == 8 || kC == 16 ? row & 7 : kC == 4 || kC == 12 ? (row >> 1) & 3 : (row >> 2) & 1;
  };
  // Workgroups go to XCDs round-robin: every eighth (request, kv head) pair to the same one,
  // whose L2 then serves the pair's keys to all of its row tiles.
  const int pairs = a.batch * a.kv_heads;
  const int l = blockIdx.x / 8, pair = l / a.row_tiles * 8 + blockIdx.x % 8, tile0 = l % a.row_tiles;
  if (pair >= pairs) return;
  const int h = pair % a.kv_heads, b = pair / a.kv_heads;
  const Request rq = request_of(a, b);
  const int64_t rows = (int64_t)rq.n * a.group;
  const int bs = 1 << a.shift, last_page = (int)a.table_width - 1;
  const int64_t plane = (int64_t)bs * HDP;
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  const cptr table = (cptr)(a.table + b * a.table_width);

  // What this thread brings of a tile: K chunks lane, lane + 64, .. of the 16 keys of group
  // `wave`, V chunks tid, tid + 256, .. (four to a dimension).
  u32x4 rk[kPer], rv[kPer];
  int id0, id1, id2, id3;  // block ids of a tile's four groups of 16 keys
  float sk, sv, sk1, sv1;
  bool bad = false, bad1 = false;
  auto load_ids = [&](int tile) {
    auto id = [&](int i) {
      const int p = (tile * KT + 16 * i) >> a.shift;
      return (int)table[p < last_page ? p : last_page];
    };
    id0 = id(0);
    id1 = id(1);
    id2 = id(2);
    id3 = id(3);
  };
  auto pick = [&](int i) {
    const int even = i & 2 ? +id2 : +id0, odd = i & 2 ? +id3 : +id1;
    return i & 1 ? odd : even;
  };
  auto block = [&](int id) { return (int64_t)((unsigned)id < (unsigned)a.num_blocks ? id : 0) * a.kv_heads + h; };
  auto load = [&](int tile) {
    const uint8_t* pk = a.k + block(pick(wave)) * plane + (int64_t)((tile * KT + 16 * wave) & (bs - 1)) * HDP;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (HDP % 64 == 0 || lane + 64 * i < HDP) rk[i] = *reinterpret_cast<const u32x4*>(pk + (lane + 64 * i) * 16);
    const int part = tid & 3;
    const uint8_t* pv = a.v + block(pick(part)) * plane + ((tile * KT + 16 * part) & (bs - 1)) + (int64_t)(tid >> 2) * bs;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (HDP % 64 == 0 || (tid >> 2) + 64 * i < HDP) rv[i] = *reinterpret_cast<const u32x4*>(pv + (int64_t)i * 64 * bs);
    const int id = pick(g);
    sk1 = a.k_scale[block(id)];
    sv1 = a.v_scale[block(id)];
    bad1 = (unsigned)id >= (unsigned)a.num_blocks;
  };
  auto put = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = lane + 64 * i, key = c / kC, row = 16 * (key >> 2) + 4 * wave + (key & 3);
      if (HDP % 64 == 0 || c < HDP) sh_k[stage][row * kC + ((c % kC) ^ swz(row))] = rk[i];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = (tid >> 2) + 64 * i;
      if (HDP % 64 == 0 || d < HDP) sh_v[stage][d * 4 + ((tid & 3) ^ ((d >> 1) & 3))] = rv[i];
    }
    sk = sk1;
    sv = sv1;
    bad = bad1;
  };

  for (int64_t at = (int64_t)tile0 * kRows; at < rows; at += (int64_t)a.row_tiles * kRows) {
    const int64_t row0 = at + wave * NR * 16;
    R w;
    w.init(a, rq, h, row0);
    // Tiles that this wave's rows see, and that any of the workgroup's do.
    const int64_t end_row = min(row0 + NR * 16, rows) - 1;
    int end = rq.len, full = rq.len, most = rq.len;
    if (a.causal) {
      end = rq.len - rq.n + (int)(end_row / a.group) + 1;
      full = rq.len - rq.n + (int)(row0 / a.group) + 1;
      most = rq.len - rq.n + (int)((min(at + kRows, rows) - 1) / a.group) + 1;
    }
    end = row0 < rows && end > 0 ? (end + KT - 1) / KT : 0;
    most = most > 0 ? (most + KT - 1) / KT : 0;
    __syncthreads();
    if (most > 0) {
      load_ids(0);
      load(0);
      put(0);
      if (most > 1) {
        load_ids(1);
        load(1);
        load_ids(2);
      }
    }
    for (int tile = 0; tile < most; ++tile) {
      lds_barrier();  // this tile's stage is written, the other one read
      const int key0 = tile * KT + 16 * g;
      const float sk0 = sk, sv0 = sv;
      const bool bad0 = bad;
      if (tile < end) {
        const u32x4 *pk = sh_k[tile & 1] + n * kC, *pv = sh_v[tile & 1];
        f32x4 s[NR][4];
        w.scores(
            s, [&](int i, int j) { return pk[i * 16 * kC + ((4 * j + g) ^ swz(n))]; },
            [&](int i) {
              return reinterpret_cast<const u32x2*>(pk + i * 16 * kC + ((4 * R::kWide + (g >> 1)) ^ swz(n)))[g & 1];
            });
        const bool slow = tile * KT + KT > full || __any(bad0);
        f16x8 p[NR][2];
        w.softmax(a, s, p, sk0, sv0, key0, bad0, slow);
        w.gather(
            p,
            [&](int t) {
              const int d = 16 * t + n;
              return __builtin_bit_cast(typename R::VWords, pv[d * 4 + (g ^ ((d >> 1) & 3))]);
            },
            slow, bad0 ? 0 : rq.len - key0);
      }
      if (tile + 1 < most) {
        put((tile + 1) & 1);
        if (tile + 2 < most) {
          load(tile + 2);
          load_ids(tile + 3);
        }
      }
    }
    if (row0 < rows) {
      w.total_l();
#pragma unroll
      for (int r = 0; r < NR; ++r) w.store(a, rq, h, row0, r, 0, true);
    }
  }
}

struct Plan {
  bool chunked;
  int sets;    // of 16 rows, a workgroup's (decode)
  int step;    // keys that a decode workgroup takes at a time
  int splits, chunk;
  int64_t row_tiles;
};

constexpr int decode_keys(int width) { return width <= 128 ? 64 : 32; }

#include <stdlib.h>
static int tune(const char* n, int d) { const char* v = getenv(n); return v ? atoi(v) : d; }
// How a call is cut.  max_new and max_len are expectations; a call that exceeds them is still
// covered (rows in a loop, longer splits).
Plan plan_of(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t max_new,
             int64_t max_len) {
  Plan p{};
  max_new = max_new < 1 ? 1 : max_new > tokens ? tokens : max_new;
  max_len = max_len < 1 ? 1 : max_len > 0x7fffff00 ? 0x7fffff00 : max_len;
  const int64_t group = heads / kv_heads, rows = max_new * group;
  static const int cr = tune("CR", 64), c2 = tune("C2", 16);
  p.chunked = rows > cr;
  p.splits = 1;
  if (p.chunked) {
    const int per = cache_width(head_dim) <= 128 ? 128 : 64;
    p.row_tiles = (rows + per - 1) / per;
    p.chunk = 0x40000000;
    return p;
  }
  p.sets = rows > c2 ? 2 : 1;
  p.row_tiles = (rows + 16 * p.sets - 1) / (16 * p.sets);
  p.step = 4 * decode_keys(cache_width(head_dim));
  const int64_t base = batch * kv_heads * p.row_tiles;
  static const int target = tune("CT", 512), one = tune("CO", 0);
  int64_t splits = (target + base - 1) / base;
  const int64_t most = (max_len + p.step - 1) / p.step;
  splits = splits < most ? splits : most;
  splits = splits < 1 ? 1 : splits > 1024 ? 1024 : splits;
  if (max_len <= one) splits = 1;
  const int64_t even = (max_len + splits - 1) / splits;
  int64_t chunk = (even + p.step - 1) / p.step * p.step;
  if (chunk < p.step) chunk = p.step;
  p.splits = (int)((max_len + chunk - 1) / chunk);
  if (p.splits < 1) p.splits = 1;
  p.chunk = (int)chunk;
  return p;
}

template <typename T, int CACHE, int HDP>
hipError_t launch(const Args& a, const Plan& p, hipStream_t stream) {
  constexpr int kKeys = decode_keys(HDP);
  if (p.chunked) {
    const int64_t grid = ((int64_t)a.batch * a.kv_heads + 7) / 8 * 8 * p.row_tiles;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL((cache_chunk_kernel<T, CACHE, HDP, HDP <= 128 ? 2 : 1>), dim3((unsigned)grid),
                       dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  const int64_t grid = (int64_t)a.batch * a.kv_heads * p.row_tiles * p.splits;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  if (p.sets == 1)
    hipLaunchKernelGGL((cache_decode_kernel<T, CACHE, HDP, 1, kKeys, 4>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((cache_decode_kernel<T, CACHE, HDP, 2, kKeys, 4>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  if (p.splits > 1) {
    const int64_t rows = (int64_t)a.tokens * a.heads;
    if (p.splits > 16)
      hipLaunchKernelGGL((cache_join_kernel<T, HDP, 4>), dim3((unsigned)rows), dim3(256), 0, stream, a, p.step);
    else
      hipLaunchKernelGGL((cache_join_kernel<T, HDP, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, stream, a,
                         p.step);
  }
  return hipGetLastError();
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
  if (width < 0 || c.tokens <= 0 || c.tokens > 0x7fffffff || c.batch <= 0 || c.table_width <= 0) return hipErrorInvalidValue;
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

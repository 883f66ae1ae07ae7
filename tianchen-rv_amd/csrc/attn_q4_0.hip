// attn_q4_0.hip -- attention over the paged Q4_0 cache.
//
// A row is one query head of one new token; the rows of one request that share a kv head are
// numbered token first, and a tile is 16 of them.  Both products run on
// v_mfma_f32_16x16x32_f16 with the rows as columns:
//   scores  S' = K q'    (16 tokens x 32 elements of a block) x (32 x 16 rows)
//   output  O' = V' P'   (16 elements x 32 tokens) x (32 x 16 rows)
// so that a lane keeps one row throughout: the weights leave the first product in the lanes and
// the order in which the second one reads them, and the row's maximum, sum and rescale are one
// register each.
//
// A dword of 8 quants becomes four operand registers: 4 bits n over the bits of 1024.0 are 1024 + n,
// and a packed subtraction leaves n - 8, exactly.  (Left at the bottom of a half, n is the denormal
// n 2^-24, and four operations fewer would do; but the product aligns denormals by their exponent
// field, and loses 3 bits.)  A block's scale multiplies what the product gives (keys) or the weight
// (values), in f32.
#include "kv_cache.h"

namespace tcrv {
namespace {

constexpr int kRows = 16;          // rows of a tile
constexpr int kWaves = 4;          // waves of a work-group, which share out a tile's tokens
constexpr int kStep = 32;          // tokens that a wave takes at a time
constexpr float kNone = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Weights are 2^(z - m + shift).  m follows the row's maximum only when that has risen by kSlack
// (2^4): a rescale of the output costs as much as the tile's products.  The shift keeps weight times
// value scale within f16's range and as high in it as the value scales seen so far let it be, by the
// top bits of their exponents: below 2^-11, 2^-7, 2, and whatever fp16 holds.
constexpr float kSlack = 4.0f;
constexpr int kLevels = 4;
__device__ __forceinline__ float shift_of(int level) {  // 2^4 2^shift scale <= 2^15
  return level == 0 ? 22.0f : level == 1 ? 18.0f : level == 2 ? 10.0f : -4.0f;
}
// the exponent bits that a scale of the level's range does not have
__device__ __forceinline__ uint32_t bits_over(int level) {
  return level == 0 ? 0x70007000u : level == 1 ? 0x60006000u : level == 2 ? 0x40004000u : 0u;
}

struct AttnArgs {
  const void *q;
  void *out;
  const uint8_t *cache;
  const int32_t *block_table, *first, *length;
  float *parts;  // workspace: [split][token][head][head_dim], then [split][token][head][2]
  size_t q_token, q_head, out_token, out_head;
  size_t table_stride, window;
  uint32_t pages, page_size, tokens, heads, share, tiles, max_added, max_length;
  uint32_t split_tokens, splits;
  float scale;
  int causal;
};

template <int n> struct Dwords {
  uint32_t v[n];
};

// n dwords (even) from a place aligned to as many bytes, at most 16
template <int n> __device__ __forceinline__ Dwords<n> load_dwords(const uint8_t *p) {
  Dwords<n> r;
  if constexpr (n % 4 == 0) {
#pragma unroll
    for (int i = 0; i < n / 4; ++i)
      *reinterpret_cast<u32x4 *>(r.v + 4 * i) = reinterpret_cast<const u32x4 *>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < n / 2; ++i)
      *reinterpret_cast<u32x2 *>(r.v + 2 * i) = reinterpret_cast<const u32x2 *>(p)[i];
  }
  return r;
}

__device__ __forceinline__ float half_of(const uint32_t *v, int i) {
  return fp16_bits_to_f32(v[i >> 1] >> (16 * (i & 1)) & 0xffffu);
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The quants in the lowest bits of a dword's halves, less 8; four dwords are an operand.
__device__ __forceinline__ uint32_t quants_of(uint32_t w) {
  const f16x2 v = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x64006400u);
  return __builtin_bit_cast(uint32_t, v + f16x2{-1032, -1032});
}
__device__ __forceinline__ f16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  u32x4 v = {quants_of(a), quants_of(b), quants_of(c), quants_of(d)};
  return __builtin_bit_cast(f16x8, v);
}

// Two values rounded to f16, and what the rounding left of them (kParts 2).  The rounded pair is
// hidden from the compiler's sight: it would form it a second time for the remainder, from the
// unrounded product in one step, and the two differ by a unit where the product lies near a tie.
template <int kParts>
__device__ __forceinline__ void split_pair(float x0, float x1, f16x8 (&part)[kParts], int i) {
  uint32_t hi = __builtin_bit_cast(
      uint32_t, f16x2{static_cast<_Float16>(x0), static_cast<_Float16>(x1)});
  asm("" : "+v"(hi));
  const f16x2 h = __builtin_bit_cast(f16x2, hi);
  part[0][i] = h[0];
  part[0][i + 1] = h[1];
  if constexpr (kParts == 2) {
    part[1][i] = static_cast<_Float16>(x0 - static_cast<float>(h[0]));
    part[1][i + 1] = static_cast<_Float16>(x1 - static_cast<float>(h[1]));
  }
}

// Over the four lanes of a row (lane, lane ^ 16, ^ 32, ^ 48).
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float row_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 tokens of one page and head, as a lane loads them: lane = 16 g + m holds quarter g of token m's
// keys, byte m of tokens 4 g .. 4 g + 3 of the values, and those four tokens' scales.
template <int NB> struct Tokens16 {
  Dwords<NB> k, v;
  Dwords<2 * NB> ks, vs;
};

template <int NB>
__device__ __forceinline__ void load_tokens(Tokens16<NB> &t, const uint8_t *head_at,
                                            const PageHead &lay, uint32_t place, int m, int g) {
  const uint32_t group = (place >> 2) + g;
  t.k = load_dwords<NB>(head_at + lay.key(NB, place + m, g, 0));
  t.ks = load_dwords<2 * NB>(head_at + lay.quants + group * NB * 8);
  t.v = load_dwords<NB>(head_at + lay.quants + lay.scales + (group * 16 + m) * NB * 4);
  t.vs = load_dwords<2 * NB>(head_at + 2 * lay.quants + lay.scales + group * NB * 8);
}

// What a lane holds of its row.  NP: the f16 parts that a query and a weight are split into.
template <int NB, int NP> struct Row {
  f16x8 q[NB][NP];      // the block's elements in the order in which the keys' nibbles come
  float unit;           // from the products' units to scores in powers of 2
  f32x4 o[2 * NB];      // 16 elements each: block o / 2, half o % 2
  float m, base, l;     // maximum so far; shift - maximum; this lane's sum of weights
  int level;            // of the shift
};

template <int NB, int NP, typename T>
__device__ __forceinline__ void load_row(Row<NB, NP> &row, const T *q, bool valid, int g,
                                         float scale) {
  float x[NB][8], top = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // pairs of nibbles (i, i + 4) of a dword: bytes 0 and 2 low, 0 and 2 high, then 1 and 3
      constexpr int kElement[8] = {0, 2, 16, 18, 1, 3, 17, 19};
      x[b][i] = valid ? widen(q[32 * b + 4 * g + kElement[i]]) : 0.0f;
      top = fmaxf(top, fabsf(x[b][i]));
    }
  }
  top = row_max(top);
  // an exact power of two brings the largest to 1 .. 2: no f16 part overflows, and what falls below
  // f16's range is 2^-24 of the largest.  The sign of `scale` goes into the queries, so that unit
  // >= 0 and a maximum of products is one of scores.
  int e = 0;
  if (top > 0.0f && top < __builtin_inff())
    (void)frexpf(top, &e);
  e = min(max(e - 1, -100), 100);
  const float into = ldexpf(scale < 0.0f ? -1.0f : 1.0f, -e);
  row.unit = ldexpf(fabsf(scale) * kLog2e, e);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      split_pair<NP>(x[b][i] * into, x[b][i + 1] * into, row.q[b], i);
  }
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i)
    row.o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  row.m = kNone;
  row.level = 0;
  row.base = shift_of(0);
  row.l = 0.0f;
}

template <int NB, int NP> __device__ __forceinline__ void rescale(Row<NB, NP> &row, float f) {
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i)
    row.o[i] *= f;
  row.l *= f;
}

// 32 tokens.  kEdge: not all of them are seen by all rows of the tile; token 4 g + r of half h is
// seen by this lane's row where bit 4 h + r of `seen` is set.
template <int NB, int NP, bool kEdge>
__device__ __forceinline__ void attend(Row<NB, NP> &row, Tokens16<NB> (&t)[2], uint32_t seen) {
  float z[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sum[4] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t w = t[h].k.v[b];
      const f16x8 keys = operand(w, w >> 4, w >> 8, w >> 12);
      f32x4 s = mfma(keys, row.q[b][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
      if constexpr (NP == 2)
        s = mfma(keys, row.q[b][1], s);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sum[r] = fmaf(s[r], half_of(t[h].ks.v + 2 * b, r), sum[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      z[4 * h + r] = kEdge && !(seen >> (4 * h + r) & 1u) ? kNone : sum[r];
  }
  uint32_t any = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      if constexpr (kEdge) {
        // what this lane's row does not see may hold anything, and a weight of 0 not cover it
        const uint32_t keep = (seen >> (4 * h + 2 * (i & 1)) & 1u ? 0xffffu : 0u) |
                              (seen >> (4 * h + 2 * (i & 1) + 1) & 1u ? 0xffff0000u : 0u);
        t[h].vs.v[i] &= keep;
      }
      any |= t[h].vs.v[i];
    }
  }
  if (__any((any & bits_over(row.level)) != 0)) {
    any |= __shfl_xor(any, 16);
    any |= __shfl_xor(any, 32);
    int level = row.level;
#pragma unroll
    for (int i = 0; i + 1 < kLevels; ++i)
      level = max(level, any & bits_over(i) ? i + 1 : 0);
    const float change = shift_of(level) - shift_of(row.level);
    rescale(row, exp2_fast(change));
    row.base += change;
    row.level = level;
  }
  float top = z[0];
#pragma unroll
  for (int i = 1; i < 8; ++i)
    top = fmaxf(top, z[i]);
  top = row_max(top) * row.unit;
  if (__any(top > row.m + kSlack)) {
    const float m = top > row.m + kSlack ? top : row.m;
    rescale(row, m == row.m ? 1.0f : exp2_fast(row.m - m));  // by 0 from no token to the first
    row.base = m == kNone ? row.base : shift_of(row.level) - m;
    row.m = m;
  }
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = exp2_fast(fmaf(z[i], row.unit, row.base));
    if (kEdge && !(seen >> i & 1u))
      p[i] = 0.0f;
    row.l += p[i];
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f16x8 w[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t *d = t[i >> 2].vs.v + 2 * b;
      split_pair<NP>(p[i] * half_of(d, i & 3), p[i + 1] * half_of(d, (i & 3) + 1), w, i);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = 4 * (2 * (b & 1) + half);
      const uint32_t *v0 = t[0].v.v + (b & ~1), *v1 = t[1].v.v + (b & ~1);
      const f16x8 values = operand(v0[0] >> at, v0[1] >> at, v1[0] >> at, v1[1] >> at);
#pragma unroll
      for (int s = 0; s < NP; ++s)
        row.o[2 * b + half] = mfma(values, w[s], row.o[2 * b + half]);
    }
  }
}

// One request's rows and what they see, from its lengths; the same in every kernel here.
struct Span {
  uint32_t first, added, rows;  // of its tokens in q; rows a kv head
  int64_t position0, length;    // of its first new token; tokens that may be read
  __device__ Span(const AttnArgs &a, uint32_t request) {
    const int64_t begin = max(a.first[request], 0), end = max(a.first[request + 1], 0);
    const int64_t last = min(end, static_cast<int64_t>(a.tokens));
    const int64_t whole = max(a.length[request], 0);
    first = static_cast<uint32_t>(begin);
    position0 = whole - max(end - begin, int64_t{0});
    added = static_cast<uint32_t>(
        min(max(last - begin, int64_t{0}), static_cast<int64_t>(a.max_added)));
    rows = added * a.share;
    length = min(min(whole, static_cast<int64_t>(a.max_length)),
                 static_cast<int64_t>(min(a.table_stride, size_t{0x7fffffff} / a.page_size)) *
                     a.page_size);
  }
  // tokens lo <= t < hi that the row of the i-th new token sees
  __device__ int64_t lo(const AttnArgs &a, uint32_t i) const {
    if (!a.window || a.window > static_cast<size_t>(0x7fffffff))
      return 0;
    return max(position0 + i + 1 - static_cast<int64_t>(a.window), int64_t{0});
  }
  __device__ int64_t hi(const AttnArgs &a, uint32_t i) const {
    return max(a.causal ? min(position0 + i + 1, length) : length, int64_t{0});
  }
};

template <int NB, int NP, typename T>
__global__ __launch_bounds__(kWaves * 64) void attn_q4_0_rows16(AttnArgs a) {
  constexpr int D = NB * 32;
  __shared__ f32x4 s_o[kWaves / 2][2 * NB][64];
  __shared__ float s_ml[kWaves / 2][2][64];
  const uint32_t request = blockIdx.x / a.tiles, tile = blockIdx.x % a.tiles;
  const uint32_t kv_head = blockIdx.y, split = blockIdx.z;
  const Span span(a, request);
  if (tile * kRows >= span.rows)
    return;
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row_at = tile * kRows + m;
  const bool valid = row_at < span.rows;
  const uint32_t i0 = tile * kRows / a.share;
  const uint32_t i1 = min(tile * kRows + kRows - 1, span.rows - 1) / a.share;
  // a row past the last one computes what the last one does, and nothing of it is kept
  const uint32_t mine = min(row_at, span.rows - 1);
  const uint32_t token = span.first + mine / a.share;
  const uint32_t head = kv_head * a.share + mine % a.share;
  // what the tile sees: its first row's first token to its last row's last
  const int64_t begin = span.lo(a, i0) / kStep * kStep + static_cast<int64_t>(split) * a.split_tokens;
  const int64_t end = min(span.hi(a, i1), begin + static_cast<int64_t>(a.split_tokens));
  if (split && begin >= end)
    return;
  const int64_t all_lo = span.lo(a, i1), all_hi = span.hi(a, i0);  // what every row sees
  const int64_t my_lo = span.lo(a, mine / a.share), my_hi = span.hi(a, mine / a.share);

  Row<NB, NP> row;
  load_row<NB, NP, T>(row,
                      static_cast<const T *>(a.q) + static_cast<size_t>(token) * a.q_token +
                          static_cast<size_t>(head) * a.q_head,
                      valid, g, a.scale);
  const PageHead lay(a.page_size, D);
  const uint32_t kv_heads = a.heads / a.share;
  const int32_t *const table = a.block_table + static_cast<size_t>(request) * a.table_stride;

  for (int64_t t0 = begin + wave * kStep; t0 < end; t0 += kWaves * kStep) {
    Tokens16<NB> t[2];
    bool there[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // 16 tokens lie in one page; past the end the first ones are read again and not seen
      const int64_t t1 = t0 + 16 * h < end ? t0 + 16 * h : t0;
      const uint32_t column = static_cast<uint32_t>(t1) / a.page_size;
      const uint32_t page = static_cast<uint32_t>(table[column]);
      there[h] = page < a.pages;
      load_tokens<NB>(t[h],
                      a.cache + (static_cast<size_t>(there[h] ? page : 0) * kv_heads + kv_head) *
                                    lay.bytes(),
                      lay, static_cast<uint32_t>(t1) - column * a.page_size, m, g);
    }
    if (t0 >= all_lo && t0 + kStep <= min(all_hi, end) && there[0] && there[1]) {
      attend<NB, NP, false>(row, t, 0);
    } else {
      uint32_t seen = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = t0 + 16 * (i >> 2) + 4 * g + (i & 3);
        seen |= at >= my_lo && at < min(my_hi, end) && there[i >> 2] ? 1u << i : 0u;
      }
      attend<NB, NP, true>(row, t, seen);
    }
  }

  // to plain units, then the waves' parts together: waves 2, 3 to 0, 1 and then 1 to 0
  row.l = row_sum(row.l);
  rescale(row, exp2_fast(-shift_of(row.level)));
#pragma unroll
  for (int half = kWaves / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)
        s_o[wave - half][i][lane] = row.o[i];
      s_ml[wave - half][0][lane] = row.m;
      s_ml[wave - half][1][lane] = row.l;
    }
    __syncthreads();
    if (wave < half) {
      const float m1 = s_ml[wave][0][lane], top = fmaxf(row.m, m1);
      const float f0 = row.m == top ? 1.0f : exp2_fast(row.m - top);
      const float f1 = m1 == top ? 1.0f : exp2_fast(m1 - top);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i)
        row.o[i] = row.o[i] * f0 + s_o[wave][i][lane] * f1;
      row.l = row.l * f0 + s_ml[wave][1][lane] * f1;
      row.m = top;
    }
    __syncthreads();
  }
  if (wave != 0 || !valid)
    return;
  if (a.splits > 1) {
    const size_t at = (static_cast<size_t>(split) * a.tokens + token) * a.heads + head;
    const size_t all = static_cast<size_t>(a.splits) * a.tokens * a.heads;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
      *reinterpret_cast<f32x4 *>(a.parts + at * D + 16 * i + 4 * g) = row.o[i];
    if (g == 0) {
      a.parts[all * D + 2 * at] = row.m;
      a.parts[all * D + 2 * at + 1] = row.l;
    }
    return;
  }
  const float inverse = row.l == 0.0f ? 0.0f : 1.0f / row.l;
  T *const out = static_cast<T *>(a.out) + static_cast<size_t>(token) * a.out_token +
                 static_cast<size_t>(head) * a.out_head;
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      v[r] = row.o[i][r] * inverse;
    store_values<4>(out + 16 * i + 4 * g, v, false);
  }
}

// The parts of a row together: a work-group a row, a thread an element.
template <typename T>
__global__ __launch_bounds__(256) void attn_q4_0_join(AttnArgs a, uint32_t head_dim) {
  const uint32_t request = blockIdx.x / a.max_added, i = blockIdx.x % a.max_added;
  const uint32_t head = blockIdx.y;
  const Span span(a, request);
  if (i >= span.added)
    return;
  const uint32_t token = span.first + i;
  // the tile's own range, as the kernel above cut it
  const uint32_t tile = (i * a.share + head % a.share) / kRows;
  const uint32_t i0 = tile * kRows / a.share;
  const uint32_t i1 = min(tile * kRows + kRows - 1, span.rows - 1) / a.share;
  const int64_t begin = span.lo(a, i0) / kStep * kStep;
  const int64_t tokens = span.hi(a, i1) - begin;
  const int64_t cut = a.split_tokens;
  const uint32_t splits =
      static_cast<uint32_t>(min(max((tokens + cut - 1) / cut, int64_t{1}),
                                static_cast<int64_t>(a.splits)));
  const size_t row = static_cast<size_t>(token) * a.heads + head;
  const size_t stride = static_cast<size_t>(a.tokens) * a.heads;
  const float *const ml = a.parts + a.splits * stride * head_dim;
  float m = kNone;
  for (uint32_t s = 0; s < splits; ++s)
    m = fmaxf(m, ml[2 * (s * stride + row)]);
  float o = 0.0f, l = 0.0f;
  const uint32_t e = threadIdx.x;
  for (uint32_t s = 0; s < splits; ++s) {
    const size_t at = s * stride + row;
    const float ms = ml[2 * at], f = ms == m ? 1.0f : exp2_fast(ms - m);
    l += ml[2 * at + 1] * f;
    o += a.parts[at * head_dim + e] * f;
  }
  static_cast<T *>(a.out)[static_cast<size_t>(token) * a.out_token +
                          static_cast<size_t>(head) * a.out_head + e] =
      narrow<T>(l == 0.0f ? 0.0f : o / l);
}

}  // namespace
}  // namespace tcrv

namespace {

using tcrv::AttnArgs;

struct Plan {
  size_t tiles, splits, split_tokens, workspace;
};

// Work-groups of one tile each; the tokens of few tiles are split, so that the card is filled, into
// parts of at least 256 tokens (two steps a wave).
Plan plan_of(size_t requests, size_t tokens, size_t max_added, size_t max_length, size_t heads,
             size_t kv_heads, size_t head_dim) {
  const size_t share = heads / kv_heads;
  Plan p;
  p.tiles = (max_added * share + tcrv::kRows - 1) / tcrv::kRows;
  const size_t groups = requests * p.tiles * kv_heads;
  const size_t most = (max_length + 255) / 256;
  size_t splits = groups >= 1024 ? 1 : (1024 + groups - 1) / groups;
  splits = splits > most ? most : splits;
  splits = splits < 1 ? 1 : splits;
  const size_t cut = ((max_length + splits - 1) / splits + 127) / 128 * 128;
  p.split_tokens = cut ? cut : 128;
  // a window's first step may begin 31 tokens before it
  p.splits = splits == 1 ? 1 : (max_length + 31 + p.split_tokens - 1) / p.split_tokens;
  if (p.splits == 1)
    p.split_tokens = max_length + 32;
  p.workspace = p.splits == 1 ? 0 : p.splits * tokens * heads * (head_dim + 2) * sizeof(float);
  return p;
}

template <int NB, int NP, typename T> void launch(const AttnArgs &a, dim3 grid, hipStream_t st) {
  tcrv::attn_q4_0_rows16<NB, NP, T><<<grid, dim3(tcrv::kWaves * 64), 0, st>>>(a);
}

template <int NP, typename T>
void launch_dim(const AttnArgs &a, size_t head_dim, dim3 grid, size_t requests, hipStream_t st) {
  switch (head_dim) {
  case 64:
    launch<2, NP, T>(a, grid, st);
    break;
  case 128:
    launch<4, NP, T>(a, grid, st);
    break;
  case 192:
    launch<6, NP, T>(a, grid, st);
    break;
  default:
    launch<8, NP, T>(a, grid, st);
    break;
  }
  if (a.splits > 1)
    tcrv::attn_q4_0_join<T>
        <<<dim3(static_cast<unsigned>(requests * a.max_added), a.heads),
           dim3(static_cast<unsigned>(head_dim)), 0, st>>>(a, static_cast<uint32_t>(head_dim));
}

bool attn_sizes_ok(size_t heads, size_t kv_heads, size_t head_dim) {
  return tcrv_host::cache_sizes_ok(16, kv_heads, head_dim) && heads != 0 &&
         heads <= tcrv_host::kMostHeads && heads % kv_heads == 0;
}

bool attn_too_large(size_t requests, size_t tokens, size_t max_added, size_t max_length,
                    size_t heads) {
  const size_t most = 0x7fffffffu;
  return requests > most || tokens > most || max_added > most || max_length > most - 4096 ||
         max_added * heads > most || requests * max_added > most ||
         requests * max_added * heads > (size_t{1} << 40);
}

}  // namespace

extern "C" {

size_t tcrv_hip_attn_q4_0_workspace_bytes(int elem, size_t requests, size_t tokens,
                                          size_t max_added, size_t max_length, size_t heads,
                                          size_t kv_heads, size_t head_dim) {
  if (!tcrv_host::float_elem_bytes(elem) || !attn_sizes_ok(heads, kv_heads, head_dim) ||
      attn_too_large(requests, tokens, max_added, max_length, heads) || !requests || !tokens ||
      !max_added)
    return 0;
  return plan_of(requests, tokens, max_added, max_length, heads, kv_heads, head_dim).workspace;
}

int tcrv_hip_attn_q4_0(int elem, const void *q, size_t q_token, size_t q_head,
                       const uint8_t *cache, size_t pages, size_t page_size,
                       const int32_t *block_table, size_t table_stride, const int32_t *first,
                       const int32_t *length, size_t requests, size_t tokens, size_t max_added,
                       size_t max_length, size_t heads, size_t kv_heads, size_t head_dim,
                       float scale, int causal, size_t window, void *out, size_t out_token,
                       size_t out_head, void *workspace, size_t workspace_bytes, void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem);
  if (!size)
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (!attn_sizes_ok(heads, kv_heads, head_dim) || !cache_sizes_ok(page_size, kv_heads, head_dim) ||
      !strides_ok(q_token, q_head, tokens, heads, head_dim) ||
      !strides_ok(out_token, out_head, tokens, heads, head_dim) || !(scale - scale == 0.0f))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (tokens == 0 || requests == 0 || max_added == 0)
    return TCRV_HIP_OK;
  if (!q || !out || !first || !length || (!cache && pages) || (!block_table && table_stride))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(q, size) || !aligned_to(out, size) || !aligned16(cache) ||
      !aligned4(block_table) || !aligned4(first) || !aligned4(length))
    return TCRV_HIP_ERR_MISALIGNED;
  if (attn_too_large(requests, tokens, max_added, max_length, heads) || pages > 0x7fffffffu ||
      table_stride > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (pages == 0)
    max_length = 0;  // nothing to read
  const Plan p = plan_of(requests, tokens, max_added, max_length, heads, kv_heads, head_dim);
  if (requests * p.tiles > 0x7fffffffu || p.splits > 65535u)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (p.workspace) {
    if (!workspace)
      return TCRV_HIP_ERR_NULL_POINTER;
    if (!aligned16(workspace))
      return TCRV_HIP_ERR_MISALIGNED;
    if (workspace_bytes < p.workspace)
      return TCRV_HIP_ERR_BAD_SIZE;
  }
  AttnArgs a{q,
             out,
             cache,
             block_table,
             first,
             length,
             static_cast<float *>(workspace),
             q_token,
             q_head,
             out_token,
             out_head,
             table_stride,
             window,
             static_cast<uint32_t>(pages),
             static_cast<uint32_t>(page_size),
             static_cast<uint32_t>(tokens),
             static_cast<uint32_t>(heads),
             static_cast<uint32_t>(heads / kv_heads),
             static_cast<uint32_t>(p.tiles),
             static_cast<uint32_t>(max_added),
             static_cast<uint32_t>(max_length),
             static_cast<uint32_t>(p.split_tokens),
             static_cast<uint32_t>(p.splits),
             scale,
             causal};
  const dim3 grid(static_cast<unsigned>(requests * p.tiles), static_cast<unsigned>(kv_heads),
                  static_cast<unsigned>(p.splits));
  hipStream_t st = as_stream(stream);
  switch (elem) {
  case TCRV_HIP_ELEM_F32:
    launch_dim<2, float>(a, head_dim, grid, requests, st);
    break;
  case TCRV_HIP_ELEM_F16:
    launch_dim<1, _Float16>(a, head_dim, grid, requests, st);
    break;
  default:
    launch_dim<1, tcrv::Bf16>(a, head_dim, grid, requests, st);
    break;
  }
  return launch_status();
}

}  // extern "C"

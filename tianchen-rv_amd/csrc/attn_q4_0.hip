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
// A dword of 8 quants becomes four operand registers.  4 bits n at the bottom of a half are the f16
// denormal n 2^-24: three shifts and four ands, and the offset -8 comes in with the keys' start value
// and goes out with the sums of the values' weights.  The product aligns denormals by their exponent
// field, which costs it 3 bits of 24: nothing beside 16-bit rows (one part), but f32 rows (two parts)
// take n over the bits of 1024.0, which is 1024 + n, and subtract 1032.
#include <algorithm>

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
  size_t table_stride;
  uint32_t table_tokens, window;  // tokens of a table's row; 0: no window
  uint32_t pages, page_size, tokens, heads, share, tiles, max_added, max_length;
  uint32_t split_tokens, splits;
  float scale;
  int causal;
  bool q_vec, out_vec;  // groups of 4 values lie on aligned places
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

// Four dwords, each with a quant in the lowest bits of its halves, as an operand: n - 8 for two parts,
// n 2^-24 for one.
template <int NP> struct Quants {
  uint32_t bits;  // of 1024.0, kept in a register: an instruction takes one constant
  __device__ Quants() : bits(0x64006400u) { asm("" : "+v"(bits)); }
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    if constexpr (NP == 1)
      return w & 0x000f000fu;
    const f16x2 v = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | bits);
    return __builtin_bit_cast(uint32_t, v + f16x2{-1032, -1032});
  }
  __device__ __forceinline__ f16x8 operator()(uint32_t a, uint32_t b, uint32_t c,
                                              uint32_t d) const {
    u32x4 v = {pair(a), pair(b), pair(c), pair(d)};
    return __builtin_bit_cast(f16x8, v);
  }
};

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

// A wave's ring of steps in LDS, filled by DMA (global_load_lds: no registers, and a step's bytes once,
// where lanes that load scales for themselves would take them sixteen times).  A stage: the keys'
// quants of both halves, the values', then the keys' scales and the values'.
constexpr int kStages = 3;
template <int NB> struct Stage {
  static constexpr int kQuants = NB * 256, kScales = NB * 32;  // of a half: 16 tokens
  static constexpr int kBytes = 4 * (kQuants + kScales);
  static constexpr int kLoads = (kBytes + 1023) / 1024;  // DMA instructions of 64 x 16 bytes
};

using lds_byte = __attribute__((address_space(3))) uint8_t;

// 16 bytes a lane from `from` into LDS at `to` + 16 lane, out of the compiler's sight, which would
// otherwise wait for all of them before any read of LDS.  M0 holds the place and is given back.
__device__ __forceinline__ void dma16(const uint8_t *from, uint32_t to) {
  uint32_t saved;
  asm volatile("s_mov_b32 %0, m0\n\t"
               "s_mov_b32 m0, %1\n\t"
               "s_nop 0\n\t"
               "global_load_lds_dwordx4 %2, off\n\t"
               "s_mov_b32 m0, %0"
               : "=&s"(saved)
               : "s"(to), "v"(from)
               : "memory");
}

template <int n> __device__ __forceinline__ void wait_loads() {
  static_assert(n < 64, "");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(n) : "memory");
}

// Until only the newest `steps` steps' loads are under way.
template <int kLoads> __device__ __forceinline__ void wait_steps(int steps) {
  if (steps >= 2)
    wait_loads<2 * kLoads>();
  else if (steps == 1)
    wait_loads<kLoads>();
  else
    wait_loads<0>();
}
static_assert(kStages <= 3, "wait_steps");

// The DMA of one step into the stage at LDS address `to`: at[h] is the place of half h's first token
// in its page's head, place[h] that token's number in the page.
template <int NB>
__device__ __forceinline__ void load_step(const uint8_t *const (&at)[2], const uint32_t (&place)[2],
                                          const PageHead &lay, uint32_t to, int lane) {
  using S = Stage<NB>;
#pragma unroll
  for (int i = 0; i < S::kLoads; ++i) {
    const int o = i * 1024 + lane * 16;
    // regions in their order: quants k0 k1 v0 v1, scales k0 k1 v0 v1
    const bool quants = o < 4 * S::kQuants;
    const int in_quants = o / S::kQuants, in_scales = (o - 4 * S::kQuants) / S::kScales;
    const int region = quants ? in_quants : in_scales;
    const int size = quants ? S::kQuants : S::kScales;
    const uint32_t within = (quants ? o : o - 4 * S::kQuants) - region * size;
    const bool values = region >= 2, second = region & 1;
    const uint32_t base = (values ? lay.quants + lay.scales : 0) + (quants ? 0 : lay.quants);
    const uint32_t p = second ? place[1] : place[0];
    const uint8_t *from = (second ? at[1] : at[0]) + (base + within + p * (quants ? NB * 16 : NB * 2));
    if (o < S::kBytes)
      dma16(from, to + i * 1024);
  }
}

template <int NB>
__device__ __forceinline__ void read_step(Tokens16<NB> (&t)[2], const uint8_t *stage, int m, int g) {
  using S = Stage<NB>;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    t[h].k = load_dwords<NB>(stage + h * S::kQuants + (m * 4 + g) * NB * 4);
    t[h].v = load_dwords<NB>(stage + (2 + h) * S::kQuants + (g * 16 + m) * NB * 4);
    t[h].ks = load_dwords<2 * NB>(stage + 4 * S::kQuants + h * S::kScales + g * NB * 8);
    t[h].vs = load_dwords<2 * NB>(stage + 4 * S::kQuants + (2 + h) * S::kScales + g * NB * 8);
  }
}

// What a lane holds of its row.  NP: the f16 parts that a query and a weight are split into.
template <int NB, int NP> struct Row {
  f16x8 q[NB][NP];      // the block's elements in the order in which the keys' nibbles come
  Quants<NP> quants;
  float unit;           // from the products' units to scores in powers of 2
  f32x4 o[2 * NB];      // 16 elements each: block o / 2, half o % 2
  // for one part, whose quants lack the -8: the keys' products start at -8 sum q, and the values'
  // take 8 times these sums of the weights off at the end
  f32x4 start[NP == 1 ? NB : 1], weights[NP == 1 ? NB : 1];
  float m, base, l;     // maximum so far; shift - maximum; this lane's sum of weights
  int level;            // of the shift
};

template <int NB, int NP, typename T>
__device__ __forceinline__ void load_row(Row<NB, NP> &row, const T *q, bool valid, bool vec, int g,
                                         float scale) {
  // pairs of nibbles (i, i + 4) of a dword: bytes 0 and 2 low, 0 and 2 high, then 1 and 3
  float x[NB][8], top = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float low[4], high[4];
    load_values<4>(low, q + 32 * b + 4 * g, vec);
    load_values<4>(high, q + 32 * b + 16 + 4 * g, vec);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[b][4 * i] = low[i];
      x[b][4 * i + 1] = low[i + 2];
      x[b][4 * i + 2] = high[i];
      x[b][4 * i + 3] = high[i + 2];
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[b][i] = valid ? x[b][i] : 0.0f;
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
  // not 0, so that a hidden token's score stays what it is
  row.unit = fmaxf(ldexpf(fabsf(scale) * kLog2e, NP == 1 ? e + 24 : e), 0x1p-100f);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      split_pair<NP>(x[b][i] * into, x[b][i + 1] * into, row.q[b], i);
      sum += static_cast<float>(row.q[b][0][i]) + static_cast<float>(row.q[b][0][i + 1]);
    }
    if constexpr (NP == 1) {
      const float c = row_sum(sum) * -0x1p-21f;
      row.start[b] = f32x4{c, c, c, c};
      row.weights[b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i)
    row.o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  row.m = kNone;
  row.level = NP == 1 ? 2 : 0;
  row.base = shift_of(row.level);
  row.l = 0.0f;
}

template <int NB, int NP> __device__ __forceinline__ void rescale(Row<NB, NP> &row, float f) {
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i)
    row.o[i] *= f;
  if constexpr (NP == 1) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
      row.weights[b] *= f;
  }
  row.l *= f;
}

// 32 tokens.  edge (the same in all lanes): not all of them are seen by all rows of the tile; token
// 4 g + r of half h is seen by this lane's row where bit 4 h + r of `seen` is set.
template <int NB, int NP>
__device__ __forceinline__ void attend(Row<NB, NP> &row, Tokens16<NB> (&t)[2], bool edge,
                                       uint32_t seen) {
  float z[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float sum[4] = {};
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const uint32_t w = t[h].k.v[b];
      const f16x8 keys = row.quants(w, w >> 4, w >> 8, w >> 12);
      f32x4 s;
      if constexpr (NP == 1) {
        s = mfma(keys, row.q[b][0], row.start[b]);
      } else {
        s = mfma(keys, row.q[b][0], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        s = mfma(keys, row.q[b][1], s);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sum[r] = fmaf(s[r], half_of(t[h].ks.v + 2 * b, r), sum[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      z[4 * h + r] = sum[r];
  }
  if (edge) {
    // what this lane's row does not see may hold anything, and a weight of 0 does not cover it
#pragma unroll
    for (int i = 0; i < 8; ++i)
      z[i] = seen >> i & 1u ? z[i] : kNone;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t keep = (seen >> (2 * i) & 1u ? 0xffffu : 0u) |
                            (seen >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        t[i >> 1].vs.v[2 * b + (i & 1)] &= keep;
    }
  }
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i)
    any |= t[0].vs.v[i] | t[1].vs.v[i];
  float top = z[0];
#pragma unroll
  for (int i = 1; i < 8; ++i)
    top = fmaxf(top, z[i]);
  top = row_max(top) * row.unit;
  if (__any(top > row.m + kSlack || (any & bits_over(row.level)) != 0)) {
    any |= __shfl_xor(any, 16);
    any |= __shfl_xor(any, 32);
    int level = row.level;
#pragma unroll
    for (int i = NP == 1 ? 2 : 0; i + 1 < kLevels; ++i)
      level = max(level, any & bits_over(i) ? i + 1 : 0);
    const float m = top > row.m + kSlack ? top : row.m;
    float f = exp2_fast(shift_of(level) - shift_of(row.level));
    if (m != row.m)
      f *= exp2_fast(row.m - m);  // by 0 from no token to the first
    rescale(row, f);
    row.level = level;
    row.m = m;
    row.base = shift_of(level) - (m == kNone ? 0.0f : m);
  }
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = exp2_fast(fmaf(z[i], row.unit, row.base));
    row.l += p[i];
  }
  f16x2 ph[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    ph[i] = f16x2{static_cast<_Float16>(p[2 * i]), static_cast<_Float16>(p[2 * i + 1])};
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f16x8 w[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t *d = t[i >> 2].vs.v + 2 * b;
      if constexpr (NP == 1) {
        const f16x2 x = ph[i / 2] * __builtin_bit_cast(f16x2, d[(i & 3) / 2]);
        w[0][i] = x[0];
        w[0][i + 1] = x[1];
      } else {
        split_pair<NP>(p[i] * half_of(d, i & 3), p[i + 1] * half_of(d, (i & 3) + 1), w, i);
      }
    }
    if constexpr (NP == 1)
      row.weights[b] = mfma(f16x8{1, 1, 1, 1, 1, 1, 1, 1}, w[0], row.weights[b]);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = 4 * (2 * (b & 1) + half);
      const uint32_t *v0 = t[0].v.v + (b & ~1), *v1 = t[1].v.v + (b & ~1);
      const f16x8 values = row.quants(v0[0] >> at, v0[1] >> at, v1[0] >> at, v1[1] >> at);
#pragma unroll
      for (int s = 0; s < NP; ++s)
        row.o[2 * b + half] = mfma(values, w[s], row.o[2 * b + half]);
    }
  }
}

// One request's rows and what they see, from its lengths; the same in every kernel here.
struct Span {
  uint32_t first, added, rows;  // of its tokens in q; rows a kv head
  int position0, length;        // of its first new token; tokens that may be read
  __device__ Span(const AttnArgs &a, uint32_t request) {
    const int begin = max(a.first[request], 0), end = max(a.first[request + 1], 0);
    const int whole = max(a.length[request], 0);
    first = static_cast<uint32_t>(begin);
    position0 = whole - max(end - begin, 0);
    added = static_cast<uint32_t>(
        min(max(min(end, static_cast<int>(a.tokens)) - begin, 0), static_cast<int>(a.max_added)));
    rows = added * a.share;
    length = min(min(whole, static_cast<int>(a.max_length)), static_cast<int>(a.table_tokens));
  }
  // tokens lo <= t < hi that the row of the i-th new token sees
  __device__ int lo(const AttnArgs &a, uint32_t i) const {
    return a.window ? max(position0 + static_cast<int>(i) + 1 - static_cast<int>(a.window), 0) : 0;
  }
  __device__ int hi(const AttnArgs &a, uint32_t i) const {
    return max(a.causal ? min(position0 + static_cast<int>(i) + 1, length) : length, 0);
  }
};

template <int NB, int NP, typename T>
__global__ __launch_bounds__(kWaves * 64, NB <= 4 ? 2 : 1) void attn_q4_0_rows16(AttnArgs a) {
  constexpr int D = NB * 32;
  // the waves' rings, and where they meet at the end
  __shared__ __align__(16) uint8_t s_ring[kWaves * kStages * Stage<NB>::kBytes];
  static_assert(sizeof(s_ring) >= kWaves / 2 * (2 * NB * 16 + 8) * 64, "");
  auto s_o = reinterpret_cast<f32x4(*)[2 * NB][64]>(s_ring);
  auto s_ml = reinterpret_cast<float(*)[2][64]>(s_ring + kWaves / 2 * 2 * NB * 64 * 16);
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
  const int begin = (span.lo(a, i0) & -kStep) + static_cast<int>(split * a.split_tokens);
  const int end = min(span.hi(a, i1), begin + static_cast<int>(a.split_tokens));
  if (split && begin >= end)
    return;
  const int all_lo = span.lo(a, i1), all_hi = min(span.hi(a, i0), end);  // what every row sees
  const int my_lo = span.lo(a, mine / a.share), my_hi = min(span.hi(a, mine / a.share), end);

  const PageHead lay(a.page_size, D);
  const uint32_t kv_heads = a.heads / a.share;
  const int32_t *const table = a.block_table + static_cast<size_t>(request) * a.table_stride;
  const size_t page_bytes = static_cast<size_t>(lay.bytes()) * kv_heads;
  const uint8_t *const head_at = a.cache + static_cast<size_t>(kv_head) * lay.bytes();

  // The wave's steps: tokens t_n = begin + 32 (wave + 4 n).  Lane 2 (n % 32) + h holds the page and the
  // place of step n's half h, for 32 steps at a time.
  const uint32_t from = static_cast<uint32_t>(begin) + wave * kStep;
  const uint32_t stop = static_cast<uint32_t>(max(end, begin));
  const int steps = from < stop ? static_cast<int>((stop - from - 1) / (kWaves * kStep)) + 1 : 0;
  uint32_t my_page = 0, my_place = 0;
  const auto look_up = [&](int n) {
    uint32_t t = from + (n + (lane >> 1)) * (kWaves * kStep) + (lane & 1) * 16;
    t = t < stop ? t : from;  // past the end the first ones are read again and not seen
    const uint32_t column = t / a.page_size;
    my_page = static_cast<uint32_t>(table[column]);
    my_place = t - column * a.page_size;
  };
  uint8_t *const ring = s_ring + wave * (kStages * Stage<NB>::kBytes);
  const uint32_t ring_at = static_cast<uint32_t>(
      __builtin_amdgcn_readfirstlane(static_cast<int>(reinterpret_cast<uintptr_t>(
          (lds_byte *)ring))));
  uint32_t there = 0;  // bit 2 (n % 16) + h: whether step n's half h lies in a page
  const auto load = [&](int n) {
    if (n % 32 == 0)
      look_up(n);
    const uint8_t *at[2];
    uint32_t place[2];
    uint32_t bits = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t page = __builtin_amdgcn_readlane(my_page, 2 * (n % 32) + h);
      place[h] = __builtin_amdgcn_readlane(my_place, 2 * (n % 32) + h);
      const bool in = page < a.pages;
      at[h] = head_at + (in ? page : 0) * page_bytes;
      bits |= in ? 1u << h : 0u;
    }
    there = (there & ~(3u << (2 * (n % 16)))) | bits << (2 * (n % 16));
    load_step<NB>(at, place, lay, ring_at + (n % kStages) * Stage<NB>::kBytes, lane);
  };
  for (int n = 0; n < kStages - 1; ++n)
    if (n < steps)
      load(n);
  Row<NB, NP> row;  // its loads behind those of the first steps, which take longer
  load_row<NB, NP, T>(row,
                      static_cast<const T *>(a.q) + static_cast<size_t>(token) * a.q_token +
                          static_cast<size_t>(head) * a.q_head,
                      valid, a.q_vec, g, a.scale);
  for (int n = 0; n < steps; ++n) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage before this one is read
    if (n + kStages - 1 < steps)
      load(n + kStages - 1);
    wait_steps<Stage<NB>::kLoads>(min(steps - 1 - n, kStages - 1));
    Tokens16<NB> t[2];
    read_step<NB>(t, ring + (n % kStages) * Stage<NB>::kBytes, m, g);
    const int t0 = static_cast<int>(from) + n * (kWaves * kStep);
    const uint32_t both = there >> (2 * (n % 16)) & 3u;
    const bool edge = t0 < all_lo || t0 + kStep > all_hi || both != 3u;
    uint32_t seen = 0;
    if (edge) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = t0 + 16 * (i >> 2) + 4 * g + (i & 3);
        seen |= at >= my_lo && at < my_hi && (both >> (i >> 2) & 1u) ? 1u << i : 0u;
      }
    }
    attend<NB, NP>(row, t, edge, seen);
  }

  // to plain units, then the waves' parts together: waves 2, 3 to 0, 1 and then 1 to 0
  row.l = row_sum(row.l);
  if constexpr (NP == 1) {
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
      row.o[i] = row.o[i] * 0x1p24f - 8.0f * row.weights[i / 2];
  }
  rescale(row, exp2_fast(-shift_of(row.level)));
  __syncthreads();
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
    store_values<4>(out + 16 * i + 4 * g, v, a.out_vec);
  }
}

// The parts of a row together: a work-group a row, a thread an element.  The parts' factors are formed
// side by side first, so that the sum's loads wait for nothing.
template <typename T>
__global__ __launch_bounds__(256) void attn_q4_0_join(AttnArgs a, uint32_t head_dim) {
  __shared__ float s_f[64], s_l[64], s_top;
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
  const int tokens = max(span.hi(a, i1) - (span.lo(a, i0) & -kStep), 1);
  const uint32_t splits = min((tokens + a.split_tokens - 1) / a.split_tokens, a.splits);
  const size_t row = static_cast<size_t>(token) * a.heads + head;
  const size_t stride = static_cast<size_t>(a.tokens) * a.heads;
  const float2 *const ml = reinterpret_cast<const float2 *>(a.parts + a.splits * stride * head_dim);
  const uint32_t e = threadIdx.x;
  float m = kNone, o = 0.0f, l = 0.0f;
  for (uint32_t s0 = 0; s0 < splits; s0 += 64) {  // 64 parts at a time
    const uint32_t n = min(splits - s0, 64u);
    float top = kNone;
    if (e < 64) {
      const float2 mine = e < n ? ml[(s0 + e) * stride + row] : make_float2(kNone, 0.0f);
      top = fmaxf(mine.x, m);
#pragma unroll
      for (int d = 1; d < 64; d <<= 1)
        top = fmaxf(top, __shfl_xor(top, d));
      s_f[e] = mine.x == top ? 1.0f : exp2_fast(mine.x - top);
      s_l[e] = mine.y;
      if (e == 0)
        s_top = top;
    }
    __syncthreads();
    top = s_top;
    const float f = m == top ? 1.0f : exp2_fast(m - top);
    o *= f;
    l *= f;
    m = top;
    const float *part = a.parts + (s0 * stride + row) * head_dim + e;
#pragma unroll 8
    for (uint32_t s = 0; s < n; ++s) {
      o += part[s * stride * head_dim] * s_f[s];
      l += s_l[s] * s_f[s];
    }
    __syncthreads();
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

// Work-groups of one tile each, two a CU; the tokens of fewer tiles are split into parts of at least
// 256 tokens (two steps a wave).  More parts cost more in work-groups' beginnings than they even out:
// decode over two contexts of 131072 75 us in 512 parts, 81 in 1024, 86 in 1536.
Plan plan_of(size_t requests, size_t tokens, size_t max_added, size_t max_length, size_t heads,
             size_t kv_heads, size_t head_dim) {
  const size_t share = heads / kv_heads;
  Plan p;
  p.tiles = (max_added * share + tcrv::kRows - 1) / tcrv::kRows;
  const size_t groups = requests * p.tiles * kv_heads;
  const size_t most = (max_length + 255) / 256;
  size_t splits = groups >= 512 ? 1 : (512 + groups - 1) / groups;
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
  return requests > most || tokens > most || max_added > most || max_length > (size_t{1} << 30) ||
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
             static_cast<uint32_t>(std::min(table_stride, size_t{0x7fffffff} / page_size) *
                                   page_size),
             window < 0x7fffffffu ? static_cast<uint32_t>(window) : 0,
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
             causal,
             groups_of_4(q, q_token, q_head, size),
             groups_of_4(out, out_token, out_head, size)};
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

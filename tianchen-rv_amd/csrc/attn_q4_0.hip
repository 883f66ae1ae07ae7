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
// denormal n 2^-24, those above them 16 n 2^-24: a shift and four ands, and the offset -8 comes in with
// the keys' start value and goes out with the sums of the values' weights.  The product aligns denormals by
// their exponent field, which costs it 3 bits of 24: nothing beside 16-bit rows (one part), but f32 rows
// (two parts) take n over the bits of 1024.0, which is 1024 + n, and subtract 1032.
//
// Few rows are bound by the read of the cache, 9/8 byte an element of a kv head and token, and the
// instructions that make operands of it: two contexts of 131072 tokens, bf16, 32 query and 8 kv heads of
// 128, 55 us and 6.7 for the join (264 MB, 4.8 TB/s without it); 64 requests of 1024 to 8192, f16, 78 and
// 5.2 (334 MB, 4.3 TB/s).  A wave reads its steps through an LDS ring of its own, so that
// no register waits for them.
#include <algorithm>
#include <type_traits>

#include "kv_cache.h"

namespace tcrv {
namespace {

using u16x2 = uint16_t __attribute__((ext_vector_type(2)));

constexpr int kRows = 16;          // rows of a tile
constexpr int kWaves = 4;          // waves of a work-group, which share out a tile's tokens
constexpr int kStep = 32;          // tokens that a wave takes at a time
constexpr float kNone = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

// Weights are 2^(z - m + shift).  m follows the row's maximum only when that has risen by kSlack
// (2^4): a rescale of the output costs as much as the tile's products.  The shift keeps weight times
// value scale within f16's range and as high in it as the value scales seen so far let it be: by the top
// bits of their exponents, which an OR of them all shows, below 2^-11, 2^-7 and 2, and from 2 on by the
// largest exponent itself.  One shift for all blocks of a row: beside a scale of 2^e, e >= 1, what a
// weight times a scale keeps ends at 2^(e - 35) of the largest weight.
constexpr float kSlack = 4.0f;
constexpr float kMostShift = 22.0f;
// 2^4 2^shift scale <= 2^15, for scales with the bits that `any` has, but for those of 2 and more
__device__ __forceinline__ float shift_of(uint32_t any) {
  const float shift = any & 0x70007000u ? 18.0f : kMostShift;
  return any & 0x60006000u ? 10.0f : shift;
}
// for those, by the field of the largest one's exponent (fp16's 2^0 is 15)
__device__ __forceinline__ float shift_of_exponent(uint32_t e) {
  return e < 16 ? kMostShift : 25.0f - static_cast<float>(e);
}
// the exponent bits that no scale of the shift's range has, or has to be looked at for
__device__ __forceinline__ uint32_t bits_over(float shift) {
  const uint32_t over = shift > 10.0f ? 0x60006000u : 0x40004000u;
  return shift > 18.0f ? 0x70007000u : over;
}

struct AttnArgs {
  const void *q;
  void *out;
  const uint8_t *cache;
  const int32_t *block_table, *first, *length;
  // workspace: outputs of parts of rows, [part][head_dim], then their maxima and sums, [part][2]; for
  // the kernel of many rows part [split][token][head], for that of few [work-group][2][row of a tile]
  float *parts;
  // workspace; for the kernel of few rows a work-group's tile that others end, for that of many the
  // tokens of a part
  uint4 *plan;
  size_t q_token, q_head, out_token, out_head;
  size_t table_stride;
  uint32_t table_tokens, window;  // tokens of a table's row; 0: no window
  uint32_t pages, page_size, tokens, heads, share, tiles, max_added, max_length;
  uint32_t few_least, few_most;  // the kernel at hand serves requests of so many rows a kv head
  uint32_t splits;  // many rows: parts of a tile, at most
  uint32_t requests, groups, unit_shift;  // few rows: work-groups that share out the work, 0: one a tile
  float scale;
  int causal;
  bool q_vec, out_vec;  // groups of 4 values lie on aligned places
  // of a tree of drafted tokens: which of the new ones a token sees, `words` of 64 bits each
  const uint64_t *ancestors;
  size_t words;
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

// Quants from the halves of dwords, as operands: n - 8 for two parts, n 2^-24 for one; kFours: of their
// bits 4 .. 7, which are left where they are, 16 times that.
template <int NP> struct Quants {
  uint32_t bits;  // of 1024.0, kept in a register: an instruction takes one constant
  __device__ Quants() : bits(0x64006400u) { asm("" : "+v"(bits)); }
  template <bool kFours> __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    constexpr uint32_t kMask = kFours ? 0x00f000f0u : 0x000f000fu;
    if constexpr (NP == 1)
      return w & kMask;
    constexpr int kOff = kFours ? -1152 : -1032;
    const f16x2 v = __builtin_bit_cast(f16x2, (w & kMask) | bits);
    return __builtin_bit_cast(uint32_t, v + f16x2{kOff, kOff});
  }
  // the keys of a dword; of one part the second and the fourth pair 16 times, which their queries make
  // up for: 5 instructions a dword for 7, 64 requests as above 87 -> 86 us
  __device__ __forceinline__ f16x8 keys(uint32_t w) const {
    u32x4 v = {pair<false>(w), pair<NP == 1>(NP == 1 ? w : w >> 4), pair<false>(w >> 8),
               pair<NP == 1>(w >> (NP == 1 ? 8 : 12))};
    return __builtin_bit_cast(f16x8, v);
  }
  // a pair of each of four dwords
  template <bool kFours>
  __device__ __forceinline__ f16x8 values(uint32_t a, uint32_t b, uint32_t c, uint32_t d) const {
    u32x4 v = {pair<kFours>(a), pair<kFours>(b), pair<kFours>(c), pair<kFours>(d)};
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
  if constexpr (kParts == 2)
    asm("" : "+v"(hi));
  const f16x2 h = __builtin_bit_cast(f16x2, hi);
  part[0][i] = h[0];
  part[0][i + 1] = h[1];
  if constexpr (kParts == 2) {
    part[1][i] = static_cast<_Float16>(x0 - static_cast<float>(h[0]));
    part[1][i + 1] = static_cast<_Float16>(x1 - static_cast<float>(h[1]));
  }
}

// Two f32 values times two fp16 ones, rounded once, to f16: the instructions that widen and narrow on the
// way, which the compiler does not form here (64 requests of 1024 to 8192 tokens, f16: 89 us by its own, 87
// so; 82 with the weight rounded first and the product again, which made the output's error 3.2e-4 of it
// where one rounding leaves 2.8e-4, its own 2.1e-4 among them).
__device__ __forceinline__ f16x2 times_pair(float x0, float x1, uint32_t d) {
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(r) : "v"(x0), "v"(d));
  asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]"
      : "+v"(r)
      : "v"(x1), "v"(d));
  return __builtin_bit_cast(f16x2, r);
}

// What rounding two f32 values to f16 left of them, as f16: exact but for f16's range.
__device__ __forceinline__ f16x2 left_of_pair(float x0, float x1, f16x2 rounded) {
  const uint32_t hi = __builtin_bit_cast(uint32_t, rounded);
  uint32_t r;
  asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(r) : "v"(x0), "v"(hi));
  asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]"
      : "+v"(r)
      : "v"(x1), "v"(hi));
  return __builtin_bit_cast(f16x2, r);
}

// A lane's own value and that of lane ^ 32 (lane ^ 16), in an order that both lanes share.
__device__ __forceinline__ float2 with_lane32(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t x = r[0], y = r[1];
  return make_float2(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float2 with_lane16(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t x = r[0], y = r[1];
  return make_float2(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float max_of(float2 v) { return fmaxf(v.x, v.y); }
__device__ __forceinline__ float sum_of(float2 v) { return v.x + v.y; }

// Over the four lanes of a row (lane, lane ^ 16, ^ 32, ^ 48).
__device__ __forceinline__ float row_max(float v) {
  return max_of(with_lane32(max_of(with_lane16(v))));
}
__device__ __forceinline__ float row_sum(float v) {
  return sum_of(with_lane32(sum_of(with_lane16(v))));
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

// The DMA of one step into the stage at LDS address `to`: at0 and at1 are the page's head that holds
// each half, place0 and place1 the number of its first token in the page.
template <int NB>
__device__ __forceinline__ void load_step(const uint8_t *at0, const uint8_t *at1, uint32_t place0,
                                          uint32_t place1, const PageHead &lay, uint32_t to,
                                          int lane) {
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
    const uint32_t p = second ? place1 : place0;
    const uint8_t *from = (second ? at1 : at0) + (base + within + p * (quants ? NB * 16 : NB * 2));
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
  f32x4 o[2 * NB];      // 16 elements each: block o / 2, half o % 2, the second ones 16 times
  // for one part, whose quants lack the -8: the keys' products start at -8 sum q, and the values'
  // take 8 times these sums of the weights off at the end
  f32x4 start[NP == 1 ? NB : 1], weights[NP == 1 ? NB : 1];
  float m, base, l;     // maximum so far; shift - maximum; this lane's sum of weights
  float shift;
  uint32_t over;        // bits_over(shift)
};

// An exact power of two, 2^-e, brings a row's largest element to 1 .. 2 (to 4 at the range's upper end,
// to less among f32's subnormals): no f16 part overflows, and what falls below f16's range is 2^-24 of the
// largest.  The sign of `scale` goes into the queries, so that the unit of the scores is positive and a
// maximum of products one of scores.
__device__ __forceinline__ int exponent_of(float top) {
  int e = 0;
  if (top > 0.0f && top < __builtin_inff())
    (void)frexpf(top, &e);
  return min(max(e - 1, -126), 126);  // either power is a normal f32
}

// |scale| log2 e 2^e.  Not 0, so that a hidden token's score stays what it is; nor infinite, where the
// scores may not be: products that differ do so by 2^-72 or more, and a unit of 2^126 as any larger one
// leaves a weight to the greatest alone.
__device__ __forceinline__ float unit_of(float scale, int e) {
  return fminf(fmaxf(ldexpf(fabsf(scale) * kLog2e, e), 0x1p-100f), 0x1p126f);
}

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
  const int e = exponent_of(top);
  const float into = ldexpf(scale < 0.0f ? -1.0f : 1.0f, -e);
  row.unit = unit_of(scale, NP == 1 ? e + 24 : e);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      // Quants::keys: a sixteenth, whose own range still ends 2^-20 below the largest
      const float fours = NP == 1 && (i & 2) ? 0x1p-4f : 1.0f;
      split_pair<NP>(x[b][i] * into * fours, x[b][i + 1] * into * fours, row.q[b], i);
      sum += (static_cast<float>(row.q[b][0][i]) + static_cast<float>(row.q[b][0][i + 1])) / fours;
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
  row.shift = row.base = kMostShift;
  row.over = bits_over(kMostShift);
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

// The largest exponent's field of a lane's value scales, of the finite ones alone where asked for: one more
// takes the others' to 0.
template <int NB, bool kFinite>
__device__ __forceinline__ uint32_t largest_exponent(const Tokens16<NB> (&t)[2]) {
  u16x2 most{};
#pragma unroll
  for (int i = 0; i < 4 * NB; ++i) {
    const uint32_t bits = t[i / (2 * NB)].vs.v[i % (2 * NB)] & 0x7c007c00u;
    u16x2 e = __builtin_bit_cast(u16x2, bits);
    if constexpr (kFinite)
      e = (e + u16x2{0x400, 0x400}) & u16x2{0x7c00, 0x7c00};
    most = __builtin_elementwise_max(most, e);
  }
  const uint32_t e = static_cast<uint32_t>(max(most[0], most[1])) >> 10;
  return kFinite ? max(e, 1u) - 1 : e;
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
      const f16x8 keys = row.quants.keys(w);
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
  float room = kMostShift;
  if (__builtin_expect(__any((any & 0x40004000u) != 0), 0)) {
    uint32_t e = largest_exponent<NB, false>(t);
    if (__any(e == 31))  // their block is lost, and is no reason to lose small weights in the others
      e = largest_exponent<NB, true>(t);
    room = shift_of_exponent(e);
    if (room >= row.shift)
      any &= ~0x40004000u;  // the shift is theirs already
  }
  float top = z[0];
#pragma unroll
  for (int i = 1; i < 8; ++i)
    top = fmaxf(top, z[i]);
  top = row_max(top) * row.unit;
  if (__any(top > row.m + kSlack || (any & row.over) != 0)) {
    any |= __shfl_xor(any, 16);
    any |= __shfl_xor(any, 32);
    const float shift = fminf(fminf(row.shift, shift_of(any)), -row_max(-room));
    const float m = top > row.m + kSlack ? top : row.m;
    float f = exp2_fast(shift - row.shift);
    if (m != row.m)
      f *= exp2_fast(row.m - m);  // by 0 from no token to the first
    rescale(row, f);
    row.shift = shift;
    row.over = bits_over(shift);
    row.m = m;
    row.base = shift - (m == kNone ? 0.0f : m);
  }
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = exp2_fast(fmaf(z[i], row.unit, row.base));
    row.l += p[i];
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f16x8 w[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t *d = t[i >> 2].vs.v + 2 * b;
      if constexpr (NP == 1) {
        const f16x2 x = times_pair(p[i], p[i + 1], d[(i & 3) / 2]);
        w[0][i] = x[0];
        w[0][i + 1] = x[1];
      } else {
        split_pair<NP>(p[i] * half_of(d, i & 3), p[i + 1] * half_of(d, (i & 3) + 1), w, i);
      }
    }
    if constexpr (NP == 1)
      row.weights[b] = mfma(f16x8{1, 1, 1, 1, 1, 1, 1, 1}, w[0], row.weights[b]);
    const int at = 8 * (b & 1);
    const uint32_t *v0 = t[0].v.v + (b & ~1), *v1 = t[1].v.v + (b & ~1);
    const uint32_t v[4] = {v0[0] >> at, v0[1] >> at, v1[0] >> at, v1[1] >> at};
    const f16x8 low = row.quants.template values<false>(v[0], v[1], v[2], v[3]);
    const f16x8 high = row.quants.template values<true>(v[0], v[1], v[2], v[3]);
#pragma unroll
    for (int s = 0; s < NP; ++s) {
      row.o[2 * b] = mfma(low, w[s], row.o[2 * b]);
      row.o[2 * b + 1] = mfma(high, w[s], row.o[2 * b + 1]);
    }
  }
}

// One request's rows and what they see, from its lengths; the same in every kernel here.
struct Span {
  uint32_t first, added, rows;  // of its tokens in q; rows a kv head
  int position0, length;        // of its first new token; tokens that may be read
  __device__ Span(const AttnArgs &a, uint32_t request)
      : Span(a, a.first[request], a.first[request + 1], a.length[request]) {}
  __device__ Span(const AttnArgs &a, int first0, int first1, int length0) {
    const int begin = max(first0, 0), end = max(first1, 0), whole = max(length0, 0);
    first = static_cast<uint32_t>(begin);
    position0 = whole - max(end - begin, 0);
    added = static_cast<uint32_t>(
        min(max(min(end, static_cast<int>(a.tokens)) - begin, 0), static_cast<int>(a.max_added)));
    rows = added * a.share;
    length = min(min(whole, static_cast<int>(a.max_length)), static_cast<int>(a.table_tokens));
  }
  // tokens lo <= t < hi that the row of the i-th new token sees; a position may lie before the first one,
  // from which a window of 2^31 - 2 would leave 32 bits
  __device__ int lo(const AttnArgs &a, uint32_t i) const {
    const int next = max(position0 + static_cast<int>(i) + 1, 0);
    return a.window ? max(next - static_cast<int>(a.window), 0) : 0;
  }
  __device__ int hi(const AttnArgs &a, uint32_t i) const {
    return max(a.causal ? min(position0 + static_cast<int>(i) + 1, length) : length, 0);
  }
};

// How the work-groups of the kernel below share out requests of all lengths.  The work is a line of
// units of 128 tokens (a step of each wave; more, by the power of two unit_shift, where their number
// would not fit 31 bits), a request's tiles after another's, a tile a kv head; every tile counts kStart
// more for its beginning and end (a fill and a drain of the loads, a meeting of the waves).  A work-group
// takes an equal stretch of the line, which may begin and end within a tile: at most two of its tiles are
// in parts.  Where the line is too short for that, a part of kLeast units or less is a stretch of its own.
// Against equal parts of the longest request, most of which the others leave empty: 64 requests of 1024
// to 8192 tokens 99 -> 82 us, of head_dim 256 129 -> 86 (48 requests), f32 and 32 of up to 4096 51 -> 43.
constexpr uint32_t kCus = 256, kStart = 3, kLeast = 2;
struct Work {
  uint32_t items, units;  // tiles times kv heads, units of each
  __device__ Work(const AttnArgs &a, const Span &span) : items(0), units(1) {
    if (!span.rows || span.rows < a.few_least || span.rows > a.few_most)
      return;
    items = (span.rows + kRows - 1) / kRows * (a.heads / a.share);
    const int seen = span.hi(a, span.added - 1) - begin(a, span);
    units = seen > 0 ? ((static_cast<uint32_t>(seen) - 1) >> (7 + a.unit_shift)) + 1 : 1;
  }
  // where a tile's units begin, for all tiles of a request
  static __device__ int begin(const AttnArgs &a, const Span &span) { return span.lo(a, 0) & -kStep; }
  __device__ Work(uint32_t items, uint32_t units) : items(items), units(units) {}
  // of the line, a tile; the units before its place x
  __device__ uint32_t parts() const { return (units + kLeast - 1) / kLeast; }
  __device__ uint32_t weight(bool small) const { return small ? parts() : units + kStart; }
  __device__ uint32_t before(bool small, uint32_t x) const {
    return small ? x * units / parts() : max(x, kStart) - kStart;
  }
};

// What the row of a tree's i-th node sees: cached tokens from `lo` on, and of the request's new ones, whose
// first is token `tree`, those from `lo` on whose bits are set.
struct Branch {
  const uint64_t *bits;
  int tree, lo;
  __device__ Branch() {}
  __device__ Branch(const AttnArgs &a, const Span &span, uint32_t i)
      : bits(a.ancestors + static_cast<size_t>(span.first + i) * a.words), tree(span.position0), lo(0) {
    if (!a.window)
      return;
    // of the bits up to the row's own, those that the window leaves: the last a.window
    uint32_t left = a.window;
    for (int w = static_cast<int>(i >> 6); w >= 0; --w) {
      uint64_t x = bits[w];
      if (w == static_cast<int>(i >> 6))
        x &= ~0ull >> (63 - (i & 63));
      const uint32_t n = __popcll(x);
      if (n >= left) {
        for (uint32_t drop = n - left; drop > 0; --drop)
          x &= x - 1;
        lo = tree + 64 * w + __builtin_ctzll(x);
        return;
      }
      left -= n;
    }
    // the others are cached tokens; a row without bits takes its own as one.  The first node may lie before
    // token 0, from where a window near 2^31 would leave 32 bits
    lo = max(max(tree, 0) - static_cast<int>(min(left, a.window - 1)), 0);
  }
  // which of tokens t .. t + 31 are cached ones or have their bits set
  __device__ uint32_t sees32(const AttnArgs &a, int t) const {
    const int before = tree - t;
    if (before >= 32)
      return ~0u;
    const uint32_t from = max(-before, 0), shift = from & 63;
    const size_t w = from >> 6;
    uint64_t x = w < a.words ? bits[w] >> shift : 0;
    if (shift > 32 && w + 1 < a.words)
      x |= bits[w + 1] << (64 - shift);
    const uint32_t some = static_cast<uint32_t>(x);
    return before > 0 ? some << before | ((1u << before) - 1) : some;
  }
};

template <int kControl, int kLines> __device__ __forceinline__ uint32_t dpp_add(uint32_t x) {
  return x + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kControl,
                                                               kLines, 0xf, false));
}

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ uint32_t lane_sums(uint32_t x) {
  x = dpp_add<0x111, 0xf>(x);  // the lane 1, 2, 4, 8 before, in a line of 16
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // the line before's last
  return dpp_add<0x143, 0xc>(x);
}

template <int kControl, int kLines> __device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kControl,
                                                                  kLines, 0xf, false)));
}

// The largest so far; the last lane has that of all.
__device__ __forceinline__ uint32_t lane_maxima(uint32_t x) {
  x = dpp_max<0x111, 0xf>(x);
  x = dpp_max<0x112, 0xf>(x);
  x = dpp_max<0x114, 0xf>(x);
  x = dpp_max<0x118, 0xf>(x);
  x = dpp_max<0x142, 0xa>(x);
  return dpp_max<0x143, 0xc>(x);
}

__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// kTree: a row sees of its request's new tokens its ancestors, by their bits, in the place of those before it.
template <int NB, int NP, typename T, bool kTree = false>
__global__ __launch_bounds__(kWaves * 64, NB <= 4 ? 2 : 1) void attn_q4_0_rows16(AttnArgs a) {
  constexpr int D = NB * 32;
  // the waves' rings, and where they meet at the end
  constexpr int kMeet = kWaves * (2 * NB * 16 + 8) * 64;
  constexpr int kRing = kWaves * kStages * Stage<NB>::kBytes;
  __shared__ __align__(16) uint8_t s_ring[kRing > kMeet ? kRing : kMeet];
  auto s_o = reinterpret_cast<f32x4(*)[2 * NB][64]>(s_ring);
  auto s_ml = reinterpret_cast<float2(*)[64]>(s_ring + kWaves * 2 * NB * 64 * 16);
  const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the line's length, and this work-group's stretch [x, line_end) of it
  const uint32_t kv_heads = a.heads / a.share;
  uint32_t x = blockIdx.x, line_end = x + 1, share = 1;
  bool small = false;
  // 64 requests at a time, one a lane: its lengths, its work, and where on the line that begins
  uint32_t base = 0, line_at = 0, lane_items = 0, lane_units = 0, lane_weight = 0, lane_from = 0;
  int lane_first0 = 0, lane_first1 = 0, lane_length = 0;
  const auto look = [&]() __attribute__((always_inline)) {
    const bool in = base + lane < a.requests;
    lane_first0 = in ? a.first[base + lane] : 0;
    lane_first1 = in ? a.first[base + lane + 1] : 0;
    lane_length = in ? a.length[base + lane] : 0;
    const Work work(a, Span(a, lane_first0, lane_first1, lane_length));
    lane_items = work.items;
    lane_units = work.units;
  };
  const auto lay_out = [&]() __attribute__((always_inline)) {
    lane_weight = lane_items * Work(lane_items, lane_units).weight(small);
    const uint32_t sum = lane_sums(lane_weight);
    lane_from = line_at + sum - lane_weight;
    line_at += lane_of(sum, 63);
  };
  if (a.groups) {
    uint32_t parts = 0, units = 0;
    for (;;) {
      look();
      parts += lane_items * Work(lane_items, lane_units).weight(true);
      units += lane_items * Work(lane_items, lane_units).weight(false);
      base += 64;
      if (base >= a.requests)
        break;
    }
    parts = lane_of(lane_sums(parts), 63);
    units = lane_of(lane_sums(units), 63);
    small = parts <= a.groups;
    share = small ? 1 : (units + a.groups - 1) / a.groups;
    x = blockIdx.x * share;
    line_end = min(x + share, small ? parts : units);
    base = 0;
    if (a.requests > 64)
      look();
    lay_out();
  }
  uint4 begun{};  // the tile that begins here and not ends: request, item, where it ends
  while (x < line_end) {
    Work work(0, 1);
    uint32_t request, item, at = 0;
    int first0, first1, length;
    if (a.groups) {
      const uint64_t here = __ballot(x - lane_from < lane_weight);
      if (!here) {
        base += 64;
        if (base >= a.requests)
          break;
        look();
        lay_out();
        continue;
      }
      const int owner = __builtin_ctzll(here);
      request = base + owner;
      first0 = static_cast<int>(lane_of(static_cast<uint32_t>(lane_first0), owner));
      first1 = static_cast<int>(lane_of(static_cast<uint32_t>(lane_first1), owner));
      length = static_cast<int>(lane_of(static_cast<uint32_t>(lane_length), owner));
      work.units = lane_of(lane_units, owner);
      const uint32_t place = x - lane_of(lane_from, owner);
      item = place / work.weight(small);
      at = place - item * work.weight(small);
    } else {
      request = x / (a.tiles * kv_heads);
      item = x - request * (a.tiles * kv_heads);
      first0 = a.first[request];
      first1 = a.first[request + 1];
      length = a.length[request];
    }
    const Span span(a, first0, first1, length);
    if (!a.groups) {
      work = Work(a, span);
      if (item >= work.items)
        return;
    }
    const uint32_t weight = work.weight(small);
    const uint32_t to = a.groups ? min(weight, at + line_end - x) : weight;
    const bool whole = at == 0 && to == weight;
    if (at == 0 && to != weight)
      begun = make_uint4(request, item, (x + weight - 1) / share, 0);
    x += to - at;
    const uint32_t tile = item / kv_heads, kv_head = item - tile * kv_heads;
    const uint32_t row_at = tile * kRows + m;
    const bool valid = row_at < span.rows;
    const uint32_t i0 = tile * kRows / a.share;
    const uint32_t i1 = min(tile * kRows + kRows - 1, span.rows - 1) / a.share;
    // a row past the last one computes what the last one does, and nothing of it is kept
    const uint32_t mine = min(row_at, span.rows - 1);
    const uint32_t token = span.first + mine / a.share;
    const uint32_t head = kv_head * a.share + mine % a.share;
    // the stretch's units, of what the request's first row's first token to its last row's last
    const uint32_t unit0 = work.before(small, at), unit1 = work.before(small, to);
    const int all = Work::begin(a, span), seen_end = span.hi(a, i1);
    const int begin = all + static_cast<int>(unit0 << (7 + a.unit_shift));
    const int end = whole ? seen_end
                          : min(seen_end, all + static_cast<int>(unit1 << (7 + a.unit_shift)));
    // what every row sees: of a tree cached tokens only, whatever the rows' depths, which are no more than
    // their numbers
    const int all_lo = span.lo(a, i1);
    const int all_hi = min(kTree ? span.position0 : span.hi(a, i0), end);
    Branch branch;
    int my_lo = span.lo(a, mine / a.share);
    if constexpr (kTree) {
      branch = Branch(a, span, mine / a.share);
      my_lo = branch.lo;
    }
    const int my_hi = min(span.hi(a, mine / a.share), end);

    const PageHead lay(a.page_size, D);
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
      const int from_lane = 2 * (n % 32);
      const uint32_t page0 = __builtin_amdgcn_readlane(my_page, from_lane);
      const uint32_t page1 = __builtin_amdgcn_readlane(my_page, from_lane + 1);
      const bool in0 = page0 < a.pages, in1 = page1 < a.pages;
      there = (there & ~(3u << (2 * (n % 16)))) |
              ((in0 ? 1u : 0u) | (in1 ? 2u : 0u)) << (2 * (n % 16));
      load_step<NB>(head_at + (in0 ? page0 : 0) * page_bytes,
                    head_at + (in1 ? page1 : 0) * page_bytes,
                    __builtin_amdgcn_readlane(my_place, from_lane),
                    __builtin_amdgcn_readlane(my_place, from_lane + 1), lay,
                    ring_at + (n % kStages) * Stage<NB>::kBytes, lane);
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
        const uint32_t bits = kTree ? branch.sees32(a, t0) : ~0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int in_step = 16 * (i >> 2) + 4 * g + (i & 3), at = t0 + in_step;
          seen |= at >= my_lo && at < my_hi && (both >> (i >> 2) & 1u) && (bits >> in_step & 1u)
                      ? 1u << i : 0u;
        }
      }
      attend<NB, NP>(row, t, edge, seen);
    }

    // to plain units, then the waves' parts together, a share of the elements a wave
    row.l = row_sum(row.l);
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      row.o[i] *= (NP == 1 ? 0x1p24f : 1.0f) * (i & 1 ? 0x1p-4f : 1.0f);
      if constexpr (NP == 1)
        row.o[i] -= 8.0f * row.weights[i / 2];
    }
    rescale(row, exp2_fast(-row.shift));
    __syncthreads();  // all have read their rings
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
      s_o[wave][i][lane] = row.o[i];
    s_ml[wave][lane] = make_float2(row.m, row.l);
    __syncthreads();
    float top = kNone, l = 0.0f, f[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      top = fmaxf(top, s_ml[w][lane].x);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float2 x = s_ml[w][lane];
      f[w] = x.x == top ? 1.0f : exp2_fast(x.x - top);
      l += x.y * f[w];
    }
    const float inverse = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
    const size_t part = (2 * blockIdx.x + (at == 0 ? 1 : 0)) * kRows + m;
    T *const out = static_cast<T *>(a.out) + static_cast<size_t>(token) * a.out_token +
                   static_cast<size_t>(head) * a.out_head;
#pragma unroll
    for (int k = 0; k < 2 * NB / kWaves; ++k) {
      const int i = wave * (2 * NB / kWaves) + k;
      f32x4 o{};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        o += s_o[w][i][lane] * f[w];
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[r] = o[r] * inverse;
      if (!valid)
        continue;
      if (!whole)
        store_values<4>(a.parts + part * D + 16 * i + 4 * g, v, true);
      else
        store_values<4>(out + 16 * i + 4 * g, v, a.out_vec);
    }
    if (!whole && valid && g == 0 && wave == 0) {
      const size_t all_parts = static_cast<size_t>(a.groups) * (2 * kRows);
      *reinterpret_cast<float2 *>(a.parts + all_parts * D + 2 * part) = make_float2(top, l);
    }
    __syncthreads();  // before the next stretch's steps are loaded over these
  }
  if (a.groups && threadIdx.x == 0)
    a.plan[blockIdx.x] = begun;
}

// ---------------------------------------------------------------------------
// Many rows: prompts.  A work-group takes its waves of 32 rows each through the tokens in steps, and
// the cache's values become f16 once for all of them: a step's quants are read 4-bit, scaled, and
// written to LDS in the order in which the matrix operands are read back, the next step's while this
// one is computed.  Both products are v_mfma_f32_32x32x16_f16, rows as columns as above, so that the
// weights again leave the first one where the second one reads them.
// A key is two f16 parts, which hold all of its 15 bits: a score's error would grow with the score.
// f16 and bf16 rows take values and weights as one part each; for f32 rows queries, values and weights
// are two parts as well, and a product three: the larger parts', and the mixed ones.  f16 rows take what the
// rounding left of every other 16 tokens' weights beside them: without it the prompt below is off by 3.11e-4
// of its output, more than 1.5 times the output's own rounding of 2.06e-4; with it by 2.90e-4, for 12 % of
// its time (other prompts 3 to 11 %); with that of all tokens' weights by 2.61e-4, for 24 %.  The rounding
// of bf16 outputs alone is 1.7e-3.
// A prompt of 4096, f16, 32 query and 8 kv heads of 128: 248 us back to back, 555 TFLOP/s (289 after 2 ms
// without work), a step of 64 tokens 3.8 us, of which the matrix instructions are 1.9 and the others and
// LDS 1.6 each: eight waves, two a SIMD, meet at every step and overlap no more.  Of head_dim 64 and
// f32 a step is 5 us; two work-groups a CU there (128 registers) spilled and took 74 us in 9 chunks where
// one took 74.
// ---------------------------------------------------------------------------
using f32x16 = float __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr float kTileShift = 10.0f;       // weights: 2^4 2^10, within f16
// A step's scales: some are 2 or more, finite ones 4096 or more, not finite.
constexpr uint32_t kKeyBig = 1, kValueBig = 2, kValueBad = 4, kKeyHuge = 16, kValueHuge = 32;
// The power of two that scales are multiplied with as they become operands, so that neither they nor the
// products with sixteenths leave f16's range: 15, 4 or 0.  With the first two a key's two parts hold all of
// it, whatever the other scales; without any they end at 2^-21 of an element.
__device__ __forceinline__ int up_of(uint32_t flags, uint32_t big, uint32_t huge) {
  const int up = flags & big ? 4 : 15;
  return flags & huge ? 0 : up;
}
// 2^e by its bits: in scalar registers where e is
__device__ __forceinline__ _Float16 power16(int e) {
  return __builtin_bit_cast(_Float16, static_cast<uint16_t>((15 + e) << 10));
}
__device__ __forceinline__ float power32(int e) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(127 + e) << 23);
}
// Scales by the fields of their exponents: the largest field, and the least that one is over 4096's (fields
// below that wrap past the others; infinity's and NaN's is 0x1000 over)
struct Exponents {
  u16x2 most{}, over{0xffff, 0xffff};
  __device__ __forceinline__ void add(uint32_t scales) {
    const u16x2 e = __builtin_bit_cast(u16x2, scales & 0x7c007c00u);
    most = __builtin_elementwise_max(most, e);
    over = __builtin_elementwise_min(over, static_cast<u16x2>(e - u16x2{0x6c00, 0x6c00}));
  }
  __device__ __forceinline__ bool bad() const { return max(most[0], most[1]) == 0x7c00; }
  __device__ __forceinline__ bool huge() const { return min(over[0], over[1]) < 0x1000; }
};
// bit kAbsentAt + i: the page of a step's i-th 16 tokens is not in the cache
constexpr uint32_t kAbsentAt = 8, kAbsent = 0xfu << kAbsentAt;

template <int NB, int NP> struct TileStep {
  // eight waves, two a SIMD, while a wave's queries and output fit 256 registers; a thread brings a
  // piece of a step, and two steps fit the LDS
  static constexpr int kWaves = NB == 8 || (NP == 2 && NB == 6) ? 4 : 8;
  static constexpr int kThreads = kWaves * 64, kTokens = kWaves * 8, kRows = kWaves * 32;
  // LDS rows: a token's keys, an element's values; 16 bytes apart from a multiple of the banks
  static constexpr int kKeyRow = NB * 64 + 16, kValueRow = kTokens * 2 + 16;
  static constexpr int kKeys = kTokens * kKeyRow, kValues = NB * 32 * kValueRow;  // of one part
  static constexpr int kBytes = 2 * kKeys + NP * kValues;
  static_assert(2 * kBytes <= 159 * 1024, "");
};

// What a thread carries from the cache to LDS: quarter g of a token's keys (the lower half of the
// threads) or byte m of four tokens' values, with their scales.
template <int NB> struct Raw {
  Dwords<NB> q;
  Dwords<2 * NB> d;  // keys: a scale a dword
};

// (n - 8) / 16 of the quants in the lowest bits of a dword's halves: over the bits of 64.0 they are
// sixteenths.  Times a scale below fp16's largest this stays below it.
__device__ __forceinline__ f16x2 sixteenths(uint32_t w) {
  const f16x2 v = __builtin_bit_cast(f16x2, (w & 0x000f000fu) | 0x54005400u);
  return v + f16x2{static_cast<_Float16>(-64.5f), static_cast<_Float16>(-64.5f)};
}

template <int NP> __device__ __forceinline__ void scaled(uint32_t w, f16x2 d, uint32_t (&part)[NP]) {
  const f16x2 n = sixteenths(w);
  const f16x2 hi = n * d;
  part[0] = __builtin_bit_cast(uint32_t, hi);
  if constexpr (NP == 2)
    part[1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n, d, -hi));
}

// What a work-group of the kernel below takes: a part of the steps of a tile.
struct Piece {
  uint32_t request, tile, kv_head, split;
  int part_tokens;  // 0: all of the tile's
};

// The w-th piece of the requests' work; false past the last.  Pieces have no gaps, since consecutive
// work-groups go to the XCDs and then to the groups of CUs in turn: where those of a request with fewer
// tiles than the longest one has ended at once, the working ones kept meeting in the same CUs.  The parts'
// length goes by the lengths of all requests: of the ways to cut the longest one into up to a.splits parts
// the one whose work-groups are done first, one a CU at a time; a part takes kPartFill steps' time more
// than its steps (a work-group's beginning and end, 9 us beside 3.4 a step), and the joining of parts
// kPartJoin.  Both together (us, f16, 8 kv heads of 128, against a grid of all tiles that there might be
// in equal parts of the longest request): 4 requests with up to 512 new tokens on up to 4096 224 -> 178, 20
// with up to 400 on 1000 147 -> 120, one with 256 on 8192 98 -> 83; 16 of 200 on 2000 with a window, f32,
// 2 kv heads of 64, 72 -> 50; one of 2048 alone, whose tiles see 1 to 32 steps, 100 -> 101.
constexpr uint32_t kPartFill = 5, kPartJoin = 2;

template <uint32_t kTileRows, uint32_t kTokens>
__device__ __forceinline__ bool find_piece(const AttnArgs &a, uint32_t w, int lane, Piece &piece) {
  const uint32_t kv_heads = a.heads / a.share;
  // of the lane's request: tiles times kv heads, the last tile's steps and the first one's
  uint32_t items = 0, steps = 1, steps0 = 1;
  const auto look = [&](uint32_t base) __attribute__((always_inline)) {
    items = 0;
    steps = steps0 = 1;
    if (base + lane < a.requests) {
      const Span span(a, base + lane);
      if (span.rows >= max(a.few_least, 1u) && span.rows <= a.few_most) {
        items = (span.rows + kTileRows - 1) / kTileRows * kv_heads;
        const int low = span.lo(a, 0) & -kStep, seen = span.hi(a, span.added - 1) - low;
        const int seen0 = span.hi(a, min(kTileRows - 1, span.rows - 1) / a.share) - low;
        steps = seen > 0 ? (seen - 1) / kTokens + 1 : 1;
        steps0 = seen0 > 0 ? (seen0 - 1) / kTokens + 1 : 1;
      }
    }
  };
  look(0);
  uint32_t part = 0;
  if (a.splits > 1) {
    uint32_t longest = 1;
    for (uint32_t base = 0;;) {
      longest = max(longest, items ? steps : 1);
      base += 64;
      if (base >= a.requests)
        break;
      look(base);
    }
    longest = lane_of(lane_maxima(longest), 63);
    // a way a lane: the longest in lane + 1 parts.  Numbers of work-groups as floats, near enough.
    part = (longest + lane) / (lane + 1);
    const float parts = 1.0f / static_cast<float>(part);
    float groups = 0.0f, work = 0.0f;
    bool alike = true;  // the tiles of each request, but for a quarter
    for (uint32_t base = 0; base < a.requests; base += 64) {
      if (a.requests > 64)
        look(base);
      for (uint32_t r = 0; r < min(a.requests - base, 64u); ++r) {
        const uint32_t last = lane_of(steps, r), first = lane_of(steps0, r);
        const float n = lane_of(items, r), mean = 0.5f * (last + first);
        const bool even = 4 * first >= 3 * last;
        alike = alike && (even || n == 0.0f);
        work += n * mean;
        groups += n * (even ? ceilf(last * parts - 0x1p-10f) : fmaxf(mean * parts + 0.5f, 1.0f));
      }
    }
    // alike they run in rounds of the CUs, else one after the other with the longest at the end, of which
    // 0.4 is not hidden (with none of it a prompt of 1024 takes 61 us for 48, 4 of 700 72 for 56; with all
    // of it the same, and one of 2048 105 for 95).  Alike from 3/4 on: from 9/10 1000 new tokens on 7192
    // take 279 for 219 and 4 times 512 on 3584 177 for 205; from 1/2 3 times 300 on 2700, f32, 99 for 127,
    // all else within 8 %
    const float one = static_cast<float>(part + kPartFill);
    const float cost = (lane ? kPartJoin : 0) +
                       (alike ? ceilf(groups * (1.0f / kCus)) * one
                              : fmaxf((work + kPartFill * groups) * (1.0f / kCus) + 0.4f * one, one));
    // the least of them, and of equal ones the fewest parts; costs are not negative: their bits order
    const uint32_t order =
        lane < static_cast<int>(a.splits) ? ~__builtin_bit_cast(uint32_t, cost) : 0;
    const uint64_t best = __ballot(order == lane_of(lane_maxima(order), 63));
    part = lane_of(part, __builtin_ctzll(best));
    if (a.requests > 64)
      look(0);
  }
  uint32_t before = 0;
  for (uint32_t base = 0;;) {
    const uint32_t pieces = items * (part ? (steps - 1) / part + 1 : 1);
    const uint32_t sum = lane_sums(pieces), from = before + sum - pieces;
    const uint64_t here = __ballot(w - from < pieces);
    if (here) {
      const int owner = __builtin_ctzll(here);
      const uint32_t of_tile = lane_of(items, owner), at = w - lane_of(from, owner);
      piece.request = base + owner;
      piece.split = at / of_tile;
      const uint32_t rest = at - piece.split * of_tile;
      // the last tiles of a prompt see the most tokens: they go first
      piece.tile = of_tile / kv_heads - 1 - rest / kv_heads;
      piece.kv_head = rest % kv_heads;
      piece.part_tokens = static_cast<int>(part * kTokens);
      return true;
    }
    before += lane_of(sum, 63);
    base += 64;
    if (base >= a.requests)
      return false;
    look(base);
  }
}

template <int NB, int NP, typename T, bool kTree = false>
__global__ __launch_bounds__((TileStep<NB, NP>::kThreads), (TileStep<NB, NP>::kWaves / 4)) void
attn_q4_0_tiles(AttnArgs a) {
  using S = TileStep<NB, NP>;
  constexpr int D = NB * 32, kTokens = S::kTokens;
  __shared__ __align__(16) uint8_t s_step[2][S::kBytes];
  __shared__ uint32_t s_flags[2][S::kWaves];
  __shared__ uint32_t s_bad[2][NB][kTokens / 32];
  Piece mine;
  if (!find_piece<S::kRows, kTokens>(a, blockIdx.x, threadIdx.x & 63, mine))
    return;
  const uint32_t kv_heads = a.heads / a.share, kv_head = mine.kv_head;
  const uint32_t tile = mine.tile, split = mine.split, request = mine.request;
  const Span span(a, request);
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, hh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = span.rows - 1;
  const uint32_t i0 = tile * S::kRows / a.share;
  const uint32_t i1 = min(tile * S::kRows + S::kRows - 1, last) / a.share;
  int begin = span.lo(a, kTree ? 0 : i0) & -kStep, end = span.hi(a, i1);
  bool cut = false;
  if (mine.part_tokens) {
    const int part = mine.part_tokens;
    if (threadIdx.x == 0)
      a.plan[0].x = static_cast<uint32_t>(part);  // the same from all
    cut = end - begin > part;
    if (split && (!cut || (end - begin - 1) / part < static_cast<int>(split)))
      return;
    begin += static_cast<int>(split) * part;
    end = min(end, begin + part);
  }
  const int steps = begin < end ? (end - begin + kTokens - 1) / kTokens : 0;

  // the wave's rows, and what they see
  const uint32_t row0 = tile * S::kRows + wave * 32;
  const uint32_t w0 = min(row0, last) / a.share, w1 = min(row0 + 31, last) / a.share;
  const int wave_lo = span.lo(a, kTree ? 0 : w0);
  const int wave_hi = row0 <= last ? min(span.hi(a, w1), end) : 0;
  const int all_lo = span.lo(a, w1);
  const int all_hi = min(kTree ? span.position0 : span.hi(a, w0), end);
  const uint32_t r = min(row0 + col, last);
  const bool valid = row0 + col <= last;
  Branch branch;
  int lo = span.lo(a, r / a.share);
  if constexpr (kTree) {
    branch = Branch(a, span, r / a.share);
    lo = branch.lo;
  }
  const int hi = min(span.hi(a, r / a.share), end);
  const uint32_t token = span.first + r / a.share, head = kv_head * a.share + r % a.share;

  // the thread's piece of a step
  const bool keys_piece = wave < S::kWaves / 2;
  const int piece = tid & (S::kThreads / 2 - 1);
  const int key_token = piece >> 2, g = piece & 3, value_group = piece >> 4, m = piece & 15;
  const int piece_token = keys_piece ? key_token : 4 * value_group;
  const PageHead lay(a.page_size, D);
  const int32_t *const table = a.block_table + static_cast<size_t>(request) * a.table_stride;
  const size_t page_bytes = static_cast<size_t>(lay.bytes()) * kv_heads;
  const uint8_t *const head_at = a.cache + static_cast<size_t>(kv_head) * lay.bytes();
  struct Place {
    uint32_t page, token;  // of the piece's first token
  };
  const auto find = [&](int n) __attribute__((always_inline)) {
    int t = begin + n * kTokens + piece_token;
    t = t < span.length ? t : begin;  // past the end something is read, and not used
    const uint32_t column = static_cast<uint32_t>(t) / a.page_size;
    return Place{static_cast<uint32_t>(table[column]),
                 static_cast<uint32_t>(t) - column * a.page_size};
  };
  Raw<NB> raw;
  bool absent = false;  // a wave of keys' pieces holds 16 tokens, which lie in one page
  const auto bring = [&](int n, const Place &p) __attribute__((always_inline)) {
    const bool in = p.page < a.pages;
    const uint8_t *at = head_at + (in ? p.page : 0) * page_bytes;
    if (keys_piece) {
      raw.q = load_dwords<NB>(at + lay.key(NB, p.token, g, 0));
#pragma unroll
      for (int b = 0; b < NB; ++b)
        raw.d.v[b] = *reinterpret_cast<const uint16_t *>(at + lay.key_scale(NB, p.token, b));
    } else {
      raw.q = load_dwords<NB>(at + lay.value(NB, p.token, m, 0));
      raw.d = load_dwords<2 * NB>(at + lay.value_scale(NB, p.token, 0));
    }
    // tokens that are not there: scales of 0, and no scores where it is their page that is missing (those
    // past the length are hidden by it)
    const int t0 = begin + n * kTokens;
    absent = false;
    if (t0 + kTokens > span.length || !__all(in)) {
      absent = __any(!in && t0 + piece_token < span.length);
      const int left = in ? span.length - (t0 + piece_token) : 0;
      if (keys_piece) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
          raw.d.v[b] = left > 0 ? raw.d.v[b] : 0;
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t keep =
              (left > 2 * i ? 0xffffu : 0u) | (left > 2 * i + 1 ? 0xffff0000u : 0u);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            raw.d.v[2 * b + i] &= keep;
        }
      }
    }
  };
  // what the step's scales are and which of its pages are missing, a word a wave
  const auto tell = [&](int n) __attribute__((always_inline)) {
    uint32_t any = 0, said = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i)
      any |= raw.d.v[i];
    if (keys_piece) {
      if (__any((any & 0x4000u) != 0)) {
        Exponents e;
#pragma unroll
        for (int b = 0; b < NB; ++b)
          e.add(raw.d.v[b]);
        said = kKeyBig | (__any(e.huge()) ? kKeyHuge : 0);
      }
      said |= absent ? 1u << (kAbsentAt + wave) : 0;
    } else {
#pragma unroll
      for (int i = NB; i < 2 * NB; ++i)
        any |= raw.d.v[i];
      if (__any((any & 0x40004000u) != 0)) {
        Exponents e;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
          e.add(raw.d.v[i]);
        said = kValueBig | (__any(e.bad()) ? kValueBad : 0) | (__any(e.huge()) ? kValueHuge : 0);
      }
    }
    if (lane == 0)
      s_flags[n & 1][wave] = said;
  };
  const auto told = [&](int n) __attribute__((always_inline)) {
    uint32_t f = 0;
#pragma unroll
    for (int w = 0; w < S::kWaves; ++w)
      f |= s_flags[n & 1][w];
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(f)));
  };
  const auto lay_out = [&](int n, uint32_t flags, int v_up) __attribute__((always_inline)) {
    if (flags & kValueBad) {  // infinite and NaN scales: noted, and taken out of the product
      if (tid < NB * (kTokens / 32))
        s_bad[n & 1][tid / (kTokens / 32)][tid % (kTokens / 32)] = 0;
      __syncthreads();
      if (!keys_piece) {
#pragma unroll
        for (int i = 0; i < 4 * NB; ++i) {
          const int token = 4 * value_group + (i & 3), s = 16 * (i & 1);
          uint32_t &w = raw.d.v[i >> 1];
          if ((w >> s & 0x7c00u) == 0x7c00u) {
            atomicOr(&s_bad[n & 1][i >> 2][token >> 5], 1u << (token & 31));
            w &= ~(0xffffu << s);
          }
        }
      }
    }
    uint8_t *const keys = s_step[n & 1], *const values = keys + 2 * S::kKeys;
    if (keys_piece) {
      const _Float16 f = power16(up_of(flags, kKeyBig, kKeyHuge));
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const _Float16 d = __builtin_bit_cast(_Float16, static_cast<uint16_t>(raw.d.v[b])) * f;
        uint32_t x[4][2];
        uint8_t *const to = keys + key_token * S::kKeyRow + (g * NB + b) * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          scaled<2>(raw.q.v[b] >> 4 * i, f16x2{d, d}, x[i]);
        *reinterpret_cast<u32x4 *>(to + S::kKeys) = u32x4{x[0][1], x[1][1], x[2][1], x[3][1]};
        *reinterpret_cast<u32x4 *>(to) = u32x4{x[0][0], x[1][0], x[2][0], x[3][0]};
      }
    } else {
      const _Float16 f = power16(v_up);
      // tokens in the order in which the weights lie: 4 of a lane's half, 4 of the other half's,
      // then 4 and 4 again
      const int at = 16 * (value_group >> 2) + 8 * (value_group & 1) + 2 * (value_group & 2);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const f16x2 d0 = __builtin_bit_cast(f16x2, raw.d.v[2 * b]) * f16x2{f, f};
        const f16x2 d1 = __builtin_bit_cast(f16x2, raw.d.v[2 * b + 1]) * f16x2{f, f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int shift = 4 * (2 * (b & 1) + half);
          uint32_t x[2][NP];
          scaled<NP>(raw.q.v[b & ~1] >> shift, d0, x[0]);
          scaled<NP>(raw.q.v[b | 1] >> shift, d1, x[1]);
#pragma unroll
          for (int s = 0; s < NP; ++s)
            *reinterpret_cast<u32x2 *>(values + s * S::kValues +
                                       (32 * b + 16 * half + m) * S::kValueRow + at * 2) =
                u32x2{x[0][s], x[1][s]};
        }
      }
    }
  };

  Place place{};
  if (steps > 0) {
    bring(0, find(0));
    place = find(1);
  }

  // The wave's rows by whole lines into LDS, where the steps will be: chunk c of a row, 8 elements,
  // holds those of keys' dword c.  (Fetched by the lanes that need them, 16 loads of 64 places each,
  // the rows take as long as four steps.)
  constexpr int kRowBytes = D * sizeof(T) + 16;
  static_assert(S::kWaves * 32 * kRowBytes <= 2 * S::kBytes, "");
  uint8_t *const rows_at = &s_step[0][0] + wave * 32 * kRowBytes;
  if (row0 <= last) {
    // where a row lies, from the lane that has it
    const size_t q_at = static_cast<size_t>(token) * a.q_token + static_cast<size_t>(head) * a.q_head;
    const int q_low = static_cast<int>(q_at), q_high = static_cast<int>(q_at >> 32);
#pragma unroll 8
    for (int first = 0; first < 32 * (D / 4); first += 64) {
      const int at = (first + lane) / (D / 4), e = 4 * ((first + lane) % (D / 4));
      const uint32_t low = static_cast<uint32_t>(__shfl(q_low, at));
      const uint32_t high = static_cast<uint32_t>(__shfl(q_high, at));
      const T *p = static_cast<const T *>(a.q) + (static_cast<size_t>(high) << 32 | low) + e;
      Values<T, 4> x;
      if (a.q_vec) {
        x = *reinterpret_cast<const Values<T, 4> *>(p);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x.v[k] = p[k];
      }
      *reinterpret_cast<Values<T, 4> *>(rows_at + at * kRowBytes + e * sizeof(T)) = x;
    }
  }
  // a wave reads only what it wrote
  f16x8 q[2 * NB][NP];
  float unit = 0.0f, sign = a.scale < 0.0f ? -1.0f : 1.0f, most = 0.0f;
  const T *const from = reinterpret_cast<const T *>(rows_at + col * kRowBytes);
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {  // the largest first, then the parts
    if (pass) {
      most = max_of(with_lane32(most));
      const int e = exponent_of(most);
      // an infinity makes the whole row NaN: its products with a key's two parts may be infinities of
      // one sign, a score that looks like that of a hidden token
      sign = most < __builtin_inff() ? ldexpf(sign, -e) : __builtin_nanf("");
      unit = unit_of(a.scale, e + 4);
    }
#pragma unroll
    for (int s = 0; s < 2 * NB; ++s) {
      const int c = 2 * s + hh;
      const T *at = from + 32 * (c % NB) + 4 * (c / NB);
      float low[4], high[4];
      load_values<4>(low, at, true);
      load_values<4>(high, at + 16, true);
      const float x[8] = {low[0], low[2], high[0], high[2], low[1], low[3], high[1], high[3]};
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        if (pass)
          split_pair<NP>(valid ? x[i] * sign : 0.0f, valid ? x[i + 1] * sign : 0.0f, q[s], i);
        else
          most = fmaxf(most, valid ? fmaxf(fabsf(x[i]), fabsf(x[i + 1])) : 0.0f);
      }
    }
  }
  f32x16 o[NB];
  float top = kNone, base = kTileShift, l = 0.0f;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    o[b] = f32x16{};

  uint32_t flags = 0;
  int v_up = 15;  // the least of the steps so far
  if (steps > 0) {
    tell(0);
    __syncthreads();  // and all have their queries
    flags = told(0);
    v_up = up_of(flags, kValueBig, kValueHuge);
    lay_out(0, flags, v_up);
    bring(1, place);
    place = find(2);
  }
  int was_up = v_up;
  // The keys' threads bring the next step in before they compute, the values' afterwards: of the two
  // waves of a SIMD one is at its matrix products while the other is not.
  const auto next_step = [&](int n) __attribute__((always_inline)) {
    lay_out(n + 1, flags, v_up);
    bring(n + 2, place);
    place = find(n + 3);
  };
  for (int n = 0; n < steps; ++n) {
    const uint32_t mine = flags;
    const int mine_up = v_up;
    if (n + 1 < steps)
      tell(n + 1);
    __syncthreads();  // this step is laid out, and the one before it read
    if (n + 1 < steps) {
      flags = told(n + 1);
      v_up = min(v_up, up_of(flags, kValueBig, kValueHuge));
      if (keys_piece)
        next_step(n);
    }
    const uint8_t *const keys = s_step[n & 1], *const values = keys + 2 * S::kKeys;
    if (mine_up != was_up) {
      const float f = power32(mine_up - was_up);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        o[b] *= f;
      was_up = mine_up;
    }
    const float u = unit * power32(-up_of(mine, kKeyBig, kKeyHuge));
    const int t0 = begin + n * kTokens;
    if (t0 < wave_hi && t0 + kTokens > wave_lo) {
      const bool edge = t0 < all_lo || t0 + kTokens > all_hi || (mine & kAbsent) != 0;
      // 32 tokens' scores
      const auto scores = [&](int sub) __attribute__((always_inline)) {
        __builtin_amdgcn_s_setprio(1);
        f32x16 z{};
        const uint8_t *const key = keys + (32 * sub + col) * S::kKeyRow + hh * 16;
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
          const f16x8 k0 = *reinterpret_cast<const f16x8 *>(key + s * 32);
          z = mfma32(k0, q[s][0], z);
          const f16x8 k1 = *reinterpret_cast<const f16x8 *>(key + S::kKeys + s * 32);
          z = mfma32(k1, q[s][0], z);
          if constexpr (NP == 2)
            z = mfma32(k0, q[s][1], z);
        }
        __builtin_amdgcn_s_setprio(0);
        return z;
      };
      // hides what the row does not see, and returns by how much a new maximum scales what is there
      const auto settle = [&](f32x16 &z, int sub) __attribute__((always_inline)) {
        if (edge) {
          // register i: token 8 (i / 4) + 4 hh + i % 4
          const int lo_at = lo - t0 - 32 * sub - 4 * hh;
          int hi_at[2];
#pragma unroll
          for (int i = 0; i < 2; ++i)
            hi_at[i] = mine >> (kAbsentAt + 2 * sub + i) & 1u ? 0 : hi - t0 - 32 * sub - 4 * hh;
          const uint32_t bits = kTree ? branch.sees32(a, t0 + 32 * sub) >> 4 * hh : ~0u;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int at = 8 * (i >> 2) + (i & 3);
            z[i] = at >= lo_at && at < hi_at[i >> 3] && (!kTree || (bits >> at & 1u)) ? z[i] : kNone;
          }
        }
        float high = z[0];
#pragma unroll
        for (int i = 1; i < 16; ++i)
          high = fmaxf(high, z[i]);
        high = max_of(with_lane32(high)) * u;
        float f = 1.0f;
        if (__any(high > top + kSlack)) {
          // by a power of two, which leaves the weights that wait for their product exact
          const bool up = high > top + kSlack;
          const float next = !up ? top : top == kNone ? high : top + ceilf(high - top);
          f = next == top ? 1.0f : exp2_fast(top - next);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            o[b] *= f;
          l *= f;
          top = next;
          base = kTileShift - (next == kNone ? 0.0f : next);
        }
        return f;
      };
      // left: of the second 16 tokens' weights, for f16 rows
      constexpr bool kLeft = std::is_same_v<T, _Float16>;
      const auto weigh = [&](const f32x16 &z, f16x8 (&w)[2][NP], f16x8 &left) {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = exp2_fast(fmaf(z[i], u, base)), p1 = exp2_fast(fmaf(z[i + 1], u, base));
          split_pair<NP>(p0, p1, w[i >> 3], i & 7);
          // one part: the sum of the rounded weights, so that a row of few tokens divides by what its
          // values were multiplied with
          if constexpr (NP == 1) {
            const f16x8 &x = w[i >> 3][0];
            const f16x2 rounded{x[i & 7], x[(i & 7) + 1]};
            l = __builtin_amdgcn_fdot2(rounded, f16x2{1, 1}, l, false);
            if (kLeft && i >= 8) {
              const f16x2 rest = left_of_pair(p0, p1, rounded);
              l = __builtin_amdgcn_fdot2(rest, f16x2{1, 1}, l, false);
              left[i & 7] = rest[0];
              left[(i & 7) + 1] = rest[1];
            }
          } else {
            l += p0 + p1;
          }
        }
      };
      const auto add_values = [&](const f16x8 (&w)[2][NP], const f16x8 &left, int sub) {
        const uint8_t *const value = values + col * S::kValueRow + (32 * sub + 8 * hh) * 2;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            f16x8 v[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p)
              v[p] = *reinterpret_cast<const f16x8 *>(value + p * S::kValues + b * 32 * S::kValueRow +
                                                      s * 32);
            o[b] = mfma32(v[0], w[s][0], o[b]);
            if (kLeft && s == 1)
              o[b] = mfma32(v[0], left, o[b]);
            if constexpr (NP == 2) {
              o[b] = mfma32(v[0], w[s][1], o[b]);
              o[b] = mfma32(v[1], w[s][0], o[b]);
            }
          }
        }
      };
      // The second 32 tokens' scores are formed between the first ones' exponentials, and the first
      // ones' output between the second ones': a wave's matrix instructions run beside its others only
      // where they alternate.
      f32x16 z0 = scores(0);
      (void)settle(z0, 0);
      f16x8 w0[2][NP], left0;
      if constexpr (kTokens == 32) {
        weigh(z0, w0, left0);
        add_values(w0, left0, 0);
      } else {
        f32x16 z1 = scores(1);
        weigh(z0, w0, left0);
        const float f = settle(z1, 1);
        if (__any(f != 1.0f)) {
          const _Float16 h = static_cast<_Float16>(f);
#pragma unroll
          for (int i = 0; i < 2 * NP; ++i)
            w0[i / NP][i % NP] *= h;
          if (kLeft)
            left0 *= h;
        }
        f16x8 w1[2][NP], left1;
        weigh(z1, w1, left1);
        add_values(w0, left0, 0);
        add_values(w1, left1, 1);
      }
      if (mine & kValueBad) {
        // a row that sees a value scale that is not finite is NaN in that block
#pragma unroll
        for (int sub = 0; sub < kTokens / 32; ++sub) {
          const int first = min(max(lo - t0 - 32 * sub, 0), 32);
          const int stop = min(max(hi - t0 - 32 * sub, 0), 32);
          uint32_t sees = static_cast<uint32_t>((1ull << stop) - (1ull << min(first, stop)));
          if constexpr (kTree)
            sees &= branch.sees32(a, t0 + 32 * sub);
#pragma unroll
          for (int b = 0; b < NB; ++b)
            o[b] += s_bad[n & 1][b][sub] & sees ? __builtin_nanf("") : 0.0f;
        }
      }
    }
    if (n + 1 < steps && !keys_piece)
      next_step(n);
  }

  if (row0 > last && cut)
    return;
  const float sum = sum_of(with_lane32(l));
  const float out_unit = power32(4 - was_up);
  if (cut) {
    if (!valid)
      return;
    const size_t at = (static_cast<size_t>(split) * a.tokens + token) * a.heads + head;
    const size_t all = static_cast<size_t>(a.splits) * a.tokens * a.heads;
    const float f = out_unit * exp2_fast(-kTileShift);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4 *>(a.parts + at * D + 32 * b + 8 * i + 4 * hh) =
            f32x4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]} * f;
    if (hh == 0) {
      a.parts[all * D + 2 * at] = top;
      a.parts[all * D + 2 * at + 1] = sum * exp2_fast(-kTileShift);
    }
    return;
  }
  // rows leave as they came, by whole lines through LDS
  __syncthreads();
  const float f = sum == 0.0f ? 0.0f : out_unit / sum;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {o[b][4 * i] * f, o[b][4 * i + 1] * f, o[b][4 * i + 2] * f,
                          o[b][4 * i + 3] * f};
      store_values<4>(reinterpret_cast<T *>(rows_at + col * kRowBytes) + 32 * b + 8 * i + 4 * hh, v,
                      true);
    }
  }
  const int rows = static_cast<int>(min(last + 1 - min(row0, last + 1), 32u));
  // where a row goes, from the lane that has had it
  const size_t out_at = static_cast<size_t>(token) * a.out_token + static_cast<size_t>(head) * a.out_head;
  const int out_low = static_cast<int>(out_at), out_high = static_cast<int>(out_at >> 32);
#pragma unroll
  for (int first = 0; first < 32 * (D / 4); first += 64) {
    const int i = first + lane, at = i / (D / 4), e = 4 * (i % (D / 4));
    const uint32_t low = static_cast<uint32_t>(__shfl(out_low, at & 31));
    const uint32_t high = static_cast<uint32_t>(__shfl(out_high, at & 31));
    if (at < rows) {
      T *p = static_cast<T *>(a.out) + (static_cast<size_t>(high) << 32 | low) + e;
      const Values<T, 4> x =
          *reinterpret_cast<const Values<T, 4> *>(rows_at + at * kRowBytes + e * sizeof(T));
      if (a.out_vec) {
        *reinterpret_cast<Values<T, 4> *>(p) = x;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          p[k] = x.v[k];
      }
    }
  }
}

// The stretches of a tile of attn_q4_0_rows16 together, of the tile that one of the kernel's work-groups has
// begun, 4 elements a thread, by groups of head_dim / 4 threads.  Of few stretches (as many as groups, up to 8)
// the groups take rows of the tile side by side, and the work-groups past them none; of more a work-group
// takes a row, and its groups share them out.  The same sums in the same order: a group that has one
// stretch leaves it as it is.  Latency bounds it, the launch and two dependent reads: 512 work-groups'
// tiles of 16 rows of 128, f16, 10.5 us a work-group a row and 5 side by side.
constexpr int kJoinThreads = 256;

template <typename T>
__global__ __launch_bounds__(kJoinThreads) void attn_q4_0_join_few(AttnArgs a, uint32_t head_dim) {
  __shared__ f32x4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  const uint4 begun = a.plan[blockIdx.x];
  if (begun.z == 0)
    return;
  const uint32_t stretches = begun.z - blockIdx.x + 1;
  const uint32_t per_head = head_dim / 4;
  const uint32_t groups = head_dim <= 64 ? 16 : head_dim <= 128 ? 8 : head_dim <= 192 ? 5 : 4;
  const bool side = stretches <= min(groups, 8u);
  if (side && blockIdx.y * groups >= kRows)
    return;
  const uint32_t kv_heads = a.heads / a.share, tile = begun.y / kv_heads;
  const uint32_t e = 4 * (threadIdx.x % per_head), group = threadIdx.x / per_head;
  // the first one's part is its work-group's second, the others' their first
  const auto at = [&](uint32_t s, uint32_t row) {
    return (2 * (blockIdx.x + s) + (s == 0 ? 1 : 0)) * static_cast<size_t>(kRows) + row;
  };
  const float2 *const ml = reinterpret_cast<const float2 *>(
      a.parts + static_cast<size_t>(a.groups) * (2 * kRows) * head_dim);
  const auto part = [&](uint32_t s, uint32_t row) {
    return *reinterpret_cast<const f32x4 *>(a.parts + at(s, row) * head_dim + e);
  };
  const auto put = [&](const Span &span, uint32_t row, const f32x4 &o, float l) {
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = l == 0.0f ? 0.0f : o[k] / l;
    const uint32_t token = span.first + row / a.share;
    const uint32_t head = (begun.y - tile * kv_heads) * a.share + row % a.share;
    store_values<4>(static_cast<T *>(a.out) + static_cast<size_t>(token) * a.out_token +
                        static_cast<size_t>(head) * a.out_head + e,
                    v, a.out_vec);
  };
  if (side) {
    const uint32_t row = blockIdx.y * groups + group;
    if (group >= groups || row >= kRows)
      return;
    // up to kMost stretches, read at once
    const auto beside = [&](auto most) __attribute__((always_inline)) {
      constexpr uint32_t kMost = decltype(most)::value;
      float2 x[kMost];
      f32x4 v[kMost];
#pragma unroll
      for (uint32_t s = 0; s < kMost; ++s) {
        const uint32_t from = min(s, stretches - 1);
        x[s] = ml[at(from, row)];
        v[s] = part(from, row);
      }
      const Span span(a, begun.x);
      if (tile * kRows + row >= span.rows)
        return;
      float top = kNone, l = 0.0f;
      f32x4 o{};
#pragma unroll
      for (uint32_t s = 0; s < kMost; ++s)
        top = fmaxf(top, x[s].x);
#pragma unroll
      for (uint32_t s = 0; s < kMost; ++s) {
        if (s < stretches) {
          const float f = x[s].x == top ? 1.0f : exp2_fast(x[s].x - top);
          l += x[s].y * f;
          o += v[s] * f;
        }
      }
      put(span, tile * kRows + row, o, l);
    };
    if (stretches <= 4)
      beside(std::integral_constant<uint32_t, 4>());
    else
      beside(std::integral_constant<uint32_t, 8>());
    return;
  }
  const Span span(a, begun.x);
  const uint32_t row = tile * kRows + blockIdx.y;
  if (row >= span.rows)
    return;
  float m = kNone, l = 0.0f;
  f32x4 o{};
  if (group < groups) {
#pragma unroll 4
    for (uint32_t s = group; s < stretches; s += groups) {
      // as they come: 16 bytes of output and 8 of its maximum and sum in one turn
      const float2 x = ml[at(s, blockIdx.y)];
      const f32x4 v = part(s, blockIdx.y);
      const float top = fmaxf(m, x.x);
      const float f = m == top ? 1.0f : exp2_fast(m - top), h = x.x == top ? 1.0f : exp2_fast(x.x - top);
      l = l * f + x.y * h;
      o = o * f + v * h;
      m = top;
    }
  }
  s_o[threadIdx.x] = o;
  s_ml[threadIdx.x] = make_float2(m, l);
  __syncthreads();
  if (group != 0)
    return;
  float top = kNone;
  for (uint32_t k = 0; k < groups; ++k)
    top = fmaxf(top, s_ml[k * per_head + threadIdx.x].x);
  o = f32x4{};
  l = 0.0f;
  for (uint32_t k = 0; k < groups; ++k) {
    const float2 x = s_ml[k * per_head + threadIdx.x];
    const float f = x.x == top ? 1.0f : exp2_fast(x.x - top);
    l += x.y * f;
    o += s_o[k * per_head + threadIdx.x] * f;
  }
  put(span, row, o, l);
}

// The parts of a row of attn_q4_0_tiles together, 4 elements a thread.  Of few parts a group of
// head_dim / 4 threads takes a head, and the groups of a work-group heads side by side; from kManyParts
// on the groups share out one head's parts.
constexpr int kManyParts = 8;

template <typename T, bool kShared>
__global__ __launch_bounds__(kJoinThreads) void attn_q4_0_join(AttnArgs a, uint32_t requests,
                                                               uint32_t head_dim,
                                                               uint32_t tile_rows) {
  __shared__ f32x4 s_o[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  const uint32_t token = blockIdx.x, lane = threadIdx.x & 63;
  // the token's request: the last one that begins at or before it, found 64 ways at a time
  uint32_t request = 0;
  for (uint32_t n = requests; n > 1;) {
    const uint32_t step = (n + 63) / 64, at = lane * step;
    const bool before = at < n && a.first[request + at] <= static_cast<int>(token);
    const uint32_t ways = __popcll(__ballot(before));
    const uint32_t skip = ways ? (ways - 1) * step : 0;
    request += skip;
    n = min(step, n - skip);
  }
  const Span span(a, request);
  if (token < span.first || token - span.first >= span.added || span.rows < a.few_least)
    return;
  const uint32_t per_head = head_dim / 4, groups = kJoinThreads / per_head;
  const uint32_t e = 4 * (threadIdx.x % per_head), group = threadIdx.x / per_head;
  const uint32_t head = kShared ? blockIdx.y : blockIdx.y * groups + group;
  const bool works = head < a.heads && group < groups;
  // the tile's own range, as the kernel cut it
  const uint32_t i = token - span.first;
  const uint32_t row0 = (i * a.share + head % a.share) / tile_rows * tile_rows;
  const uint32_t i0 = row0 / a.share, i1 = min(row0 + tile_rows - 1, span.rows - 1) / a.share;
  const int tokens = max(span.hi(a, i1) - (span.lo(a, a.ancestors ? 0 : i0) & -kStep), 1);
  const uint32_t part_tokens = a.plan[0].x;
  const uint32_t splits = min((tokens + part_tokens - 1) / part_tokens, a.splits);
  if (splits == 1)
    return;  // whole, of all rows of the tile
  const size_t row = static_cast<size_t>(token) * a.heads + head;
  const size_t stride = static_cast<size_t>(a.tokens) * a.heads;
  const float2 *const ml =
      reinterpret_cast<const float2 *>(a.parts + a.splits * stride * head_dim) + row;
  const float *const part = a.parts + row * head_dim + e;
  const uint32_t s0 = kShared ? group : 0, by = kShared ? groups : 1;
  float m = kNone, l = 0.0f;
  f32x4 o{};
  if (works) {
#pragma unroll 8
    for (uint32_t s = s0; s < splits; s += by)
      m = fmaxf(m, ml[s * stride].x);
#pragma unroll 8
    for (uint32_t s = s0; s < splits; s += by) {
      const float2 x = ml[s * stride];
      const float f = x.x == m ? 1.0f : exp2_fast(x.x - m);
      l += x.y * f;
      o += *reinterpret_cast<const f32x4 *>(part + s * stride * head_dim) * f;
    }
  }
  if constexpr (kShared) {
    s_o[threadIdx.x] = o;
    s_ml[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (group != 0)
      return;
    float top = kNone;
    for (uint32_t k = 0; k < groups; ++k)
      top = fmaxf(top, s_ml[k * per_head + threadIdx.x].x);
    o = f32x4{};
    l = 0.0f;
    for (uint32_t k = 0; k < groups; ++k) {
      const float2 x = s_ml[k * per_head + threadIdx.x];
      const float f = x.x == top ? 1.0f : exp2_fast(x.x - top);
      l += x.y * f;
      o += s_o[k * per_head + threadIdx.x] * f;
    }
  }
  if (!works)
    return;
  float v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = l == 0.0f ? 0.0f : o[k] / l;
  store_values<4>(static_cast<T *>(a.out) + static_cast<size_t>(token) * a.out_token +
                      static_cast<size_t>(head) * a.out_head + e,
                  v, a.out_vec);
}

}  // namespace
}  // namespace tcrv

namespace {

using tcrv::AttnArgs;

// Requests of few rows a kv head (decode, drafted tokens) run on attn_q4_0_rows16, the others (prompts
// and their chunks) on attn_q4_0_tiles; a call that may hold both launches both, and each leaves the
// other's requests alone.  Few is one tile of 16; in a call of nothing longer up to four of them, where
// the requests and kv heads alone are 64 work-groups and more (us, f16, head_dim 128, 8 kv heads, rows16
// / tiles: 64 requests of 4096 tokens and 8 new ones, 32 rows, 100 / 205, 32 of 2048 42 / 75, 8 of 4096
// and 16 new 42 / 56; one request of 4096 and 16 new 32 / 24; 8 of 4096 and 64 new, up to 256 rows, with
// the limit at 64 rows 77, at 16 63).
// Of trees up to four tiles, whatever else there is (us, f16, 8 kv heads of 128, rows16 / tiles: one request of
// 531 and 7 nodes, 28 rows, 12 / 19, of 4096 and 16 22 / 24, 8 of up to 4096 and 16 41 / 52, 64 of up to 4096
// and 8 98 / 295; f32, 8 of 4096 and 32, 128 rows, 77 / 63, bf16, 6 of 8192 and 64 126 / 87).
size_t few_rows_of(bool tree, size_t requests, size_t max_rows, size_t kv_heads) {
  return max_rows <= 64 && (tree || requests * kv_heads >= 64) ? 64 : 16;
}

// Rows of a tile of attn_q4_0_tiles.
size_t many_rows(int elem, size_t head_dim) {
  using tcrv::TileStep;
  const bool two = elem == TCRV_HIP_ELEM_F32;
  return head_dim <= 128   ? TileStep<4, 2>::kRows
         : head_dim == 192 ? (two ? TileStep<6, 2>::kRows : TileStep<6, 1>::kRows)
                           : TileStep<8, 1>::kRows;
}

// Work-groups of the kernel of few rows that the card runs at a time, by their registers and LDS: the
// shares of its work (64 requests of 1024 to 8192 tokens, f16, 32 query and 8 kv heads of 128: 112 us in
// 256 shares, 86 in 512, 96 in 768).
size_t most_groups(size_t head_dim) { return head_dim <= 128 ? 512 : 256; }

// Requests so short that a work-group a tile serves them sooner, where the tiles fill the card (us, whole
// tiles / shares, contexts from an eighth of the longest up: 64 requests of up to 1024 tokens 21 / 29,
// 2048 31 / 35, 4096 54 / 52, 8192 99 / 82; 128 of 2048 56 / 59, of 8192 155 / 146), in
// proportion where they do not (32 of 1024 17 / 23; f32, 32 of 4096 68 / 51; one of 531 15 / 14).
constexpr size_t kWholeTokens = 2560;

struct Plan {
  size_t tile_rows, tiles, workspace;
  size_t splits;                      // many rows
  size_t groups, unit_shift;          // few rows: shares (0: a tile a work-group)
  size_t launch;                      // work-groups
};

size_t parts_bytes(size_t parts, size_t head_dim) {
  return parts * (head_dim + 2) * sizeof(float);
}

// The shares of the kernel of few rows, for lengths up to max_length; none where no tile has enough
// tokens to be cut.
Plan few_plan(bool tree, size_t requests, size_t max_added, size_t max_length, size_t window,
              size_t heads, size_t kv_heads, size_t head_dim) {
  Plan p{};
  const size_t share = heads / kv_heads;
  const size_t rows =
      std::min(max_added * share, few_rows_of(tree, requests, max_added * share, kv_heads));
  p.tile_rows = tcrv::kRows;
  p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  const size_t items = requests * p.tiles * kv_heads;
  // what is seen begins at a multiple of 32; `window` is 0 where it does not bound that
  size_t seen = max_length + 31;
  if (window && window < seen)
    seen = std::min(seen, window + max_added + 31);
  const auto units = [&] { return std::max((seen - 1) >> (7 + p.unit_shift), size_t{0}) + 1; };
  while (items * (units() + tcrv::kStart) > 0x7fffffffu && units() > 1)
    ++p.unit_shift;
  const size_t parts = (units() + tcrv::kLeast - 1) / tcrv::kLeast;
  p.launch = items;
  const size_t most = most_groups(head_dim);
  if (parts > 1 && seen - 31 > kWholeTokens * std::min(items, most) / most) {
    p.launch = p.groups = std::min(items * parts, most);
    p.workspace = parts_bytes(p.groups * 2 * tcrv::kRows, head_dim) +
                  p.groups * sizeof(uint4);
  }
  return p;
}

// Tiles that may be fewer than kMostParts work-groups are cut into parts of 256 tokens and more, which the
// kernel chooses by the requests' lengths.
constexpr size_t kMostParts = 768, kLeastPart = 256;

Plan many_plan(int elem, size_t requests, size_t tokens, size_t max_added, size_t max_length,
               size_t window, size_t heads, size_t kv_heads, size_t head_dim) {
  const size_t share = heads / kv_heads;
  Plan p{};
  p.tile_rows = many_rows(elem, head_dim);
  p.tiles = (max_added * share + p.tile_rows - 1) / p.tile_rows;
  // as many tiles as full ones, and one that is not a request
  const size_t groups =
      std::min(requests * p.tiles, tokens * share / p.tile_rows + requests) * kv_heads;
  const auto parts_of = [&](size_t seen) {
    const size_t most = std::max((seen + kLeastPart - 1) / kLeastPart, size_t{1});
    return std::min(std::min(std::max(kMostParts / groups, size_t{1}), most), size_t{64});
  };
  // what a tile sees begins at a multiple of 32; `window` is 0 where it does not bound that.  A tree's tile also
  // sees from its request's first node's window on: its parts, no more than these, are longer then
  size_t seen = max_length + 31;
  if (window && window < seen)
    seen = std::min(seen, window + p.tile_rows / share + 34);
  p.splits = parts_of(seen);
  p.launch = groups * p.splits;
  // for any window: a smaller one has no more parts
  const size_t most = parts_of(max_length + 31);
  p.workspace = most == 1 ? 0 : sizeof(uint4) + parts_bytes(most * tokens * heads, head_dim);
  return p;
}

// Which of the two kernels a call launches, and the rows up to which the first serves.
struct Kernels {
  bool few, many;
  size_t few_rows;
};
Kernels kernels_of(bool tree, size_t requests, size_t tokens, size_t max_added, size_t heads,
                   size_t kv_heads) {
  const size_t rows = max_added * (heads / kv_heads);
  const size_t few = few_rows_of(tree, requests, rows, kv_heads);
  if (rows <= few)
    return {true, false, few};
  // one request, or all as long as the longest: none is short
  return {requests > 1 && tokens < requests * max_added, true, few};
}

template <int NP, typename T, bool kTree>
void launch_rows16(const AttnArgs &a, size_t head_dim, unsigned groups, hipStream_t st) {
  const dim3 grid(groups), block(tcrv::kWaves * 64);
  switch (head_dim) {
  case 64:
    tcrv::attn_q4_0_rows16<2, NP, T, kTree><<<grid, block, 0, st>>>(a);
    break;
  case 128:
    tcrv::attn_q4_0_rows16<4, NP, T, kTree><<<grid, block, 0, st>>>(a);
    break;
  case 192:
    tcrv::attn_q4_0_rows16<6, NP, T, kTree><<<grid, block, 0, st>>>(a);
    break;
  default:
    tcrv::attn_q4_0_rows16<8, NP, T, kTree><<<grid, block, 0, st>>>(a);
    break;
  }
}

template <int NB, int NP, typename T, bool kTree>
void launch_tiles(const AttnArgs &a, dim3 grid, hipStream_t st) {
  tcrv::attn_q4_0_tiles<NB, NP, T, kTree><<<grid, dim3(tcrv::TileStep<NB, NP>::kThreads), 0, st>>>(a);
}

template <int NP, typename T, bool kTree>
void launch_tiles(const AttnArgs &a, size_t head_dim, dim3 grid, hipStream_t st) {
  switch (head_dim) {
  case 64:
    launch_tiles<2, NP, T, kTree>(a, grid, st);
    break;
  case 128:
    launch_tiles<4, NP, T, kTree>(a, grid, st);
    break;
  case 192:
    launch_tiles<6, NP, T, kTree>(a, grid, st);
    break;
  default:
    launch_tiles<8, NP, T, kTree>(a, grid, st);
    break;
  }
}

template <int NP, typename T, bool kTree>
void launch_all(AttnArgs a, Kernels k, const Plan &few, const Plan &many, size_t head_dim,
                size_t requests, hipStream_t st) {
  const unsigned n = static_cast<unsigned>(requests);
  float *const workspace = a.parts;
  const uint32_t few_most = !k.few ? 0 : k.many ? static_cast<uint32_t>(k.few_rows) : 0xffffffffu;
  const uint32_t dim = static_cast<uint32_t>(head_dim);
  const dim3 join_block(tcrv::kJoinThreads);
  a.requests = n;
  if (k.few) {
    a.groups = static_cast<uint32_t>(few.groups);
    a.unit_shift = static_cast<uint32_t>(few.unit_shift);
    a.tiles = static_cast<uint32_t>(few.tiles);
    a.plan = reinterpret_cast<uint4 *>(workspace);
    a.parts = workspace + few.groups * (sizeof(uint4) / sizeof(float));
    a.few_least = 0;
    a.few_most = few_most;
    launch_rows16<NP, T, kTree>(a, head_dim, static_cast<unsigned>(few.launch), st);
    if (few.groups) {
      const size_t rows = std::min(static_cast<size_t>(a.max_added) * a.share, few.tile_rows);
      tcrv::attn_q4_0_join_few<T>
          <<<dim3(a.groups, static_cast<unsigned>(rows)), join_block, 0, st>>>(a, dim);
    }
  }
  if (k.many) {
    a.plan = reinterpret_cast<uint4 *>(workspace + (k.few ? few.workspace / sizeof(float) : 0));
    a.parts = reinterpret_cast<float *>(a.plan + 1);
    a.tiles = static_cast<uint32_t>(many.tiles);
    a.splits = static_cast<uint32_t>(many.splits);
    a.few_least = few_most ? few_most + 1 : 0;
    a.few_most = 0xffffffffu;
    launch_tiles<NP, T, kTree>(a, head_dim, dim3(static_cast<unsigned>(many.launch)), st);
    if (many.splits > 1) {
      const uint32_t tile_rows = static_cast<uint32_t>(many.tile_rows);
      const uint32_t groups = tcrv::kJoinThreads / (dim / 4);
      // shared out while the rows alone are few work-groups
      if (many.splits >= tcrv::kManyParts && static_cast<size_t>(a.tokens) * a.heads <= 4096)
        tcrv::attn_q4_0_join<T, true>
            <<<dim3(a.tokens, a.heads), join_block, 0, st>>>(a, n, dim, tile_rows);
      else
        tcrv::attn_q4_0_join<T, false>
            <<<dim3(a.tokens, (a.heads + groups - 1) / groups), join_block, 0, st>>>(a, n, dim,
                                                                                    tile_rows);
    }
  }
}

bool attn_sizes_ok(size_t heads, size_t kv_heads, size_t head_dim) {
  return tcrv_host::cache_sizes_ok(16, kv_heads, head_dim) && heads != 0 &&
         heads <= tcrv_host::kMostHeads && heads % kv_heads == 0;
}

bool attn_too_large(size_t requests, size_t tokens, size_t max_added, size_t max_length,
                    size_t heads) {
  const size_t most = 0x7fffffffu;
  return requests > most || tokens > tcrv_host::kMostTokens || max_added > most ||
         max_length > (size_t{1} << 30) ||
         max_added * heads > most || requests * max_added > most ||
         requests * max_added * heads > (size_t{1} << 40);
}

size_t workspace_bytes_of(bool tree, int elem, size_t requests, size_t tokens, size_t max_added,
                          size_t max_length, size_t heads, size_t kv_heads, size_t head_dim) {
  if (!tcrv_host::float_elem_bytes(elem) || !attn_sizes_ok(heads, kv_heads, head_dim) ||
      attn_too_large(requests, tokens, max_added, max_length, heads) || !requests || !tokens ||
      !max_added)
    return 0;
  const Kernels k = kernels_of(tree, requests, tokens, max_added, heads, kv_heads);
  size_t need = 0;
  for (const bool few : {true, false})
    if (few ? k.few : k.many)
      need += (few ? few_plan(tree, requests, max_added, max_length, 0, heads, kv_heads, head_dim)
                   : many_plan(elem, requests, tokens, max_added, max_length, 0, heads, kv_heads, head_dim))
                  .workspace;
  return need;
}

// kTree: the entry of drafted tokens.
template <bool kTree>
int attend(int elem, const void *q, size_t q_token, size_t q_head, const uint8_t *cache, size_t pages,
           size_t page_size, const int32_t *block_table, size_t table_stride, const int32_t *first,
           const int32_t *length, const uint64_t *ancestors, size_t words, size_t requests,
           size_t tokens, size_t max_added, size_t max_length, size_t heads, size_t kv_heads,
           size_t head_dim, float scale, int causal, size_t window, void *out, size_t out_token,
           size_t out_head, void *workspace, size_t workspace_bytes, void *stream) {
  constexpr bool tree = kTree;
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
  if (!q || !out || !first || !length || (!cache && pages) || (!block_table && table_stride) ||
      (tree && !ancestors))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(ancestors, 8) || !aligned_to(q, size) || !aligned_to(out, size) || !aligned16(cache) ||
      !aligned4(block_table) || !aligned4(first) || !aligned4(length))
    return TCRV_HIP_ERR_MISALIGNED;
  if (attn_too_large(requests, tokens, max_added, max_length, heads) || pages > 0x7fffffffu ||
      table_stride > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (!rows_apart(out_token, out_head, tokens, heads, head_dim) ||
      (tree && words < (max_added + 63) / 64))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (pages == 0)
    max_length = 0;  // nothing to read
  const Kernels k = kernels_of(tree, requests, tokens, max_added, heads, kv_heads);
  const size_t bound = causal ? window : 0;
  const Plan few =
      few_plan(tree, requests, max_added, max_length, bound, heads, kv_heads, head_dim);
  const Plan many =
      many_plan(elem, requests, tokens, max_added, max_length, bound, heads, kv_heads, head_dim);
  // rows16 numbers its tiles in 32 bits; a work-group of the other kernel has two threads a row
  if ((k.few && (requests * few.tiles * kv_heads > 0x7fffffffu || few.launch > kMostGroups)) ||
      (k.many && many.launch > 0xffffffffu / (2 * many.tile_rows)))
    return TCRV_HIP_ERR_TOO_LARGE;
  const size_t need = (k.few ? few.workspace : 0) + (k.many ? many.workspace : 0);
  if (need) {
    if (!workspace)
      return TCRV_HIP_ERR_NULL_POINTER;
    if (!aligned16(workspace))
      return TCRV_HIP_ERR_MISALIGNED;
    if (workspace_bytes < need)
      return TCRV_HIP_ERR_BAD_SIZE;
  }
  AttnArgs a{q,
             out,
             cache,
             block_table,
             first,
             length,
             static_cast<float *>(workspace),
             nullptr,
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
             0,  // the plans': launch_all
             static_cast<uint32_t>(max_added),
             static_cast<uint32_t>(max_length),
             0,
             0,
             0,
             0,
             0,
             0,
             scale,
             causal,
             groups_of_4(q, q_token, q_head, size),
             groups_of_4(out, out_token, out_head, size),
             ancestors,
             words};
  hipStream_t st = as_stream(stream);
  switch (elem) {
  case TCRV_HIP_ELEM_F32:
    launch_all<2, float, kTree>(a, k, few, many, head_dim, requests, st);
    break;
  case TCRV_HIP_ELEM_F16:
    launch_all<1, _Float16, kTree>(a, k, few, many, head_dim, requests, st);
    break;
  default:
    launch_all<1, tcrv::Bf16, kTree>(a, k, few, many, head_dim, requests, st);
    break;
  }
  return launch_status();
}

}  // namespace

extern "C" {

size_t tcrv_hip_attn_q4_0_workspace_bytes(int elem, size_t requests, size_t tokens,
                                          size_t max_added, size_t max_length, size_t heads,
                                          size_t kv_heads, size_t head_dim) {
  return workspace_bytes_of(false, elem, requests, tokens, max_added, max_length, heads, kv_heads,
                            head_dim);
}

size_t tcrv_hip_attn_tree_q4_0_workspace_bytes(int elem, size_t requests, size_t tokens,
                                               size_t max_added, size_t max_length, size_t heads,
                                               size_t kv_heads, size_t head_dim) {
  return workspace_bytes_of(true, elem, requests, tokens, max_added, max_length, heads, kv_heads,
                            head_dim);
}

int tcrv_hip_attn_q4_0(int elem, const void *q, size_t q_token, size_t q_head,
                       const uint8_t *cache, size_t pages, size_t page_size,
                       const int32_t *block_table, size_t table_stride, const int32_t *first,
                       const int32_t *length, size_t requests, size_t tokens, size_t max_added,
                       size_t max_length, size_t heads, size_t kv_heads, size_t head_dim,
                       float scale, int causal, size_t window, void *out, size_t out_token,
                       size_t out_head, void *workspace, size_t workspace_bytes, void *stream) {
  return attend<false>(elem, q, q_token, q_head, cache, pages, page_size, block_table, table_stride,
                       first, length, nullptr, 0, requests, tokens, max_added, max_length, heads,
                       kv_heads, head_dim, scale, causal, window, out, out_token, out_head, workspace,
                       workspace_bytes, stream);
}

int tcrv_hip_attn_tree_q4_0(int elem, const void *q, size_t q_token, size_t q_head,
                            const uint8_t *cache, size_t pages, size_t page_size,
                            const int32_t *block_table, size_t table_stride, const int32_t *first,
                            const int32_t *length, const uint64_t *ancestors, size_t words,
                            size_t requests, size_t tokens, size_t max_added, size_t max_length,
                            size_t heads, size_t kv_heads, size_t head_dim, float scale,
                            size_t window, void *out, size_t out_token, size_t out_head,
                            void *workspace, size_t workspace_bytes, void *stream) {
  return attend<true>(elem, q, q_token, q_head, cache, pages, page_size, block_table, table_stride,
                      first, length, ancestors, words, requests, tokens, max_added, max_length, heads,
                      kv_heads, head_dim, scale, 1, window, out, out_token, out_head, workspace,
                      workspace_bytes, stream);
}

}  // extern "C"

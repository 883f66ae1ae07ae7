// gated.hip -- the first half of a gated feed-forward: gate and up projection of Q8_0 rows by Q4_0 weight
// rows, the activation of the one and its product with the other, out in the element type or as Q8_0 rows.
//
// Both sums of a block are integers (|sum| <= 32 8 128), exact in whatever order; each is scaled by the
// weights' and the token's scale and added in f32.
#include <type_traits>

#include "kv_cache.h"
#include "mfma_fold.h"
#include "q8_block.h"

namespace tcrv {
namespace {

typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32a2 __attribute__((aligned(2)));

struct GatedArgs {
  const uint8_t *gate, *up, *vy;
  void *out;
  uint8_t *q8;
  size_t bx, by, out_token, q8_token;
  uint32_t nr, nc, nb;
  int act;
  bool out_vec;  // groups of 4 outputs lie on aligned places
};

// g / (1 + e^-x)
__device__ __forceinline__ float times_sigmoid(float g, float x) { return g / (1.0f + expf(-x)); }

__device__ __forceinline__ float activation(float g, int act) {
  switch (act) {
  case TCRV_HIP_ACT_SILU:
    return times_sigmoid(g, g);
  case TCRV_HIP_ACT_GELU_TANH:  // (1 + tanh z) / 2 is the logistic function of 2 z
    return times_sigmoid(g, 1.5957691216057308f * fmaf(0.044715f * g * g, g, g));
  case TCRV_HIP_ACT_GELU:
    return 0.5f * g * erfcf(g * -0.70710678118654752f);
  default:
    return g > 0.0f ? g : g * 0.0f;  // a NaN stays one
  }
}

// Lane `part` of eight with four of the 32 outputs from feature `at` on, of one token.
template <typename T, bool kBlocks = true>
__device__ __forceinline__ void emit(const GatedArgs &a, size_t token, uint32_t at, int part,
                                     const float (&v)[4]) {
  const uint32_t f = at + 4 * part;
  if (a.out) {
    T *const to = static_cast<T *>(a.out) + token * a.out_token + f;
    if (f + 4 <= a.nr) {
      store_values<4>(to, v, a.out_vec);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f + i < a.nr)
          to[i] = narrow<T>(v[i]);
    }
  }
  if (kBlocks && a.q8 && at + kQK <= a.nr)
    store_q8_part(a.q8 + token * a.q8_token + static_cast<size_t>(at / kQK) * kQ8Bytes, part, v);
}

struct Q4Block {
  u32x4a2 q;
  uint16_t d;
};
struct Q8Block {
  u32x4a2 q[2];
  uint16_t d;
};

__device__ __forceinline__ Q4Block load_q4(const uint8_t *p) {
  return {*reinterpret_cast<const u32x4a2 *>(p + 2), *reinterpret_cast<const uint16_t *>(p)};
}
__device__ __forceinline__ Q8Block load_q8(const uint8_t *p) {
  return {{*reinterpret_cast<const u32x4a2 *>(p + 2), *reinterpret_cast<const u32x4a2 *>(p + 18)},
          *reinterpret_cast<const uint16_t *>(p)};
}

// ---------------------------------------------------------------------------
// One token, or a few: a wave takes a feature, a lane a pair of the blocks of its two rows (or the one that they
// have).  A work-group is four features; of the 32 of a Q8_0 block (kBlocks) its sixteen waves take two each.  The
// read of the weights bounds it: 2 x 14336 features of 4096, past the last-level cache, 12.6 us (5.2 TB/s) into
// elements and 13.9 us into Q8_0; 2 x 4096 of 4096 5.4 us.  Two features a wave, which share the tokens' loads,
// took as long for 2 tokens and longer for 4: those are bound by VALU issue.
// ---------------------------------------------------------------------------
constexpr int one_waves(bool blocks) { return blocks ? 16 : 4; }

// The sum over the lanes, in the last one.
__device__ __forceinline__ float lanes_sum(float v) {
  const auto add = [&](auto control, auto lines) __attribute__((always_inline)) {
    v += __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(control)::value,
                                           decltype(lines)::value, 0xf, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // 1, 2, 4, 8 before, in 16
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // the last of the 16 before
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());
  return v;
}

// sum of (n - 8) y over a block: 16 bytes of quants n, 32 of y, and -8 times the sum of y
__device__ __forceinline__ float block_sum(const uint32_t (&q)[4], const uint32_t (&y)[8], int seed) {
  int sum = seed;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sum = sdot4(q[k] & 0x0f0f0f0fu, y[k], sum);
    sum = sdot4(q[k] >> 4 & 0x0f0f0f0fu, y[k + 4], sum);
  }
  return static_cast<float>(sum);
}

__device__ __forceinline__ int seed_of(const uint32_t (&y)[8]) {
  int sum = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    sum = sdot4(y[k], 0x01010101u, sum);
  return -8 * sum;
}

template <typename T, int kTokens, bool kPairs, bool kBlocks>
__global__ __launch_bounds__(one_waves(kBlocks) * 64) void gated_one(GatedArgs a) {
  constexpr int kWaves = one_waves(kBlocks), kTurns = kBlocks ? 2 : 1, kFeatures = kWaves * kTurns;
  __shared__ __align__(16) float s_out[kTokens][kFeatures];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t at = blockIdx.x * kFeatures;
  const uint32_t items = kPairs ? (a.nb + 1) / 2 : a.nb;
  // past the last one that one again
  const auto token = [&](uint32_t n) { return a.vy + min(n, a.nc - 1) * a.by; };
  for (int turn = 0; turn < kTurns; ++turn) {
    const size_t feature = min(at + turn * kWaves + wave, a.nr - 1);
    const uint8_t *const row[2] = {a.gate + feature * a.bx, a.up + feature * a.bx};
    float acc[kTokens][2] = {};
    for (uint32_t i0 = 0; i0 < items; i0 += 64) {
      const uint32_t i = min(i0 + lane, items - 1);
      const bool live = i0 + lane < items;
      if constexpr (kPairs) {
        // an odd number's last block is the second of the pair with the one before it
        const uint32_t b = min(2 * i, a.nb - 2);
        uint32_t w[2][9];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const u32a2 *const p = reinterpret_cast<const u32a2 *>(row[r] + b * kQ4Bytes);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const u32x4a2 v = *reinterpret_cast<const u32x4a2 *>(p + 4 * k);
            w[r][4 * k] = v.x;
            w[r][4 * k + 1] = v.y;
            w[r][4 * k + 2] = v.z;
            w[r][4 * k + 3] = v.w;
          }
          w[r][8] = p[8];
        }
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
          const u32a2 *const p = reinterpret_cast<const u32a2 *>(token(n) + b * kQ8Bytes);
          uint32_t y[17];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const u32x4a2 v = *reinterpret_cast<const u32x4a2 *>(p + 4 * k);
            y[4 * k] = v.x;
            y[4 * k + 1] = v.y;
            y[4 * k + 2] = v.z;
            y[4 * k + 3] = v.w;
          }
          y[16] = p[16];
          // the even block's quants lie 2 bytes off a dword, the odd one's on one
          uint32_t even[8], odd[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            even[k] = funnel16(y[k], y[k + 1]);
            odd[k] = y[k + 9];
          }
          const int even_seed = seed_of(even), odd_seed = seed_of(odd);
          const float even_d = live && b == 2 * i ? fp16_bits_to_f32(y[0] & 0xffffu) : 0.0f;
          const float odd_d = live ? fp16_bits_to_f32(y[8] >> 16) : 0.0f;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t e[4] = {funnel16(w[r][0], w[r][1]), funnel16(w[r][1], w[r][2]),
                                   funnel16(w[r][2], w[r][3]), funnel16(w[r][3], w[r][4])};
            const uint32_t o[4] = {w[r][5], w[r][6], w[r][7], w[r][8]};
            float &to = acc[n][r];
            to = fmaf(block_sum(e, even, even_seed) * fp16_bits_to_f32(w[r][0] & 0xffffu), even_d, to);
            to = fmaf(block_sum(o, odd, odd_seed) * fp16_bits_to_f32(w[r][4] >> 16), odd_d, to);
          }
        }
      } else {
        const Q4Block w[2] = {load_q4(row[0] + i * kQ4Bytes), load_q4(row[1] + i * kQ4Bytes)};
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
          const Q8Block b = load_q8(token(n) + i * kQ8Bytes);
          uint32_t y[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            y[k] = b.q[0][k];
            y[k + 4] = b.q[1][k];
          }
          const int seed = seed_of(y);
          const float d = live ? fp16_bits_to_f32(b.d) : 0.0f;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t q[4] = {w[r].q.x, w[r].q.y, w[r].q.z, w[r].q.w};
            acc[n][r] = fmaf(block_sum(q, y, seed) * fp16_bits_to_f32(w[r].d), d, acc[n][r]);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
      const float g = lanes_sum(acc[n][0]), u = lanes_sum(acc[n][1]);
      if (lane == 63)
        s_out[n][turn * kWaves + wave] = activation(g, a.act) * u;
    }
  }
  __syncthreads();
  const uint32_t part = threadIdx.x % (kFeatures / 4), n = threadIdx.x / (kFeatures / 4);
  if (n < kTokens && n < a.nc) {
    const float4 x = *reinterpret_cast<const float4 *>(&s_out[n][4 * part]);
    const float v[4] = {x.x, x.y, x.z, x.w};
    emit<T, kBlocks>(a, n, at, static_cast<int>(part), v);
  }
}

// ---------------------------------------------------------------------------
// Prompts: 32 kFT features x 128 tokens a work-group of eight waves, a wave kFW tiles of 32 features x 32 tokens
// of both projections, so that their sums meet in its registers.  The rows of kCB blocks are laid out in LDS
// as int8, the next ones on their way in registers.
//
// v_mfma_i32_32x32x32_i8 takes a block at a time, tokens as its rows, so that a lane holds one feature and
// 16 tokens: a weight's scale is one value a lane, and the tokens' 16 serve 2 kFW products.  Quants stay
// in the upper half of their bytes, 16 (n - 8) with a flipped top bit.  The accumulator starts at the bits of
// M = 1.5 2^23: read as floats its results are M + sum exactly (|sum| <= 16 32 8 128 < 2^22), and fma(M + sum,
// d, -M d) is the scaled sum, rounded once.
//
// VALU issue bounds it, 77 % of the SIMDs' cycles, 60 % the two instructions that scale and add a block's sum:
// 2 x 14336 features of 4096, 2048 tokens, 637 us (0.76 POP/s) where tiles whose blocks several waves shared out took
// 1488.  Rows in LDS are padded; swizzled ones took longer, and so did two chunks under way by hand (828 us).
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 512, kTileTokens = 128;

template <int kFT> struct Tiles {
  static constexpr int kCB = 4, kFW = kFT * (kTileTokens / 32) / (kTileThreads / 64);
  static constexpr int kWRows = 64 * kFT, kRows = kWRows + kTileTokens;
  static constexpr int kRow = kCB * kQK + 16;  // 16 bytes of 16 neighbouring rows in banks of their own
  static constexpr int kQuants = kRows * kRow, kStage = kQuants + kCB * kRows * 4;
  static constexpr int kWTasks = kWRows * kCB / kTileThreads;
  static constexpr int kYTasks = kTileTokens * kCB / kTileThreads;
  static constexpr int kOutRow = kFT * 32 + 4, kOut = kTileTokens * kOutRow * 4;
  static constexpr int kLds = 2 * kStage > kOut ? 2 * kStage : kOut;
  static __device__ __forceinline__ int at(int r, int b) { return r * kRow + b * kQK; }
};

template <typename T, int kFT>
__global__ __launch_bounds__(kTileThreads, 2) void gated_tiles(GatedArgs a) {
  using S = Tiles<kFT>;
  constexpr int kCB = S::kCB, kFW = S::kFW;
  __shared__ __align__(16) uint8_t lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = wave & 3, ft = (wave >> 2) * kFW;
  uint32_t tm, tn;
  tile_of(blockIdx.x, (a.nr + 32 * kFT - 1) / (32 * kFT), (a.nc + kTileTokens - 1) / kTileTokens, tm, tn);
  const uint32_t m0 = tm * (32 * kFT), n0 = tn * kTileTokens;

  // The thread's blocks of a chunk: block t % kCB of row t / kCB.  Weight rows by tiles: 32 of the
  // gate, 32 of the up projection.
  const int block = tid % kCB, row = tid / kCB;
  constexpr int kRowsATask = kTileThreads / kCB;
  const uint8_t *w_at[S::kWTasks], *y_at[S::kYTasks];
#pragma unroll
  for (int j = 0; j < S::kWTasks; ++j) {
    const int r = row + j * kRowsATask;
    const size_t f = min(m0 + (r >> 6) * 32 + (r & 31), a.nr - 1);
    w_at[j] = (r & 32 ? a.up : a.gate) + f * a.bx;
  }
#pragma unroll
  for (int j = 0; j < S::kYTasks; ++j)
    y_at[j] = a.vy + static_cast<size_t>(min(n0 + row + j * kRowsATask, a.nc - 1)) * a.by;
  Q4Block w[S::kWTasks];
  Q8Block y[S::kYTasks];
  // past the last block that one again, which nothing folds
  const auto load = [&](int c) __attribute__((always_inline)) {
    const uint32_t b = min(static_cast<uint32_t>(c * kCB + block), a.nb - 1);
#pragma unroll
    for (int j = 0; j < S::kWTasks; ++j)
      w[j] = load_q4(w_at[j] + b * kQ4Bytes);
#pragma unroll
    for (int j = 0; j < S::kYTasks; ++j)
      y[j] = load_q8(y_at[j] + b * kQ8Bytes);
  };
  const auto put = [&](uint8_t *stage) __attribute__((always_inline)) {
    float *const scales = reinterpret_cast<float *>(stage + S::kQuants) + block * S::kRows;
#pragma unroll
    for (int j = 0; j < S::kWTasks; ++j) {
      const int r = row + j * kRowsATask;
      u32x4 low, high;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t q = w[j].q[k] ^ 0x88888888u;
        low[k] = q << 4 & 0xf0f0f0f0u;
        high[k] = q & 0xf0f0f0f0u;
      }
      u32x4 *const to = reinterpret_cast<u32x4 *>(stage + S::at(r, block));
      to[0] = low;
      to[1] = high;
      scales[r] = 0.0625f * fp16_bits_to_f32(w[j].d);
    }
#pragma unroll
    for (int j = 0; j < S::kYTasks; ++j) {
      const int r = S::kWRows + row + j * kRowsATask;
      u32x4 *const to = reinterpret_cast<u32x4 *>(stage + S::at(r, block));
      to[0] = y[j].q[0];
      to[1] = y[j].q[1];
      scales[r] = fp16_bits_to_f32(y[j].d);
    }
  };

  v16i seed;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    seed[e] = kSeedBits;
  asm("" : "+v"(seed));  // kept in registers: as a constant it is made anew for every product
  float acc[2 * kFW][16] = {};
  const int w_row = ft * 64 + li, y_row = S::kWRows + nt * 32;
  const auto fold = [&](const uint8_t *stage, int b) __attribute__((always_inline)) {
    const float *const d = reinterpret_cast<const float *>(stage + S::kQuants) + b * S::kRows;
    const v4i tokens = *reinterpret_cast<const v4i *>(stage + S::at(y_row + li, b) + 16 * h);
    float dy[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 v = *reinterpret_cast<const float4 *>(d + y_row + 8 * k + 4 * h);
      dy[4 * k] = v.x;
      dy[4 * k + 1] = v.y;
      dy[4 * k + 2] = v.z;
      dy[4 * k + 3] = v.w;
    }
    const auto product = [&](int i) __attribute__((always_inline)) {
      const v4i weights =
          *reinterpret_cast<const v4i *>(stage + S::at(w_row + 32 * i, b) + 16 * h);
      return __builtin_bit_cast(
          v16f, __builtin_amdgcn_mfma_i32_32x32x32_i8(tokens, weights, seed, 0, 0, 0));
    };
    v16f sums = product(0);
#pragma unroll
    for (int i = 0; i < 2 * kFW; ++i) {
      v16f next;
      if (i + 1 < 2 * kFW)
        next = product(i + 1);  // on its way while this one is added
      const float dx = d[w_row + 32 * i], off = -kSeed * dx;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc[i][e] = fmaf(fmaf(sums[e], dx, off), dy[e], acc[i][e]);
      if (i + 1 < 2 * kFW)
        sums = next;
    }
  };

  if (a.nb > 0) {
    const int whole = static_cast<int>(a.nb / kCB);
    load(0);
    put(lds);
    load(1);
    __syncthreads();
    // chunk c is folded, c + 1 laid out, c + 2 set out for
    for (int c = 0; c < whole; ++c) {
      const uint8_t *const stage = lds + (c & 1) * S::kStage;
#pragma unroll
      for (int b = 0; b < kCB; ++b) {
        fold(stage, b);
        __builtin_amdgcn_sched_barrier(0);
      }
      put(lds + ((c + 1) & 1) * S::kStage);
      load(c + 2);
      __syncthreads();
    }
    for (int b = whole * kCB; b < static_cast<int>(a.nb); ++b)
      fold(lds + (whole & 1) * S::kStage, b - whole * kCB);
    __syncthreads();
  }

  // through LDS, so that a block's values are whole and rows are written by whole lines
  float *const out = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int f = 0; f < kFW; ++f)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      out[(nt * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * S::kOutRow + (ft + f) * 32 + li] =
          activation(acc[2 * f][e], a.act) * acc[2 * f + 1][e];
  __syncthreads();
  for (int t = tid; t < kTileTokens * kFT * 8; t += kTileThreads) {
    const int part = t & 7, block = (t >> 3) % kFT, row = t / (8 * kFT);
    const float4 x = *reinterpret_cast<const float4 *>(out + row * S::kOutRow + block * 32 + 4 * part);
    const float v[4] = {x.x, x.y, x.z, x.w};
    if (n0 + row < a.nc && m0 + block * 32 < a.nr)
      emit<T>(a, n0 + row, m0 + block * 32, part, v);
  }
}

// ---------------------------------------------------------------------------
// Some tens of tokens: 32 (or 16) features x 32 tokens a work-group.  Sixteen blocks of its rows at a time go to LDS as
// they lie in memory, in pieces of 16 bytes, and each of the eight waves takes a pair of them through both
// tiles; the waves' sums come together at the end.
//
// An operand of v_mfma_i32_32x32x32_i8 is 16 quants of a row a lane: lane group h (lanes 32 h ..) takes those
// of a Q4_0 block's bytes 8 h .. 8 h + 7, 8 h .. and 16 + 8 h .., and the same of a token's.  Of a pair the even
// block's quants lie 2 bytes off a dword, the odd one's on one; the dwords that hold them also hold the even
// scale in group 0 and the odd one in group 1, the operands of the v_mfma_f32_32x32x8_f16 that gives the
// products of the scales.  Quants stay in the upper half of their bytes, 16 (n - 8) with a flipped top bit.
//
// Where work-groups are one or two a CU the chain of a chunk bounds it, reads of LDS, two products and the sums'
// scaling: more chunks' loads under way or sixteen waves a work-group changed nothing.  2 x 11008 features of 4096,
// 29 tokens, 20 us (23 past the last-level cache; the weights alone 10.5 at a copy's rate); 2 x 14336 and 64 tokens
// 41 us.
// ---------------------------------------------------------------------------
constexpr int kSpanWaves = 8, kSpanThreads = kSpanWaves * 64, kSpanBlocks = 2 * kSpanWaves;

// kTiles: of 32 weight rows.  Two are 32 features' gate and up rows; one holds those of 16.
template <int kTiles> struct Spans {
  static constexpr int kWSpan = kSpanBlocks * kQ4Bytes, kYSpan = kSpanBlocks * kQ8Bytes;
  // twice an odd number of dwords: a dword of 32 rows in banks of its own each
  static constexpr int kWRow = kWSpan + 8, kYRow = kYSpan + 8;
  static_assert(kWRow % 16 == 8 && kYRow % 16 == 8, "");
  // pieces by 64, of one matrix each; a thread's
  static constexpr int kWGroups = 32 * (kWSpan / 16) / 64, kYGroups = 32 * (kYSpan / 16) / 64;
  static constexpr int kFeatures = 16 * kTiles;
  static constexpr int kGroups = kTiles * kWGroups + kYGroups;
  static constexpr int kPieces = (kGroups + kSpanWaves - 1) / kSpanWaves;
  static constexpr int kYAt = 32 * kTiles * kWRow, kStage = kYAt + 32 * kYRow;
  static constexpr int kMine = 16 / kSpanWaves;  // a lane's sums of a projection
  static constexpr int kParts = kSpanWaves * 16 * 64 * 4, kOutRow = 36;
  static constexpr int kLds = 2 * kStage;
  static_assert(kLds >= kParts + 32 * kOutRow * 4, "");
};

template <typename T, int kTiles>
__global__ __launch_bounds__(kSpanThreads, 4) void gated_spans(GatedArgs a) {
  using S = Spans<kTiles>;
  __shared__ __align__(16) uint8_t lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, h = lane >> 5;
  const int ks = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t tm, tn;
  tile_of(blockIdx.x, (a.nr + S::kFeatures - 1) / S::kFeatures, (a.nc + 31) / 32, tm, tn);
  const uint32_t m0 = tm * S::kFeatures, n0 = tn * 32;
  // The thread's pieces, by 64 of one matrix: its address stays in scalar registers.  Waves that have one
  // less take the last group's again.
  struct Piece {
    const uint8_t *base;   // of the matrix's rows in this work-group, and of the chunk
    uint32_t row, at, to;  // the row's offset, the place in it, the place in LDS
    bool tokens;
  };
  const auto piece_of = [&](int j) __attribute__((always_inline)) {
    const int g = min(j * kSpanWaves + ks, S::kGroups - 1), tile = min(g / S::kWGroups, kTiles);
    const int q = (g - tile * S::kWGroups) * 64 + lane;
    Piece p;
    p.tokens = tile == kTiles;
    const int r = p.tokens ? q / (S::kYSpan / 16) : q / (S::kWSpan / 16);
    p.at = 16 * (p.tokens ? q % (S::kYSpan / 16) : q % (S::kWSpan / 16));
    p.to = (p.tokens ? S::kYAt + r * S::kYRow : (32 * tile + r) * S::kWRow) + p.at;
    // of one tile the upper half are up rows
    const bool up = kTiles == 2 ? tile == 1 : r >= S::kFeatures;
    const uint32_t feature = r - (kTiles == 1 && up ? S::kFeatures : 0);
    p.base = p.tokens ? a.vy + static_cast<size_t>(n0) * a.by
                      : (up ? a.up : a.gate) + static_cast<size_t>(m0) * a.bx;
    p.row = p.tokens ? min(static_cast<uint32_t>(r), a.nc - 1 - n0) * static_cast<uint32_t>(a.by)
                     : min(feature, a.nr - 1 - m0) * static_cast<uint32_t>(a.bx);
    return p;
  };
  const uint8_t *base[S::kPieces];
  uint32_t from[S::kPieces], to[S::kPieces], step[S::kPieces];
#pragma unroll
  for (int j = 0; j < S::kPieces; ++j) {
    const Piece p = piece_of(j);
    base[j] = p.base;
    from[j] = p.row + p.at;
    to[j] = p.to;
    step[j] = p.tokens ? S::kYSpan : S::kWSpan;
  }
  u32x4a2 held[S::kPieces];
  const auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < S::kPieces; ++j) {
      held[j] = *reinterpret_cast<const u32x4a2 *>(base[j] + from[j]);
      base[j] += step[j];
    }
  };
  const auto put = [&](uint8_t *stage) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < S::kPieces; ++j) {
      u32x2 *const p = reinterpret_cast<u32x2 *>(stage + to[j]);
      p[0] = u32x2{held[j].x, held[j].y};
      p[1] = u32x2{held[j].z, held[j].w};
    }
  };
  // a part of a chunk: a row's last piece begins 16 bytes before its end, and goes as much before its
  // place; so do those that lie past it
  const auto lay_part = [&](uint8_t *stage, int blocks) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < S::kPieces; ++j) {
      const Piece p = piece_of(j);
      const uint32_t end = blocks * (p.tokens ? kQ8Bytes : kQ4Bytes) - 16, at = min(p.at, end);
      *reinterpret_cast<u32x4a2 *>(stage + p.to - (p.at - at)) =
          *reinterpret_cast<const u32x4a2 *>(base[j] + (p.row + at));
    }
  };

  const uint32_t m_even = h ? 0u : 0xffffu, m_odd = h ? 0xffff0000u : 0u;
  const int w_at = li * S::kWRow + ks * (2 * kQ4Bytes) + 8 * h;
  const int y_at = S::kYAt + li * S::kYRow + ks * (2 * kQ8Bytes) + 8 * h;
  float acc[kTiles][16] = {};
  const auto weights = [&](uint32_t q0, uint32_t q1) __attribute__((always_inline)) {
    q0 ^= 0x88888888u;
    q1 ^= 0x88888888u;
    const u32x4 v = {q0 << 4 & 0xf0f0f0f0u, q1 << 4 & 0xf0f0f0f0u, q0 & 0xf0f0f0f0u, q1 & 0xf0f0f0f0u};
    return __builtin_bit_cast(v4i, v);
  };
  const auto fold = [&](float (&to)[16], const u32x4 &y, const v4i &w, uint32_t dy,
                        uint32_t dw) __attribute__((always_inline)) {
    const v16i sums = q8_sumi(__builtin_bit_cast(v4i, y), w);
    const v16f scales = q8_dxy(dy, dw);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      to[e] = fmaf(static_cast<float>(sums[e]), scales[e], to[e]);
    // one product at a time, folded here and nothing moved across: 128 registers hold no two
#pragma unroll
    for (int e = 0; e < 16; ++e)
      asm volatile("" : "+v"(to[e]));
    __builtin_amdgcn_sched_barrier(0);
  };
  // the wave's pair of a chunk, or its even block alone
  const auto pair = [&](const uint8_t *stage, bool odd) __attribute__((always_inline)) {
    const uint32_t *x[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      x[i] = reinterpret_cast<const uint32_t *>(stage + w_at + i * 32 * S::kWRow);
    const uint32_t *const y = reinterpret_cast<const uint32_t *>(stage + y_at);
    v4i w[kTiles];
    uint32_t dw[kTiles], odd_dw[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      w[i] = weights(funnel16(x[i][0], x[i][1]), funnel16(x[i][1], x[i][2]));
      dw[i] = x[i][0] & m_even;
      odd_dw[i] = x[i][2] & m_odd;
    }
    const u32x4 even = {funnel16(y[0], y[1]), funnel16(y[1], y[2]), funnel16(y[4], y[5]),
                        funnel16(y[5], y[6])};
    const uint32_t odd_dy = y[6] & m_odd;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      fold(acc[i], even, w[i], y[0] & m_even, dw[i]);
    if (!odd)
      return;
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      w[i] = weights(x[i][5], x[i][6]);
    const u32x4 last = {y[9], y[10], y[13], y[14]};
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
      fold(acc[i], last, w[i], odd_dy, odd_dw[i]);
  };
  const int whole = static_cast<int>(a.nb / kSpanBlocks);
  const int rest = static_cast<int>(a.nb) - whole * kSpanBlocks;
  if (whole > 0) {
    load();
    put(lds);
    if (whole > 1)
      load();
    __syncthreads();
    for (int c = 0; c < whole; ++c) {
      pair(lds + (c & 1) * S::kStage, true);
      if (c + 1 < whole) {
        put(lds + ((c + 1) & 1) * S::kStage);
        if (c + 2 < whole)
          load();
      }
      __syncthreads();
    }
  }
  if (rest > 0) {
    lay_part(lds, rest);
    __syncthreads();
    if (2 * ks < rest)
      pair(lds, 2 * ks + 1 < rest);
    __syncthreads();
  }

  // the waves' sums together, kMine of a lane's each
  float *const parts = reinterpret_cast<float *>(lds);
  float *const out = reinterpret_cast<float *>(lds + S::kParts);
  float sum[kTiles][S::kMine];
#pragma unroll
  for (int p = 0; p < kTiles; ++p) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      parts[(ks * 16 + e) * 64 + lane] = acc[p][e];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < S::kMine; ++q) {
      sum[p][q] = 0.0f;
#pragma unroll
      for (int k = 0; k < kSpanWaves; ++k)
        sum[p][q] += parts[(k * 16 + ks * S::kMine + q) * 64 + lane];
      sum[p][q] *= 0.0625f;  // of the quants
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < S::kMine; ++q) {
    const int e = ks * S::kMine + q;
    float &to = out[(8 * (e >> 2) + 4 * h + (e & 3)) * S::kOutRow + li];
    if constexpr (kTiles == 2)
      to = activation(sum[0][q], a.act) * sum[1][q];
    else
      to = sum[0][q];
  }
  __syncthreads();
  constexpr int kOuts = S::kFeatures / 4;  // of a token, by four
  if (tid < 32 * kOuts) {
    const int part = tid % kOuts, row = tid / kOuts;
    const float4 x = *reinterpret_cast<const float4 *>(out + row * S::kOutRow + 4 * part);
    float v[4] = {x.x, x.y, x.z, x.w};
    if constexpr (kTiles == 1) {
      const float4 u = *reinterpret_cast<const float4 *>(out + row * S::kOutRow + S::kFeatures + 4 * part);
      const float by[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = activation(v[k], a.act) * by[k];
    }
    if (n0 + row < a.nc)
      emit<T, kTiles == 2>(a, n0 + row, m0, part, v);
  }
}

size_t up_by(size_t n, size_t by) { return (n + by - 1) / by; }

template <typename T, int kTiles> int launch_spans(const GatedArgs &a, hipStream_t st) {
  const size_t tiles = up_by(a.nr, Spans<kTiles>::kFeatures) * up_by(a.nc, 32);
  if (tiles > 0xffffffffu / kSpanThreads)
    return TCRV_HIP_ERR_TOO_LARGE;
  gated_spans<T, kTiles><<<dim3(static_cast<unsigned>(tiles)), dim3(kSpanThreads), 0, st>>>(a);
  return tcrv_host::launch_status();
}

template <typename T, int kFT> int launch_tiles(const GatedArgs &a, hipStream_t st) {
  const size_t tiles = up_by(a.nr, 32 * kFT) * up_by(a.nc, kTileTokens);
  if (tiles > 0xffffffffu / kTileThreads)
    return TCRV_HIP_ERR_TOO_LARGE;
  gated_tiles<T, kFT>
      <<<dim3(static_cast<unsigned>(tiles)), dim3(kTileThreads), 0, st>>>(a);
  return tcrv_host::launch_status();
}

template <typename T, int kTokens, bool kBlocks> int launch_one(const GatedArgs &a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(up_by(a.nr, kBlocks ? kQK : one_waves(false))));
  const dim3 block(one_waves(kBlocks) * 64);
  if (a.nb > 1)
    gated_one<T, kTokens, true, kBlocks><<<grid, block, 0, st>>>(a);
  else
    gated_one<T, kTokens, false, kBlocks><<<grid, block, 0, st>>>(a);
  return tcrv_host::launch_status();
}

template <typename T> int launch_elem(const GatedArgs &a, hipStream_t st) {
  // Each token more costs gated_one 3.5 us beside its 12.6 at 14336 features of 4096, gated_spans nothing; us,
  // gated_one / gated_spans: 2 tokens, 4096 features 6.8 / 13.5, 11008 13 / 21, 14336 16 / 23 and into Q8_0 20 / 23;
  // 4 tokens, 4096 9.5 / 13.5, 11008 19 / 21, 14336 24 / 23, into Q8_0 4096 15.1 / 13.7.
  if (a.nc == 1)
    return a.q8 ? launch_one<T, 1, true>(a, st) : launch_one<T, 1, false>(a, st);
  if (a.nc == 2)
    return a.q8 ? launch_one<T, 2, true>(a, st) : launch_one<T, 2, false>(a, st);
  if (a.nc <= 4 && !a.q8 && a.nr <= 12288)
    return launch_one<T, 4, false>(a, st);
  // 16 features a work-group where all of those run at once, and no block of 32 outputs is wanted: 8 tokens,
  // 4096 features of 4096, 10.2 us against 13.5, of 14336 25 against 34; past one a CU 15.4 and 14.3 (64 tokens)
  if (!a.q8 && up_by(a.nr, Spans<1>::kFeatures) * up_by(a.nc, 32) <= 256)
    return launch_spans<T, 1>(a, st);
  // By what the kernels take for a block of K, in ns: rounds of 256 work-groups, one a CU, of the tiles; the
  // spans', two a CU, go on as CUs are free.  Measured at K 4096, us, spans / 64 features x 128 tokens / 128 x
  // 128: 11008 features x 33 tokens 33 / 58 / 92, 14336 x 128 69 / 62 / 95, 11008 x 200 91 / 118 / 96, 4096 x
  // 512 72 / 61 / 93, 14336 x 512 265 / 229 / 187, 2048 960 / 780 / 640.  At K 1024 and 14336 what is taken is at most
  // 13 % over the best kernel (11008 x 200 of 14336 292 for 259), but for 3 and 4 tokens above at K 1024 (4096 features
  // 7.2 where 16 features a work-group take 5.2).
  const size_t groups = up_by(a.nr, kQK) * up_by(a.nc, 32);
  const size_t spans = groups <= 256 ? 100 : groups * 3 / 10;
  const size_t mid = 460 * up_by(up_by(a.nr, 64) * up_by(a.nc, kTileTokens), 256);
  const size_t wide = 720 * up_by(up_by(a.nr, 128) * up_by(a.nc, kTileTokens), 256);
  if (spans <= wide && spans <= mid)
    return launch_spans<T, 2>(a, st);
  return mid <= wide ? launch_tiles<T, 2>(a, st) : launch_tiles<T, 4>(a, st);
}

}  // namespace
}  // namespace tcrv

// A launch holds less than 2^32 threads along an axis: work-groups of 256, one four features.
constexpr size_t kMostFeatures = ((size_t{1} << 24) - 1) * 4;
// 32 rows' offsets are 32-bit.
constexpr size_t kMostStride = size_t{1} << 26;

extern "C" int tcrv_hip_gated_q4_0_q8_0(int elem, int act, size_t n, void *out, size_t out_token,
                                        uint8_t *q8, size_t q8_token, const uint8_t *gate,
                                        const uint8_t *up, size_t bx, const uint8_t *vy, size_t by,
                                        size_t nr, size_t nc, void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem), nb = n / tcrv::kQK;
  if (!size || act < TCRV_HIP_ACT_SILU || act > TCRV_HIP_ACT_RELU)
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (nr == 0 || nc == 0)
    return TCRV_HIP_OK;
  if (nr > kMostFeatures || nc > kMostTokens || nb > kMostStride / tcrv::kQ8Bytes ||
      (nr > 1 && bx > kMostStride) || (nc > 1 && by > kMostStride))
    return TCRV_HIP_ERR_TOO_LARGE;
  if ((!out && !q8) || (nb && (!gate || !up || !vy)))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(out, size) || !aligned2(q8) || (q8 && nc > 1 && q8_token & 1u) ||
      (nb && (!aligned2(gate) || !aligned2(up) || !aligned2(vy) || (nr > 1 && bx & 1u) ||
              (nc > 1 && by & 1u))))
    return TCRV_HIP_ERR_MISALIGNED;
  if ((nc > 1 && ((out && out_token < nr) || (q8 && q8_token < nr / tcrv::kQK * tcrv::kQ8Bytes) ||
                  (nb && by < nb * tcrv::kQ8Bytes))) ||
      (nr > 1 && nb && bx < nb * tcrv::kQ4Bytes))
    return TCRV_HIP_ERR_BAD_SIZE;
  const tcrv::GatedArgs a{gate,
                          up,
                          vy,
                          out,
                          q8,
                          bx,
                          by,
                          out_token,
                          q8_token,
                          static_cast<uint32_t>(nr),
                          static_cast<uint32_t>(nc),
                          static_cast<uint32_t>(nb),
                          act,
                          aligned_to(out, 4 * size) && (nc == 1 || out_token % 4 == 0)};
  hipStream_t st = as_stream(stream);
  if (elem == TCRV_HIP_ELEM_F32)
    return tcrv::launch_elem<float>(a, st);
  if (elem == TCRV_HIP_ELEM_F16)
    return tcrv::launch_elem<_Float16>(a, st);
  return tcrv::launch_elem<tcrv::Bf16>(a, st);
}

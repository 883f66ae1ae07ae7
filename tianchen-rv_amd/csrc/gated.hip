// gated.hip -- the first half of a gated feed-forward: gate and up projection of Q8_0 rows by Q4_0 weight
// rows, the activation of the one and its product with the other, out in the element type or as Q8_0 rows.
//
// Both sums of a block are integers (|sum| <= 32 8 128), exact in whatever order; each is scaled by the
// weights' and the token's scale and added in f32.
#include "kv_cache.h"
#include "mfma_fold.h"
#include "q8_block.h"

namespace tcrv {
namespace {

typedef uint32_t u32x4a2 __attribute__((ext_vector_type(4), aligned(2)));

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
template <typename T>
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
  if (a.q8 && at + kQK <= a.nr)
    store_q8_part(a.q8 + token * a.q8_token + static_cast<size_t>(at / kQK) * kQ8Bytes, part, v);
}

// ---------------------------------------------------------------------------
// A few tokens: a work-group takes 32 features, a wave kF of them, a lane one block in 64 of their rows.
// ---------------------------------------------------------------------------
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

__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1)
    v += __shfl_xor(v, m);
  return v;
}

template <typename T, int kCols, int kF>
__global__ __launch_bounds__(32 / kF * 64) void gated_few(GatedArgs a) {
  __shared__ float s_out[kCols][kQK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t at = blockIdx.x * kQK, f0 = at + wave * kF;
  const uint8_t *row[2 * kF];
#pragma unroll
  for (int f = 0; f < kF; ++f) {
    const size_t r = min(f0 + f, a.nr - 1);
    row[2 * f] = a.gate + r * a.bx;
    row[2 * f + 1] = a.up + r * a.bx;
  }
  float acc[kCols][2 * kF] = {};
  for (uint32_t b0 = 0; b0 < a.nb; b0 += 64) {
    const uint32_t b = min(b0 + lane, a.nb - 1);
    const bool live = b0 + lane < a.nb;
    Q4Block w[2 * kF];
#pragma unroll
    for (int r = 0; r < 2 * kF; ++r)
      w[r] = load_q4(row[r] + static_cast<size_t>(b) * kQ4Bytes);
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const Q8Block y = load_q8(a.vy + c * a.by + static_cast<size_t>(b) * kQ8Bytes);
      int seed = 0;  // the quants are n - 8
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        seed = sdot4(y.q[0][k], 0x01010101u, seed);
        seed = sdot4(y.q[1][k], 0x01010101u, seed);
      }
      const float dy = live ? fp16_bits_to_f32(y.d) : 0.0f;
#pragma unroll
      for (int r = 0; r < 2 * kF; ++r) {
        int sum = -8 * seed;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sum = sdot4(w[r].q[k] & 0x0f0f0f0fu, y.q[0][k], sum);
          sum = sdot4(w[r].q[k] >> 4 & 0x0f0f0f0fu, y.q[1][k], sum);
        }
        acc[c][r] = fmaf(static_cast<float>(sum) * fp16_bits_to_f32(w[r].d), dy, acc[c][r]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kCols; ++c)
#pragma unroll
    for (int f = 0; f < kF; ++f) {
      const float g = lanes_sum(acc[c][2 * f]), u = lanes_sum(acc[c][2 * f + 1]);
      if (lane == 0)
        s_out[c][wave * kF + f] = activation(g, a.act) * u;
    }
  __syncthreads();
  if (threadIdx.x < 8 * kCols) {
    const int c = threadIdx.x >> 3, part = threadIdx.x & 7;
    const float v[4] = {s_out[c][4 * part], s_out[c][4 * part + 1], s_out[c][4 * part + 2],
                        s_out[c][4 * part + 3]};
    emit<T>(a, c, at, part, v);
  }
}

// ---------------------------------------------------------------------------
// More tokens: kFT x kNT tiles of 32 features x 32 tokens a work-group, kKS waves a tile, which share out
// its blocks.  A wave holds the gate's and the up projection's sums of its tile, so that they meet in its
// registers.  The rows of kCB blocks are laid out in LDS as int8, the next ones loaded meanwhile.
//
// v_mfma_i32_32x32x32_i8 takes a block at a time, tokens as its rows, so that a lane holds one feature and
// 16 tokens: a weight's scale is one value a lane.  Its accumulator starts at the bits of M = 1.5 2^23:
// read as floats its results are M + sum exactly, and fma(M + sum, d, -M d) is the scaled sum, rounded once.
// ---------------------------------------------------------------------------
template <int kFT, int kNT, int kKS, int kCB> struct Tiles {
  static constexpr int kWaves = kFT * kNT * kKS, kThreads = kWaves * 64;
  static constexpr int kWRows = 64 * kFT, kYRows = 32 * kNT, kRows = kWRows + kYRows;
  static constexpr int kRow = kCB * kQK + 16;  // 16-byte reads of 16 neighbouring rows meet no bank twice
  static constexpr int kQuants = kRows * kRow, kStage = kQuants + kCB * kRows * 4;
  static constexpr int kWTasks = (kWRows * kCB + kThreads - 1) / kThreads;
  static constexpr int kYTasks = (kYRows * kCB + kThreads - 1) / kThreads;
  static constexpr int kParts = kKS > 1 ? kWaves * 16 * 64 * 4 : 0;  // of one projection's sums
  static constexpr int kOutRow = kFT * 32 + 4;
  static constexpr int kOut = kYRows * kOutRow * 4;
  static constexpr int kLds = 2 * kStage > kParts + kOut ? 2 * kStage : kParts + kOut;
};

template <typename T, int kFT, int kNT, int kKS, int kCB>
__global__ __launch_bounds__((Tiles<kFT, kNT, kKS, kCB>::kThreads)) void gated_tiles(GatedArgs a) {
  using S = Tiles<kFT, kNT, kKS, kCB>;
  __shared__ __align__(16) uint8_t lds[S::kLds];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ks = wave % kKS, nt = wave / kKS % kNT, ft = wave / (kKS * kNT);
  uint32_t tm, tn;
  tile_of(blockIdx.x, (a.nr + 32 * kFT - 1) / (32 * kFT), (a.nc + 32 * kNT - 1) / (32 * kNT), tm, tn);
  const uint32_t m0 = tm * (32 * kFT), n0 = tn * (32 * kNT);

  // The thread's blocks of a chunk: block t % kCB of row t / kCB.  Weight rows by tiles: 32 of the
  // gate, 32 of the up projection.
  const uint8_t *w_at[S::kWTasks], *y_at[S::kYTasks];
#pragma unroll
  for (int j = 0; j < S::kWTasks; ++j) {
    const int t = j * S::kThreads + tid, r = min(t / kCB, S::kWRows - 1);
    const size_t f = min(m0 + (r >> 6) * 32 + (r & 31), a.nr - 1);
    w_at[j] = (r & 32 ? a.up : a.gate) + f * a.bx + t % kCB * kQ4Bytes;
  }
#pragma unroll
  for (int j = 0; j < S::kYTasks; ++j) {
    const int t = j * S::kThreads + tid, r = min(t / kCB, S::kYRows - 1);
    y_at[j] = a.vy + static_cast<size_t>(min(n0 + r, a.nc - 1)) * a.by + t % kCB * kQ8Bytes;
  }
  Q4Block w[S::kWTasks];
  Q8Block y[S::kYTasks];
  const auto load = [&](int blocks) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < S::kWTasks; ++j) {
      if ((j * S::kThreads + tid) % kCB < blocks)
        w[j] = load_q4(w_at[j]);
      w_at[j] += kCB * kQ4Bytes;
    }
#pragma unroll
    for (int j = 0; j < S::kYTasks; ++j) {
      if ((j * S::kThreads + tid) % kCB < blocks)
        y[j] = load_q8(y_at[j]);
      y_at[j] += kCB * kQ8Bytes;
    }
  };
  const auto put = [&](uint8_t *stage, int blocks) __attribute__((always_inline)) {
    float *const scales = reinterpret_cast<float *>(stage + S::kQuants);
#pragma unroll
    for (int j = 0; j < S::kWTasks; ++j) {
      const int t = j * S::kThreads + tid, r = t / kCB, b = t % kCB;
      if (t >= S::kWRows * kCB || b >= blocks)
        continue;
      u32x4 *const to = reinterpret_cast<u32x4 *>(stage + r * S::kRow + b * kQK);
      u32x4 low, high;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        low[k] = nibbles_to_i8x4(w[j].q[k]);
        high[k] = nibbles_to_i8x4(w[j].q[k] >> 4);
      }
      to[0] = low;
      to[1] = high;
      scales[b * S::kRows + r] = fp16_bits_to_f32(w[j].d);
    }
#pragma unroll
    for (int j = 0; j < S::kYTasks; ++j) {
      const int t = j * S::kThreads + tid, r = S::kWRows + t / kCB, b = t % kCB;
      if (t >= S::kYRows * kCB || b >= blocks)
        continue;
      u32x4 *const to = reinterpret_cast<u32x4 *>(stage + r * S::kRow + b * kQK);
      to[0] = y[j].q[0];
      to[1] = y[j].q[1];
      scales[b * S::kRows + r] = fp16_bits_to_f32(y[j].d);
    }
  };

  v16i seed;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    seed[e] = kSeedBits;
  asm("" : "+v"(seed));  // kept in registers: as a constant it is made anew for every product
  float acc[2][16] = {};
  const int g_row = ft * 64 + li, y_row = S::kWRows + nt * 32;
  const auto fold = [&](const uint8_t *stage, int b) __attribute__((always_inline)) {
    const uint8_t *const q = stage + b * kQK + 16 * h;
    const float *const d = reinterpret_cast<const float *>(stage + S::kQuants) + b * S::kRows;
    const v4i tokens = *reinterpret_cast<const v4i *>(q + (y_row + li) * S::kRow);
    float dy[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 v = *reinterpret_cast<const float4 *>(d + y_row + 8 * k + 4 * h);
      dy[4 * k] = v.x;
      dy[4 * k + 1] = v.y;
      dy[4 * k + 2] = v.z;
      dy[4 * k + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const v4i weights = *reinterpret_cast<const v4i *>(q + (g_row + 32 * i) * S::kRow);
      const float dx = d[g_row + 32 * i], off = -kSeed * dx;
      const v16f sums = __builtin_bit_cast(
          v16f, __builtin_amdgcn_mfma_i32_32x32x32_i8(tokens, weights, seed, 0, 0, 0));
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc[i][e] = fmaf(fmaf(sums[e], dx, off), dy[e], acc[i][e]);
    }
  };

  const int chunks = static_cast<int>((a.nb + kCB - 1) / kCB);
  const auto blocks_of = [&](int c) { return min(static_cast<int>(a.nb) - c * kCB, kCB); };
  if (chunks > 0) {
    load(blocks_of(0));
    put(lds, blocks_of(0));
  }
  __syncthreads();
  for (int c = 0; c < chunks; ++c) {
    const uint8_t *const stage = lds + (c & 1) * S::kStage;
    const int blocks = blocks_of(c);
    if (c + 1 < chunks)
      load(blocks_of(c + 1));
    if (blocks == kCB) {
#pragma unroll
      for (int b = 0; b < kCB / kKS; ++b) {
        fold(stage, b * kKS + ks);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      for (int b = ks; b < blocks; b += kKS)
        fold(stage, b);
    }
    if (c + 1 < chunks)
      put(lds + ((c + 1) & 1) * S::kStage, blocks_of(c + 1));
    __syncthreads();
  }

  // the tile's outputs, 16 / kKS elements a wave
  float *const out = reinterpret_cast<float *>(lds + S::kParts);
  constexpr int kMine = 16 / kKS;
  float sum[2][kMine];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (kKS == 1) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sum[i][e] = acc[i][e];
    } else {
      float *const parts = reinterpret_cast<float *>(lds) + (wave - ks) * 1024;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        parts[ks * 1024 + e * 64 + lane] = acc[i][e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kMine; ++e) {
        sum[i][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < kKS; ++k)
          sum[i][e] += parts[k * 1024 + (ks * kMine + e) * 64 + lane];
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int e = ks * kMine + i;
    out[(nt * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) * S::kOutRow + ft * 32 + li] =
        activation(sum[0][i], a.act) * sum[1][i];
  }
  __syncthreads();
  static_assert(S::kYRows * kFT * 8 % S::kThreads == 0 || S::kThreads > S::kYRows * kFT * 8, "");
  for (int t = tid; t < S::kYRows * kFT * 8; t += S::kThreads) {
    const int part = t & 7, block = (t >> 3) % kFT, row = t / (8 * kFT);
    const float4 x = *reinterpret_cast<const float4 *>(out + row * S::kOutRow + block * 32 + 4 * part);
    const float v[4] = {x.x, x.y, x.z, x.w};
    if (n0 + row < a.nc && m0 + block * 32 < a.nr)
      emit<T>(a, n0 + row, m0 + block * 32, part, v);
  }
}

template <typename T, int kCols> void launch_few(const GatedArgs &a, hipStream_t st) {
  gated_few<T, kCols, 4><<<dim3((a.nr + kQK - 1) / kQK), dim3(512), 0, st>>>(a);
}

template <typename T, int kFT, int kNT, int kKS, int kCB>
int launch_tiles(const GatedArgs &a, hipStream_t st) {
  const uint64_t tiles = static_cast<uint64_t>((a.nr + 32 * kFT - 1) / (32 * kFT)) *
                         ((a.nc + 32 * kNT - 1) / (32 * kNT));
  using S = Tiles<kFT, kNT, kKS, kCB>;
  if (tiles > 0xffffffffu / S::kThreads)
    return TCRV_HIP_ERR_TOO_LARGE;
  gated_tiles<T, kFT, kNT, kKS, kCB>
      <<<dim3(static_cast<unsigned>(tiles)), dim3(S::kThreads), 0, st>>>(a);
  return tcrv_host::launch_status();
}

template <typename T> int launch_elem(const GatedArgs &a, hipStream_t st) {
  switch (a.nc) {
  case 1:
    launch_few<T, 1>(a, st);
    break;
  case 2:
    launch_few<T, 2>(a, st);
    break;
  case 3:
    launch_few<T, 3>(a, st);
    break;
  case 4:
    launch_few<T, 4>(a, st);
    break;
  default:
    return a.nc <= 128 ? launch_tiles<T, 1, 1, 8, 8>(a, st) : launch_tiles<T, 4, 4, 1, 4>(a, st);
  }
  return tcrv_host::launch_status();
}

}  // namespace
}  // namespace tcrv

// A launch holds less than 2^32 threads along an axis: work-groups of 512, one 32 features.
constexpr size_t kMostFeatures = ((size_t{1} << 23) - 1) * tcrv::kQK;

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
  if (nr > kMostFeatures || nc > kMostTokens || nb > 0x7fffffffu / tcrv::kQ8Bytes)
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

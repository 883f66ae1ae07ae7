// rms_norm.hip -- the residual's addition and the root-mean-square norm, in the element type or as the
// Q8_0 rows that the next quantized product takes.
//
// A row's values stay in registers between the sum of their squares and their scaling, so that it is
// read once; rows past what registers hold are read twice.  Squares are summed in f64: exact products
// and sums off by some 2^-50 of theirs, so that c = 1 / sqrt(mean + eps) rounds to the same f32 for all
// but one row in tens of millions, however its work is laid out.
//
// Memory bounds it for many rows, what it reads and writes once: 4096 rows of 4096 with residual and sum
// into elements take 54 us in f32 (5.0 TB/s, a large copy's rate) and 30 us in f16 (4.5 TB/s), into Q8_0
// 50 and 29 us.  Of one row latency does: 2.6 us into elements, 3.2 us into Q8_0, a few round trips to
// memory and an empty kernel's 1.5 us.
#include <type_traits>

#include "kv_cache.h"
#include "q8_block.h"

namespace tcrv {
namespace {

struct NormArgs {
  const void *x, *residual;
  void *sum, *y;
  const float *weight;
  uint8_t *q8;
  size_t x_token, residual_token, sum_token, y_token, q8_token;
  double eps, per_value;  // 1 / n
  uint32_t tokens, n;
};

constexpr int kLongThreads = 1024;

// The sum over groups of kLanes lanes, 16 or 64, in all of them.
template <int kLanes> __device__ __forceinline__ double group_sum(double v) {
  const auto add = [&](auto control, auto lines) __attribute__((always_inline)) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t low = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(x), decltype(control)::value, decltype(lines)::value, 0xf, false));
    const uint32_t high = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(x >> 32), decltype(control)::value, decltype(lines)::value, 0xf, false));
    v += __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());  // 1, 2, 4, 8 before, in 16
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  if constexpr (kLanes == 16)
    return __shfl(v, threadIdx.x | 15);
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // the last of the 16 before
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());
  const uint64_t x = __builtin_bit_cast(uint64_t, v);
  const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(x), 63);
  const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(x >> 32), 63);
  return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}

// kV of a block's values as this lane's part of it, into LDS; 32 / kV neighbouring lanes take part.
template <int kV>
__device__ __forceinline__ void put_q8_part(uint8_t *block, int part, const float (&v)[kV]) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < kV; ++i)
    top = fmaxf(top, fabsf(v[i]));
  top = kV == 8 ? max4(top) : max8(top);
  const float d = __fdiv_rn(top, 127.0f);
  const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
  uint16_t *const to = reinterpret_cast<uint16_t *>(block);
#pragma unroll
  for (int i = 0; i < kV; i += 2)
    to[1 + (kV * part + i) / 2] =
        static_cast<uint16_t>(quant_byte(v[i], id) | quant_byte(v[i + 1], id) << 8);
  if (part == 0)
    to[0] = __builtin_bit_cast(uint16_t, static_cast<_Float16>(d));
}

// kThreads a row, kRows rows a work-group; a thread's group k is kV elements from kV (t + k kThreads) on, so
// that 32 / kV lanes hold a block.  kVec: all groups are whole and aligned.  kPer 0: rows of any length,
// read twice.  Blocks go out through LDS, by whole lines.
template <typename T, int kThreads, int kRows, int kPer, int kV, bool kVec>
__global__ __launch_bounds__(kThreads *kRows) void add_rms_norm_rows(NormArgs a) {
  constexpr int kWaves = kThreads > 64 ? kThreads / 64 : 1, kHeld = kPer ? kPer : 1;
  constexpr int kStaged = kThreads * kV / kQK * kQ8Bytes;  // bytes of a round of groups
  __shared__ double s_sum[kRows][kWaves];
  // each row's begin at a 16-byte place, also where the caller's rows have others than these
  constexpr int kQ8Row = (kHeld * kStaged + 15) & -16;
  static_assert(kQ8Row % 16 == 0, "copy_lds_to_span reads from 16-byte places");
  __shared__ __align__(16) uint8_t s_q8[kRows][kQ8Row];
  const int t = threadIdx.x % kThreads, r = threadIdx.x / kThreads;
  const uint32_t row = (blockIdx.y * gridDim.x + blockIdx.x) * kRows + r;
  const uint32_t token = min(row, a.tokens - 1);
  const bool live = row < a.tokens;
  const T *const x = static_cast<const T *>(a.x) + token * a.x_token;
  const T *const residual =
      a.residual ? static_cast<const T *>(a.residual) + token * a.residual_token : nullptr;
  const auto group = [&](uint32_t at, float (&h)[kV]) __attribute__((always_inline)) {
    float other[kV] = {};
    if constexpr (kVec) {
      if (at < a.n) {
        load_values<kV>(h, x + at, true);
        if (residual)
          load_values<kV>(other, residual + at, true);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i)
          h[i] = 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const bool in = at + i < a.n;
        h[i] = in ? widen(x[at + i]) : 0.0f;
        other[i] = in && residual ? widen(residual[at + i]) : 0.0f;
      }
    }
    if (residual) {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        h[i] += other[i];
    }
  };
  const auto put = [&](T *to, uint32_t at, const float (&v)[kV]) __attribute__((always_inline)) {
    if constexpr (kVec) {
      if (at < a.n)
        store_values<kV>(to + at, v, true);
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (at + i < a.n)
          to[at + i] = narrow<T>(v[i]);
    }
  };
  const auto finish = [&](uint32_t at, int k, const float (&h)[kV], float c) __attribute__((
                          always_inline)) {
    if (a.sum && live)
      put(static_cast<T *>(a.sum) + token * a.sum_token, at, h);
    float y[kV], w[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i)
      w[i] = 1.0f;
    if (a.weight) {
      if constexpr (kVec) {
        if (at < a.n) {
#pragma unroll
          for (int i = 0; i < kV; i += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(a.weight + at + i);
            w[i] = v.x;
            w[i + 1] = v.y;
            w[i + 2] = v.z;
            w[i + 3] = v.w;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i)
          if (at + i < a.n)
            w[i] = a.weight[at + i];
      }
    }
#pragma unroll
    for (int i = 0; i < kV; ++i)
      y[i] = h[i] * c * w[i];
    if (a.y && live)
      put(static_cast<T *>(a.y) + token * a.y_token, at, y);
    if (a.q8)
      put_q8_part<kV>(s_q8[r] + k * kStaged + t * kV / kQK * kQ8Bytes, t % (kQK / kV), y);
  };
  // the blocks from element `at` on; a row's lanes in one wave need no meeting
  const auto blocks_out = [&](uint32_t at) __attribute__((always_inline)) {
    if constexpr (kThreads <= 64)
      wave_lds_sync();
    else
      __syncthreads();
    const uint32_t first = at / kQK, all = a.n / kQK;
    const int blocks = min(static_cast<int>(max(all, first) - first), kHeld * kThreads * kV / kQK);
    if (live && blocks > 0)
      copy_lds_to_span(a.q8 + token * a.q8_token + static_cast<size_t>(first) * kQ8Bytes, s_q8[r],
                       blocks * kQ8Bytes, t, kThreads);
  };

  float h[kHeld][kV];
  double total = 0.0;
  const auto add = [&](const float (&v)[kV]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      total = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), total);
  };
  if constexpr (kPer) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      group(kV * (t + k * kThreads), h[k]);
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      add(h[k]);
  } else {
    for (uint32_t at = kV * t; at < a.n; at += kV * kThreads) {
      group(at, h[0]);
      add(h[0]);
    }
  }
  total = group_sum<kThreads < 64 ? kThreads : 64>(total);
  if constexpr (kWaves > 1) {
    if ((t & 63) == 0)
      s_sum[r][t >> 6] = total;
    __syncthreads();
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      total += s_sum[r][w];
  }
  const float c = static_cast<float>(rsqrt(fma(total, a.per_value, a.eps)));
  if constexpr (kPer) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      finish(kV * (t + k * kThreads), k, h[k], c);
    if (a.q8)
      blocks_out(0);
  } else {
    // a thread takes in the group before it writes there
    for (uint32_t at = 0; at < a.n; at += kV * kThreads) {
      group(at + kV * t, h[0]);
      finish(at + kV * t, 0, h[0], c);
      if (a.q8) {
        blocks_out(at);
        __syncthreads();
      }
    }
  }
}

template <typename T, int kThreads, int kRows, int kPer, int kV, bool kVec>
void launch(const NormArgs &a, hipStream_t st) {
  // along x less than 2^32 threads
  const uint32_t groups = (a.tokens + kRows - 1) / kRows, most = 1u << 20;
  const dim3 grid(groups < most ? groups : most, (groups + most - 1) / most), block(kThreads * kRows);
  add_rms_norm_rows<T, kThreads, kRows, kPer, kV, kVec><<<grid, block, 0, st>>>(a);
}

// Threads of a row by its length, so that they have work and the row stays in registers.  16 for the short
// rows of heads: 60000 rows of 128 f16 into Q8_0 take 16 us, 65 us with a wave a row.  1024 for a few long
// rows, whose latency counts: one of 4096 f32 takes 2.6 us, 3.6 us with 256.  Into Q8_0, us, fewer threads /
// 1024: rows of 4096 f16, 64 4.0 / 3.7, 256 5.5 / 5.0, 384 6.2 / 6.8; f32, 64 6.2 / 4.0, 512 10.4 / 9.3; of 1024
// f32, 512 6.4 / 5.4, 768 6.5 / 6.9.
template <typename T, int kV, bool kVec> void launch_size(const NormArgs &a, hipStream_t st) {
  constexpr uint32_t kFewTokens = kV == 8 ? 256 : 512;
  const uint32_t groups = (a.n + kV - 1) / kV;
  if (groups <= 16)
    launch<T, 16, 16, 1, kV, kVec>(a, st);
  else if (groups <= 64)
    launch<T, 16, 16, 4, kV, kVec>(a, st);
  else if (a.tokens <= kFewTokens && groups <= kLongThreads)
    launch<T, kLongThreads, 1, 1, kV, kVec>(a, st);
  else if (groups <= 128)
    launch<T, 64, 4, 2, kV, kVec>(a, st);
  else if (groups <= 256)
    launch<T, 64, 4, 4, kV, kVec>(a, st);
  else if (groups <= 512)
    launch<T, 256, 1, 2, kV, kVec>(a, st);
  else if (groups <= 1024)
    launch<T, 256, 1, 4, kV, kVec>(a, st);
  else if (groups <= 4 * kLongThreads)
    launch<T, kLongThreads, 1, 4, kV, kVec>(a, st);
  else
    launch<T, kLongThreads, 1, 0, kV, kVec>(a, st);
}

template <typename T> void launch_elem(const NormArgs &a, bool by_4, bool by_8, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (by_8) {
      launch_size<T, 8, true>(a, st);
      return;
    }
  }
  by_4 ? launch_size<T, 4, true>(a, st) : launch_size<T, 4, false>(a, st);
}

}  // namespace
}  // namespace tcrv

extern "C" int tcrv_hip_add_rms_norm(int elem, const void *x, size_t x_token, const void *residual,
                                     size_t residual_token, void *sum, size_t sum_token,
                                     const float *weight, double eps, void *y, size_t y_token,
                                     uint8_t *q8, size_t q8_token, size_t tokens, size_t n,
                                     void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem);
  if (!size)
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (!(eps >= 0.0) || !(eps - eps == 0.0))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (tokens == 0 || n == 0)
    return TCRV_HIP_OK;
  if (tokens > kMostTokens || n > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (tokens > 1 && (x_token < n || (residual && residual_token < n) || (sum && sum_token < n) ||
                     (y && y_token < n) || (q8 && q8_token < n / tcrv::kQK * tcrv::kQ8Bytes)))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (!x || (!sum && !y && !q8))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(x, size) || !aligned_to(residual, size) || !aligned_to(sum, size) ||
      !aligned_to(y, size) || !aligned4(weight) || !aligned2(q8) || (q8 && tokens > 1 && q8_token & 1u))
    return TCRV_HIP_ERR_MISALIGNED;
  // groups of so many values on aligned places
  const auto by = [&](size_t values) {
    const auto fits = [&](const void *p, size_t stride) {
      return !p || (aligned_to(p, values * size) && (tokens == 1 || stride % values == 0));
    };
    return n % values == 0 && fits(x, x_token) && fits(residual, residual_token) &&
           fits(sum, sum_token) && fits(y, y_token) && aligned16(weight);
  };
  const bool by_4 = by(4), by_8 = by(8);
  const tcrv::NormArgs a{x,        residual, sum,            y,         weight,
                         q8,       x_token,  residual_token, sum_token, y_token,
                         q8_token, eps,      1.0 / static_cast<double>(n), static_cast<uint32_t>(tokens),
                         static_cast<uint32_t>(n)};
  hipStream_t st = as_stream(stream);
  if (elem == TCRV_HIP_ELEM_F32)
    tcrv::launch_elem<float>(a, by_4, by_8, st);
  else if (elem == TCRV_HIP_ELEM_F16)
    tcrv::launch_elem<_Float16>(a, by_4, by_8, st);
  else
    tcrv::launch_elem<tcrv::Bf16>(a, by_4, by_8, st);
  return launch_status();
}

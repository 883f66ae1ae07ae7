// rms_norm.hip -- the residual's addition and the root-mean-square norm, in the element type or as the
// Q8_0 rows that the next quantized product takes.
//
// A row's values stay in registers between the sum of their squares and their scaling, so that it is
// read once; rows past what registers hold are read twice.  Squares are summed in f64: exact products
// and sums off by some 2^-50 of theirs, so that c = 1 / sqrt(mean + eps) rounds to the same f32 in any
// order and the quants of a row do not depend on how its work is laid out.
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
  double eps;
  uint32_t tokens, n;
};

constexpr int kLongThreads = 1024;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1)
    v += __shfl_xor(v, m);
  return v;
}

// kThreads a row, kRows rows a work-group; a thread's group k is elements 4 (t + k kThreads) and the
// three after, so that eight lanes hold a block.  kVec: all groups are whole and aligned.  kPer 0: rows
// of any length, read twice.
template <typename T, int kThreads, int kRows, int kPer, bool kVec>
__global__ __launch_bounds__(kThreads *kRows) void add_rms_norm_rows(NormArgs a) {
  constexpr int kWaves = kThreads / 64;
  __shared__ double s_sum[kRows][kWaves];
  const int t = threadIdx.x % kThreads, r = threadIdx.x / kThreads;
  const uint32_t row = (blockIdx.y * gridDim.x + blockIdx.x) * kRows + r;
  const uint32_t token = min(row, a.tokens - 1);
  const bool live = row < a.tokens;
  const T *const x = static_cast<const T *>(a.x) + token * a.x_token;
  const T *const residual =
      a.residual ? static_cast<const T *>(a.residual) + token * a.residual_token : nullptr;
  const auto group = [&](uint32_t at, float (&h)[4]) __attribute__((always_inline)) {
    float other[4] = {};
    if constexpr (kVec) {
      if (at < a.n) {
        load_values<4>(h, x + at, true);
        if (residual)
          load_values<4>(other, residual + at, true);
      } else {
        h[0] = h[1] = h[2] = h[3] = 0.0f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = at + i < a.n;
        h[i] = in ? widen(x[at + i]) : 0.0f;
        other[i] = in && residual ? widen(residual[at + i]) : 0.0f;
      }
    }
    if (residual) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        h[i] += other[i];
    }
  };
  const auto put = [&](T *to, uint32_t at, const float (&v)[4]) __attribute__((always_inline)) {
    if constexpr (kVec) {
      if (at < a.n)
        store_values<4>(to + at, v, true);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + i < a.n)
          to[at + i] = narrow<T>(v[i]);
    }
  };
  const auto finish = [&](uint32_t at, const float (&h)[4], float c) __attribute__((always_inline)) {
    if (a.sum && live)
      put(static_cast<T *>(a.sum) + token * a.sum_token, at, h);
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = a.weight && at + i < a.n ? a.weight[at + i] : 1.0f;
      y[i] = h[i] * c * w;
    }
    if (a.y && live)
      put(static_cast<T *>(a.y) + token * a.y_token, at, y);
    if (a.q8 && live && at / kQK < a.n / kQK)  // the same in the eight lanes of a block
      store_q8_part(a.q8 + token * a.q8_token + static_cast<size_t>(at / kQK) * kQ8Bytes, t & 7, y);
  };

  constexpr int kHeld = kPer ? kPer : 1;
  float h[kHeld][4];
  double total = 0.0;
  const auto add = [&](const float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      total = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), total);
  };
  if constexpr (kPer) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      group(4 * (t + k * kThreads), h[k]);
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      add(h[k]);
  } else {
    for (uint32_t at = 4 * t; at < a.n; at += 4 * kThreads) {
      group(at, h[0]);
      add(h[0]);
    }
  }
  total = wave_sum(total);
  if constexpr (kWaves > 1) {
    if ((t & 63) == 0)
      s_sum[r][t >> 6] = total;
    __syncthreads();
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      total += s_sum[r][w];
  }
  const float c = static_cast<float>(1.0 / sqrt(total / a.n + a.eps));
  if constexpr (kPer) {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      finish(4 * (t + k * kThreads), h[k], c);
  } else {
    // a thread takes in the group before it writes there; eight lanes go on together, for a block of q8
    for (uint32_t at = 4 * t; at < (a.n + kQK - 1) / kQK * kQK; at += 4 * kThreads) {
      group(at, h[0]);
      finish(at, h[0], c);
    }
  }
}

template <typename T, int kThreads, int kRows, int kPer>
void launch(const NormArgs &a, bool vec, hipStream_t st) {
  // along x less than 2^32 threads
  const uint32_t groups = (a.tokens + kRows - 1) / kRows, most = 1u << 20;
  const dim3 grid(groups < most ? groups : most, (groups + most - 1) / most), block(kThreads * kRows);
  if (vec)
    add_rms_norm_rows<T, kThreads, kRows, kPer, true><<<grid, block, 0, st>>>(a);
  else
    add_rms_norm_rows<T, kThreads, kRows, kPer, false><<<grid, block, 0, st>>>(a);
}

template <typename T> void launch_elem(const NormArgs &a, bool vec, hipStream_t st) {
  if (a.n <= 1024)
    launch<T, 64, 4, 4>(a, vec, st);
  else if (a.n <= 4096)
    launch<T, 256, 1, 4>(a, vec, st);
  else if (a.n <= 16384)
    launch<T, kLongThreads, 1, 4>(a, vec, st);
  else
    launch<T, kLongThreads, 1, 0>(a, vec, st);
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
  const auto by_4 = [&](const void *p, size_t stride) {
    return !p || (aligned_to(p, 4 * size) && (tokens == 1 || stride % 4 == 0));
  };
  const bool vec = n % 4 == 0 && by_4(x, x_token) && by_4(residual, residual_token) &&
                   by_4(sum, sum_token) && by_4(y, y_token) && aligned16(weight);
  const tcrv::NormArgs a{x,       residual,       sum,       y,       weight,
                         q8,      x_token,        residual_token, sum_token, y_token,
                         q8_token, eps,           static_cast<uint32_t>(tokens),
                         static_cast<uint32_t>(n)};
  hipStream_t st = as_stream(stream);
  if (elem == TCRV_HIP_ELEM_F32)
    tcrv::launch_elem<float>(a, vec, st);
  else if (elem == TCRV_HIP_ELEM_F16)
    tcrv::launch_elem<_Float16>(a, vec, st);
  else
    tcrv::launch_elem<tcrv::Bf16>(a, vec, st);
  return launch_status();
}

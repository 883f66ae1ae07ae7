// kv_cache.h -- what the kernels over the paged Q4_0 cache share: the activations' element
// types, the layout of a page (include/tcrv_hip.h) and the rotation of a pair.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "tcrv_hip_internal.h"

namespace tcrv {

using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

struct Bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return static_cast<float>(x); }
__device__ __forceinline__ float widen(Bf16 x) {
  return __builtin_bit_cast(float, static_cast<uint32_t>(x.bits) << 16);
}

// Nearest even; a NaN stays one (its quiet bit is set, so that the cut leaves no infinity).
template <typename T> __device__ __forceinline__ T narrow(float x);
template <> __device__ __forceinline__ float narrow<float>(float x) { return x; }
template <> __device__ __forceinline__ _Float16 narrow<_Float16>(float x) {
  return static_cast<_Float16>(x);
}
template <> __device__ __forceinline__ Bf16 narrow<Bf16>(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const uint32_t up = u + 0x7fffu + ((u >> 16) & 1u);
  return Bf16{static_cast<uint16_t>((x != x ? (u | 0x400000u) : up) >> 16)};
}

// n values as one access, of 16 bytes at a time where they are more.
template <typename T, int n> struct alignas(n * sizeof(T) < 16 ? n * sizeof(T) : 16) Values {
  T v[n];
};

// `n` values from p, at once where `vec` says that p is aligned to them all, to 16 bytes at most.
template <int n, typename T>
__device__ __forceinline__ void load_values(float *out, const T *p, bool vec) {
  if (vec) {
    const Values<T, n> x = *reinterpret_cast<const Values<T, n> *>(p);
#pragma unroll
    for (int i = 0; i < n; ++i)
      out[i] = widen(x.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i)
      out[i] = widen(p[i]);
  }
}

template <int n, typename T>
__device__ __forceinline__ void store_values(T *p, const float *x, bool vec) {
  Values<T, n> y;
#pragma unroll
  for (int i = 0; i < n; ++i)
    y.v[i] = narrow<T>(x[i]);
  if (vec) {
    *reinterpret_cast<Values<T, n> *>(p) = y;
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i)
      p[i] = y.v[i];
  }
}

// One page's part of one head: byte offsets of its four regions, and of a token in them.
struct PageHead {
  uint32_t quants, scales;  // bytes of a region of quants, of scales

  __host__ __device__ PageHead(uint32_t page_size, uint32_t head_dim)
      : quants(page_size * head_dim / 2), scales(page_size * head_dim / 16) {}
  __host__ __device__ uint32_t bytes() const { return 2 * (quants + scales); }
  // dword g of block b of a token's keys
  __device__ uint32_t key(uint32_t nb, uint32_t token, uint32_t g, uint32_t b) const {
    return (token * 4 + g) * nb * 4 + b * 4;
  }
  // the 16-bit unit of byte m of blocks 2 pair and 2 pair + 1 of a token's values
  __device__ uint32_t value(uint32_t nb, uint32_t token, uint32_t m, uint32_t pair) const {
    return quants + scales + (((token >> 2) * 16 + m) * (nb / 2) + pair) * 8 + (token & 3) * 2;
  }
  __device__ uint32_t key_scale(uint32_t nb, uint32_t token, uint32_t b) const {
    return quants + ((token >> 2) * nb + b) * 8 + (token & 3) * 2;
  }
  __device__ uint32_t value_scale(uint32_t nb, uint32_t token, uint32_t b) const {
    return 2 * quants + scales + ((token >> 2) * nb + b) * 8 + (token & 3) * 2;
  }
};

}  // namespace tcrv

namespace tcrv_host {

// 0 for what is no activation type
inline size_t float_elem_bytes(int elem) {
  return elem == TCRV_HIP_ELEM_F32 ? 4
         : elem == TCRV_HIP_ELEM_F16 || elem == TCRV_HIP_ELEM_BF16 ? 2
                                                                   : 0;
}

inline bool aligned_to(const void *p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// A page's bytes have to fit the kernels' 32-bit offsets within a page's head, and heads a grid.
constexpr size_t kMostPageSize = 65536;
constexpr size_t kMostHeads = 65535;
// A launch holds less than 2^32 threads along an axis: work-groups of 256, one a token.
constexpr size_t kMostGroups = 0xffffffu, kMostTokens = kMostGroups;

inline bool cache_sizes_ok(size_t page_size, size_t kv_heads, size_t head_dim) {
  return page_size != 0 && page_size % 16 == 0 && page_size <= kMostPageSize && kv_heads != 0 &&
         kv_heads <= kMostHeads &&
         (head_dim == 64 || head_dim == 128 || head_dim == 192 || head_dim == 256);
}

// Whether groups of 4 values of every row lie on aligned places.
inline bool groups_of_4(const void *p, size_t token, size_t head, size_t size) {
  return aligned_to(p, 4 * size) && token % 4 == 0 && head % 4 == 0;
}

// Rows that are read: a head's row begins past the one before it, and a token's likewise.  In other
// pairs they may overlap.
inline bool strides_ok(size_t token, size_t head, size_t tokens, size_t heads, size_t dim) {
  return (heads <= 1 || head >= dim) && (tokens <= 1 || token >= dim);
}

// Rows that are written: no two of them overlap.  Token t's head h lies t * token + h * head on, so that
// i > 0 heads on and j > 0 tokens back must be a row away either way: looked at for the two j next to where
// these meet.
inline bool rows_apart(size_t token, size_t head, size_t tokens, size_t heads, size_t dim) {
  using Wide = unsigned __int128;
  if (!strides_ok(token, head, tokens, heads, dim))
    return false;
  if (tokens <= 1 || heads <= 1 || Wide{token} >= Wide{head} * (heads - 1) + dim ||
      Wide{head} >= Wide{token} * (tokens - 1) + dim)
    return true;
  if (token == 0)
    return dim == 0;
  for (size_t i = 1; i < heads; ++i) {
    const Wide on = Wide{head} * i, j = on / token;
    if (j >= 1 && j < tokens && on - j * token < dim)
      return false;
    if (j + 1 < tokens && (j + 1) * token - on < dim)
      return false;
  }
  return true;
}

}  // namespace tcrv_host

// kv_cache.hip -- the paged Q4_0 cache: block tables and slots, the store, and the reading back.
#include "kv_cache.h"

namespace tcrv {
namespace {

// ---------------------------------------------------------------------------
// Tables.  Two exclusive sums over the requests (added tokens, new pages) give every token and
// every new page its place; the token at place i then finds its request by a binary search in
// the sums.  All work-groups form the sums of all requests for themselves, kTableThreads requests
// at a time, and share out the tokens and the new pages: one launch, no order between work-groups.
// A slot in a new page is formed from free_pages itself, so that it does not wait for the table's
// entry, which another work-group writes.  64 requests of a token each 4.5 us, 301 of up to 700 tokens
// 6.8: a launch and four loads that follow one another.
// ---------------------------------------------------------------------------
constexpr int kTableThreads = 256;
constexpr int kTableWaves = kTableThreads / 64;

struct TablesArgs {
  const int32_t *context, *added, *free_pages;
  int32_t *block_table, *first, *length, *positions;
  int64_t *slots;
  int32_t *taken;
  size_t requests, free_count, table_stride, max_tokens;
  uint32_t page_size;
};

__device__ __forceinline__ int32_t saturated(int64_t x) {
  return static_cast<int32_t>(min(x, static_cast<int64_t>(0x7fffffff)));
}

// Inclusive sum over a wave.
__device__ __forceinline__ int64_t wave_sum(int64_t x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(x, d);
    x += lane >= d ? y : 0;
  }
  return x;
}

// The last of n ascending values (v[0] <= key) that is at most key.
__device__ __forceinline__ int last_at_most(const int64_t *v, int n, int64_t key) {
  int lo = 0;
  while (n > 1) {
    const int half = n >> 1;
    lo += v[lo + half] <= key ? half : 0;
    n -= half;
  }
  return lo;
}

__global__ __launch_bounds__(kTableThreads) void kv_tables(TablesArgs a) {
  __shared__ int64_t s_token[kTableThreads], s_page[kTableThreads];  // where a request's begin
  __shared__ int32_t s_context[kTableThreads], s_held[kTableThreads];
  __shared__ int64_t s_sums[2][kTableWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTableThreads;
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * kTableThreads + tid;
  const int64_t ps = a.page_size, stride = static_cast<int64_t>(a.table_stride);
  const int64_t most = static_cast<int64_t>(a.max_tokens);
  int64_t token0 = 0, page0 = 0;  // of the requests before this run of kTableThreads
  for (size_t base = 0; base < a.requests; base += kTableThreads) {
    const int n = static_cast<int>(min(a.requests - base, static_cast<size_t>(kTableThreads)));
    int64_t context = 0, added = 0, held = 0, need = 0;
    if (tid < n) {
      context = max(a.context[base + tid], 0);
      added = max(a.added[base + tid], 0);
      held = min((context + ps - 1) / ps, stride);
      need = min((context + added + ps - 1) / ps, stride);
    }
    const int64_t tokens = wave_sum(added, lane), pages = wave_sum(need - held, lane);
    if (lane == 63) {
      s_sums[0][wave] = tokens;
      s_sums[1][wave] = pages;
    }
    __syncthreads();
    int64_t token = token0 + tokens - added, page = page0 + pages - (need - held);
#pragma unroll
    for (int w = 0; w < kTableWaves; ++w) {
      token += w < wave ? s_sums[0][w] : 0;
      page += w < wave ? s_sums[1][w] : 0;
      token0 += s_sums[0][w];
      page0 += s_sums[1][w];
    }
    s_token[tid] = token;
    s_page[tid] = page;
    s_context[tid] = static_cast<int32_t>(context);
    s_held[tid] = static_cast<int32_t>(held);
    __syncthreads();
    if (blockIdx.x == 0 && tid < n) {
      a.first[base + tid] = saturated(token);
      a.length[base + tid] = saturated(context + added);
    }
    // the new pages and the tokens of these requests, by their places in all of them
    for (int64_t i = s_page[0] + mine; i < page0; i += step) {
      const int r = last_at_most(s_page, n, i);
      const int64_t column = s_held[r] + (i - s_page[r]);
      int32_t got = -1;
      if (static_cast<size_t>(i) < a.free_count)
        got = max(a.free_pages[i], -1);
      a.block_table[(base + r) * a.table_stride + column] = got;
    }
    for (int64_t i = s_token[0] + mine; i < token0 && i < most; i += step) {
      const int r = last_at_most(s_token, n, i);
      const int64_t position = s_context[r] + (i - s_token[r]);
      const int64_t column = position / ps;
      int64_t at = -1;
      if (column < s_held[r]) {
        at = a.block_table[(base + r) * a.table_stride + column];
      } else if (column < stride) {
        const int64_t k = s_page[r] + (column - s_held[r]);
        if (static_cast<size_t>(k) < a.free_count)
          at = a.free_pages[k];
      }
      a.positions[i] = saturated(position);
      a.slots[i] = at < 0 ? -1 : at * ps + (position - column * ps);
    }
    __syncthreads();  // before the next run's sums are written over these
  }
  for (int64_t i = token0 + mine; i < most; i += step) {
    a.positions[i] = -1;
    a.slots[i] = -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.first[a.requests] = saturated(token0);
    a.taken[0] = saturated(page0);
  }
}

// ---------------------------------------------------------------------------
// The store.  Bound by memory: keys and values read once, 9/16 byte an element written.  A block
// of 32 elements is 8 lanes of 4 (as in quantize_q8_0), a row of 16 lanes two blocks: the nibbles
// of a byte meet by a move of 4 lanes, and the two bytes of a unit of the values by one of 8.
// A work-group takes a token: 8191 tokens x 8 heads x 128, f32, 24 us for 81 MB that have to move.  It moves
// 98: a token's value bytes are 2 of every 8, beside those of three neighbours whose work-groups run on
// other XCDs, and 25 MB are written for 9.4.  The slot, the position and the table row come one after the
// other before 9 KB of work.  Four tokens a work-group, whose bytes leave 8 at a time, took 32 to 35 us, an
// item's loads sent before the one before it is worked on 33.
// ---------------------------------------------------------------------------
struct StoreArgs {
  const void *k, *v;
  const int32_t *positions;
  const float *table;
  const int64_t *slots;
  uint8_t *cache;
  size_t k_token, k_head, v_token, v_head;
  size_t table_rows, slots_in_all;
  uint32_t page_size, kv_heads, nb, n_dims;
  bool k_vec, v_vec, row_vec;  // aligned groups of 4 values, of 4 pairs
};

template <int kControl> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_mov_dpp(static_cast<int>(v), kControl, 0xf, 0xf, true));
}

__device__ __forceinline__ uint32_t max8_bits(uint32_t v) {
  v = max(v, dpp<0xB1>(v));         // lane ^ 1
  v = max(v, dpp<0x4E>(v));         // lane ^ 2
  return max(v, dpp<0x141>(v));     // the other four of eight
}

__device__ __forceinline__ uint32_t min8(uint32_t v) { return ~max8_bits(~v); }

// 4 elements of a block on each of 8 lanes -> their nibbles, a byte each; *scale the block's d.
__device__ __forceinline__ uint32_t quantize4(const float *x, int lane8, float *scale) {
  // magnitudes order as their bits do, and a NaN lies above infinity: it becomes the scale
  uint32_t mag[4], top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mag[i] = __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu;
    top = max(top, mag[i]);
  }
  top = max8_bits(top);
  uint32_t at = 64;  // twice the first place of the largest magnitude, and 1 if it is negative
#pragma unroll
  for (int i = 3; i >= 0; --i)
    if (mag[i] == top)
      at = 2 * (4 * lane8 + i) + (__builtin_bit_cast(uint32_t, x[i]) >> 31);
  at = min8(at);
  const float d = __builtin_bit_cast(float, top | (at & 1u) << 31) / -8.0f;
  const float id = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
  uint32_t q = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // in 0.5 .. 16.5 for finite blocks; fmaxf takes a NaN to 0
    const float t = fminf(fmaxf(x[i] * id + 8.5f, 0.0f), 15.0f);
    q |= static_cast<uint32_t>(t) << (8 * i);
  }
  // out of the compiler's sight: it would round the division to f16 as fma(x, -1/8, +0), which takes the
  // scale of an empty block from -0 to +0
  float kept = d;
  asm("" : "+v"(kept));
  *scale = kept;
  return q;
}

// The page of a slot that lies in the cache, by a 32-bit division where that does (the 64-bit one is long).
// A page takes 1152 bytes or more, so that pages number less than 2^32 in any memory.
__device__ __forceinline__ uint32_t page_of(int64_t slot, uint32_t page_size) {
  return slot >> 32 ? static_cast<uint32_t>(static_cast<uint64_t>(slot) / page_size)
                    : static_cast<uint32_t>(slot) / page_size;
}

// Lane i of a row of 16 takes lane i + kBy.
template <int kBy> __device__ __forceinline__ uint32_t from_lane_above(uint32_t v) {
  return dpp<0x100 + kBy>(v);
}

constexpr int kStoreThreads = 256;

// 4 elements of a key, those of places e .. e + 3 of `x`, turned.
template <typename T, bool kHalf>
__device__ __forceinline__ void turn4(float *v, const T *x, const float *row, uint32_t e,
                                      uint32_t n_dims, bool vec, bool row_vec) {
  if constexpr (kHalf) {
    const uint32_t half = n_dims / 2;
    if (half % 4 == 0) {  // the partners are four neighbours, n_dims / 2 away
      const bool second = e >= half;
      const uint32_t j = second ? e - half : e;
      float w[4], cs[8];
      load_values<4>(w, x + (second ? j : e + half), vec);
      load_values<8>(cs, row + 2 * j, row_vec);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = second ? w[i] * cs[2 * i + 1] + v[i] * cs[2 * i]
                      : v[i] * cs[2 * i] - w[i] * cs[2 * i + 1];
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = e + i;
      if (at < n_dims) {
        const bool second = at >= half;
        const uint32_t j = second ? at - half : at;
        const float c = row[2 * j], s = row[2 * j + 1];
        const float w = widen(x[second ? j : at + half]);
        v[i] = second ? w * s + v[i] * c : v[i] * c - w * s;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      if (e + i < n_dims) {
        const float c = row[e + i], s = row[e + i + 1];
        const float y = v[i] * c - v[i + 1] * s;
        v[i + 1] = v[i] * s + v[i + 1] * c;
        v[i] = y;
      }
    }
  }
}

template <typename T, bool kHalf>
__global__ __launch_bounds__(kStoreThreads) void kv_store_q4_0(StoreArgs a) {
  const size_t token = blockIdx.x;
  const int64_t slot = a.slots[token];
  if (slot < 0 || static_cast<size_t>(slot) >= a.slots_in_all)
    return;
  const uint32_t nb = a.nb, dim = nb * 32;
  const size_t page = page_of(slot, a.page_size);
  const uint32_t place = static_cast<uint32_t>(static_cast<size_t>(slot) - page * a.page_size);
  const PageHead lay(a.page_size, dim);
  uint8_t *const page_at = a.cache + page * lay.bytes() * a.kv_heads;
  const int lane16 = threadIdx.x & 15, lane8 = lane16 & 7;
  const float *row = nullptr;
  if (a.n_dims) {
    const int32_t p = a.positions[token];
    if (p >= 0 && static_cast<size_t>(p) < a.table_rows)
      row = a.table + static_cast<size_t>(p) * a.n_dims;
  }
  // an item: 64 elements of one head, keys first
  const uint32_t pairs = nb / 2, items = 2 * a.kv_heads * pairs;
  for (uint32_t item = blockIdx.y * (kStoreThreads / 16) + (threadIdx.x >> 4); item < items;
       item += gridDim.y * (kStoreThreads / 16)) {
    const uint32_t pair = item % pairs;
    uint32_t head = item / pairs;
    const bool values = head >= a.kv_heads;
    head -= values ? a.kv_heads : 0;
    const uint32_t e = pair * 64 + lane16 * 4;
    const T *x = values ? static_cast<const T *>(a.v) + token * a.v_token + head * a.v_head
                        : static_cast<const T *>(a.k) + token * a.k_token + head * a.k_head;
    const bool vec = values ? a.v_vec : a.k_vec;
    float v[4];
    load_values<4>(v, x + e, vec);
    if (!values && row && e < a.n_dims)
      turn4<T, kHalf>(v, x, row, e, a.n_dims, vec, a.row_vec);
    float d;
    uint32_t q = quantize4(v, lane8, &d);
    q |= from_lane_above<4>(q) << 4;  // lanes 0..3 of 8: bytes 4 lane8 .. + 3 of the block
    const uint32_t b = 2 * pair + (lane16 >> 3);
    uint8_t *const at = page_at + static_cast<size_t>(head) * lay.bytes();
    if (lane8 == 0)
      *reinterpret_cast<_Float16 *>(
          at + (values ? lay.value_scale(nb, place, b) : lay.key_scale(nb, place, b))) =
          static_cast<_Float16>(d);
    if (!values) {
      if (lane8 < 4)
        *reinterpret_cast<uint32_t *>(at + lay.key(nb, place, lane8, b)) = q;
    } else {
      const uint32_t other = from_lane_above<8>(q);  // lanes 0..3 of 16: block 2 pair + 1's
      if (lane16 < 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint16_t *>(at + lay.value(nb, place, 4 * lane16 + i, pair)) =
              static_cast<uint16_t>((q >> (8 * i) & 255u) | (other >> (8 * i) & 255u) << 8);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The reading back: (q - 8) d is exact in f32.  The lanes' places as in the store; 8191 tokens as there
// 26 us for 77 MB: 102 move, 35 of the cache for the 9.4 that are there, by the neighbours' shared lines.
// ---------------------------------------------------------------------------
struct LoadArgs {
  const uint8_t *cache;
  const int64_t *slots;
  void *k, *v;
  size_t k_token, k_head, v_token, v_head;
  size_t slots_in_all;
  uint32_t page_size, kv_heads, nb;
  bool k_vec, v_vec;
};

template <typename T>
__global__ __launch_bounds__(kStoreThreads) void kv_load_q4_0(LoadArgs a) {
  const size_t token = blockIdx.x;
  const int64_t slot = a.slots[token];
  const bool known = slot >= 0 && static_cast<size_t>(slot) < a.slots_in_all;
  const uint32_t nb = a.nb, dim = nb * 32;
  const size_t page = known ? page_of(slot, a.page_size) : 0;
  const uint32_t place =
      known ? static_cast<uint32_t>(static_cast<size_t>(slot) - page * a.page_size) : 0;
  const PageHead lay(a.page_size, dim);
  const uint8_t *const page_at = a.cache + page * lay.bytes() * a.kv_heads;
  const int lane16 = threadIdx.x & 15, lane8 = lane16 & 7, byte = 4 * (lane8 & 3);
  const uint32_t pairs = nb / 2, items = 2 * a.kv_heads * pairs;
  for (uint32_t item = blockIdx.y * (kStoreThreads / 16) + (threadIdx.x >> 4); item < items;
       item += gridDim.y * (kStoreThreads / 16)) {
    const uint32_t pair = item % pairs;
    uint32_t head = item / pairs;
    const bool values = head >= a.kv_heads;
    head -= values ? a.kv_heads : 0;
    const uint32_t b = 2 * pair + (lane16 >> 3);
    const uint8_t *const at = page_at + static_cast<size_t>(head) * lay.bytes();
    float v[4] = {};
    if (known) {
      const float d = static_cast<float>(*reinterpret_cast<const _Float16 *>(
          at + (values ? lay.value_scale(nb, place, b) : lay.key_scale(nb, place, b))));
      uint32_t q = 0;
      if (values) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q |= static_cast<uint32_t>(at[lay.value(nb, place, byte + i, pair) + (b & 1)]) << (8 * i);
      } else {
        q = *reinterpret_cast<const uint32_t *>(at + lay.key(nb, place, lane8 & 3, b));
      }
      q >>= lane8 >= 4 ? 4 : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = static_cast<float>(static_cast<int>(q >> (8 * i) & 15u) - 8) * d;
    }
    T *y = values ? static_cast<T *>(a.v) + token * a.v_token + head * a.v_head
                  : static_cast<T *>(a.k) + token * a.k_token + head * a.k_head;
    store_values<4>(y + pair * 64 + lane16 * 4, v, values ? a.v_vec : a.k_vec);
  }
}

}  // namespace
}  // namespace tcrv

namespace {

// Work-groups of 16 items a token: enough for few tokens, else one that walks all of them.
unsigned item_groups(size_t tokens, size_t items) {
  const size_t all = (items + 15) / 16, wanted = (2048 + tokens - 1) / tokens;
  return static_cast<unsigned>(all < wanted ? all : wanted);
}

}  // namespace

extern "C" {

size_t tcrv_hip_kv_q4_0_page_bytes(size_t page_size, size_t kv_heads, size_t head_dim) {
  if (!tcrv_host::cache_sizes_ok(page_size, kv_heads, head_dim))
    return 0;
  return static_cast<size_t>(tcrv::PageHead(static_cast<uint32_t>(page_size),
                                            static_cast<uint32_t>(head_dim))
                                 .bytes()) *
         kv_heads;
}

int tcrv_hip_kv_tables(const int32_t *context, const int32_t *added, size_t requests,
                       size_t page_size, const int32_t *free_pages, size_t free_count,
                       int32_t *block_table, size_t table_stride, int32_t *first,
                       int32_t *length, int32_t *positions, int64_t *slots, size_t max_tokens,
                       int32_t *taken, void *stream) {
  using namespace tcrv_host;
  if (page_size == 0 || page_size > kMostPageSize)
    return TCRV_HIP_ERR_BAD_SIZE;
  if (!first || !taken || (requests && (!context || !added || !length)) ||
      (requests && table_stride && !block_table) || (free_count && !free_pages) ||
      (max_tokens && (!positions || !slots)))
    return TCRV_HIP_ERR_NULL_POINTER;
  for (const void *p : {static_cast<const void *>(context), static_cast<const void *>(added),
                        static_cast<const void *>(free_pages),
                        static_cast<const void *>(block_table), static_cast<const void *>(first),
                        static_cast<const void *>(length), static_cast<const void *>(positions),
                        static_cast<const void *>(taken)})
    if (!aligned4(p))
      return TCRV_HIP_ERR_MISALIGNED;
  if (!aligned_to(slots, 8))
    return TCRV_HIP_ERR_MISALIGNED;
  if (requests > 0x7fffffffu || max_tokens > 0x7fffffffu || table_stride > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  tcrv::TablesArgs a{context, added,  free_pages, block_table, first,        length,     positions,
                     slots,   taken,  requests,   free_count,  table_stride, max_tokens,
                     static_cast<uint32_t>(page_size)};
  const size_t groups = (max_tokens + tcrv::kTableThreads - 1) / tcrv::kTableThreads;
  tcrv::kv_tables<<<dim3(static_cast<unsigned>(groups < 1 ? 1 : groups > 512 ? 512 : groups)),
                    dim3(tcrv::kTableThreads), 0, as_stream(stream)>>>(a);
  return launch_status();
}

int tcrv_hip_kv_store_q4_0(int elem, const void *k, size_t k_token, size_t k_head, const void *v,
                           size_t v_token, size_t v_head, int layout, const int32_t *positions,
                           const float *table, size_t table_rows, size_t n_dims,
                           const int64_t *slots, uint8_t *cache, size_t pages, size_t page_size,
                           size_t tokens, size_t kv_heads, size_t head_dim, void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem);
  if (!size || (n_dims && layout != TCRV_HIP_ROPE_INTERLEAVED && layout != TCRV_HIP_ROPE_HALF))
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (!cache_sizes_ok(page_size, kv_heads, head_dim) || n_dims % 2 || n_dims > head_dim ||
      !strides_ok(k_token, k_head, tokens, kv_heads, head_dim) ||
      !strides_ok(v_token, v_head, tokens, kv_heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (tokens == 0)
    return TCRV_HIP_OK;
  if (!k || !v || !slots || (!cache && pages) || (n_dims && (!positions || (!table && table_rows))))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(k, size) || !aligned_to(v, size) || !aligned_to(slots, 8) || !aligned16(cache) ||
      (n_dims && (!aligned4(positions) || !aligned4(table))))
    return TCRV_HIP_ERR_MISALIGNED;
  if (tokens > kMostTokens || pages > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  const uint32_t nb = static_cast<uint32_t>(head_dim / 32);
  tcrv::StoreArgs a{k,       v,       positions, table,      slots,
                    cache,   k_token, k_head,    v_token,    v_head,
                    table_rows, pages * page_size, static_cast<uint32_t>(page_size),
                    static_cast<uint32_t>(kv_heads), nb, static_cast<uint32_t>(n_dims),
                    groups_of_4(k, k_token, k_head, size), groups_of_4(v, v_token, v_head, size),
                    aligned16(table) && n_dims % 4 == 0};
  const dim3 grid(static_cast<unsigned>(tokens), item_groups(tokens, kv_heads * nb));
  const dim3 block(tcrv::kStoreThreads);
  hipStream_t st = as_stream(stream);
  const bool half = layout == TCRV_HIP_ROPE_HALF;
  switch (elem) {
  case TCRV_HIP_ELEM_F32:
    half ? tcrv::kv_store_q4_0<float, true><<<grid, block, 0, st>>>(a)
         : tcrv::kv_store_q4_0<float, false><<<grid, block, 0, st>>>(a);
    break;
  case TCRV_HIP_ELEM_F16:
    half ? tcrv::kv_store_q4_0<_Float16, true><<<grid, block, 0, st>>>(a)
         : tcrv::kv_store_q4_0<_Float16, false><<<grid, block, 0, st>>>(a);
    break;
  default:
    half ? tcrv::kv_store_q4_0<tcrv::Bf16, true><<<grid, block, 0, st>>>(a)
         : tcrv::kv_store_q4_0<tcrv::Bf16, false><<<grid, block, 0, st>>>(a);
    break;
  }
  return launch_status();
}

int tcrv_hip_kv_load_q4_0(int elem, const uint8_t *cache, size_t pages, size_t page_size,
                          const int64_t *slots, void *k, size_t k_token, size_t k_head, void *v,
                          size_t v_token, size_t v_head, size_t tokens, size_t kv_heads,
                          size_t head_dim, void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem);
  if (!size)
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (!cache_sizes_ok(page_size, kv_heads, head_dim) ||
      !strides_ok(k_token, k_head, tokens, kv_heads, head_dim) ||
      !strides_ok(v_token, v_head, tokens, kv_heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (tokens == 0)
    return TCRV_HIP_OK;
  if (!k || !v || !slots || (!cache && pages))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(k, size) || !aligned_to(v, size) || !aligned_to(slots, 8) || !aligned16(cache))
    return TCRV_HIP_ERR_MISALIGNED;
  if (tokens > kMostTokens || pages > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (!rows_apart(k_token, k_head, tokens, kv_heads, head_dim) ||
      !rows_apart(v_token, v_head, tokens, kv_heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  const uint32_t nb = static_cast<uint32_t>(head_dim / 32);
  tcrv::LoadArgs a{cache,   slots,  k, v, k_token, k_head, v_token, v_head, pages * page_size,
                   static_cast<uint32_t>(page_size), static_cast<uint32_t>(kv_heads), nb,
                   groups_of_4(k, k_token, k_head, size), groups_of_4(v, v_token, v_head, size)};
  const dim3 grid(static_cast<unsigned>(tokens), item_groups(tokens, kv_heads * nb));
  const dim3 block(tcrv::kStoreThreads);
  hipStream_t st = as_stream(stream);
  switch (elem) {
  case TCRV_HIP_ELEM_F32:
    tcrv::kv_load_q4_0<float><<<grid, block, 0, st>>>(a);
    break;
  case TCRV_HIP_ELEM_F16:
    tcrv::kv_load_q4_0<_Float16><<<grid, block, 0, st>>>(a);
    break;
  default:
    tcrv::kv_load_q4_0<tcrv::Bf16><<<grid, block, 0, st>>>(a);
    break;
  }
  return launch_status();
}

}  // extern "C"

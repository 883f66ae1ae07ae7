// tree.hip -- drafted tokens as a tree: what each of them sees of the others and its position, and the
// accepted path's rows of the paged Q4_0 cache to the places after the cached tokens.
#include <algorithm>

#include "kv_cache.h"

namespace tcrv {
namespace {

// A request's new tokens: where they begin in its step's rows, how many, and the tokens cached before.
struct Nodes {
  int first, count, cached;
  __device__ Nodes(const int32_t *begins, const int32_t *length, uint32_t request, uint32_t most) {
    const int begin = max(begins[request], 0), end = max(begins[request + 1], 0);
    first = begin;
    count = max(min(end, static_cast<int>(most)) - begin, 0);
    cached = max(length[request], 0) - max(end - begin, 0);
  }
};

constexpr int kTreeThreads = 256;
constexpr int kTreeHeld = 4096;  // nodes in LDS, whole words

// A work-group a request.  First a wave takes 64 nodes, those of one word of bits, and each node's ancestors
// among them: a lane holds the nodes of its path up to another lane's, or out of the word, and takes on that
// one's, so that six turns reach the top.  Then a thread takes a node and goes from word to word: its own
// nodes there, then those of the ancestor at which its path enters the next.  Latency bounds it: 4 requests
// of 64 nodes and 301 of 17 2.7 us each, where an empty kernel takes 1.5 us (node by node 3.7 and 3.5); a chain
// of 64 4.0 us, of 1024 13 us (8.9 and 444).  The work-groups past the requests' fill what lies past the last
// token.
__global__ __launch_bounds__(kTreeThreads) void tree_tables(const int32_t *parents,
                                                            const int32_t *first,
                                                            const int32_t *length,
                                                            uint32_t requests, uint64_t *ancestors,
                                                            size_t words, int32_t *positions,
                                                            uint32_t tokens) {
  __shared__ uint64_t s_path[kTreeHeld];  // the node and its ancestors in its word
  __shared__ int32_t s_up[kTreeHeld];     // the first ancestor in a word below; -1 for none
  if (blockIdx.x >= requests) {
    const uint64_t end = requests ? max(first[requests], 0) : 0;
    const uint64_t by = static_cast<uint64_t>(gridDim.x - requests) * kTreeThreads;
    for (uint64_t i = end + (blockIdx.x - requests) * kTreeThreads + threadIdx.x; i < tokens; i += by) {
      positions[i] = -1;
      for (size_t w = 0; w < words; ++w)
        ancestors[i * words + w] = 0;
    }
    return;
  }
  const Nodes nodes(first, length, blockIdx.x, tokens);
  const int32_t *const mine = parents + nodes.first;
  const auto parent = [&](int i) {
    const int up = mine[i];
    return up < i ? max(up, -1) : -1;
  };
  const int lane = threadIdx.x & 63, held = min(nodes.count, kTreeHeld);
  for (int i0 = threadIdx.x - lane; i0 < held; i0 += kTreeThreads) {
    const int i = i0 + lane;
    uint64_t path = 1ull << lane;
    int up = i < held ? parent(i) : -1;
    for (int turn = 0; turn < 6 && __any(up >= i0); ++turn) {
      const int from = up >= i0 ? up - i0 : lane;
      const uint64_t its = __shfl(path, from);
      const int its_up = __shfl(up, from);
      if (up >= i0) {
        path |= its;
        up = its_up;
      }
    }
    if (i < held) {
      s_path[i] = path;
      s_up[i] = up;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nodes.count; i += kTreeThreads) {
    uint64_t *const row = ancestors + (static_cast<size_t>(nodes.first) + i) * words;
    int at = i, depth = -1;
    size_t word = words;  // those from here on are written
    while (at >= 0) {
      const size_t w = static_cast<size_t>(at) >> 6;
      uint64_t path = 0;
      int up = at;
      if (at < held) {
        path = s_path[at];
        up = s_up[at];
      } else {
        do {
          path |= 1ull << (up & 63);
          up = parent(up);
        } while (up >= 0 && static_cast<size_t>(up) >> 6 == w);
      }
      while (word > w) {
        --word;
        row[word] = word == w ? path : 0;
      }
      depth += __popcll(path);
      at = up;
    }
    while (word > 0)
      row[--word] = 0;
    positions[nodes.first + i] = nodes.cached + depth;
  }
}

// A row's bytes of one head in units of 16 bits: keys' quants lie side by side, the others 8 bytes apart.
struct RowUnits {
  uint32_t nb, keys, all;
  __device__ explicit RowUnits(uint32_t head_dim)
      : nb(head_dim / kQK), keys(head_dim / 4), all(2 * (keys + nb)) {}
  __device__ uint32_t at(const PageHead &lay, uint32_t token, uint32_t unit) const {
    if (unit < keys)
      return lay.key(nb, token, 0, 0) + 2 * unit;
    unit -= keys;
    if (unit < nb)
      return lay.key_scale(nb, token, unit);
    unit -= nb;
    if (unit < keys)
      return lay.value(nb, token, 0, 0) + 8 * unit;
    return lay.value_scale(nb, token, unit - keys);
  }
};

struct KeepArgs {
  uint8_t *cache;
  const int32_t *block_table, *first, *length, *path, *count;
  size_t table_stride, path_stride;
  uint32_t pages, page_size, max_added, kv_heads, head_dim;
};

constexpr int kKeepWaves = 4, kKeepTokens = 16;
constexpr int kKeepUnits = 2 * (256 / 4 + 256 / kQK);  // at most, of a row

// A work-group a request and head takes kKeepTokens nodes of the path at a time, a wave every fourth of
// them: their rows into registers, then from there to their places.  Nodes ascend and lie at or past
// their new places, so that what is still to be read lies past what has been written.  A thread a node
// looks up both places first: the chain of reads (path, table, row) bounds the call.  The rows' units of
// 16 bits lie in lines that hold four tokens', so that more is moved than the rows' bytes.  128 requests of
// 64 drafted tokens, 8 heads of 128: 7.6 us (12.9 us with a look-up for each unit and the rows in LDS);
// one request of 7: 2.7 us, where an empty kernel takes 1.5 us.
__global__ __launch_bounds__(kKeepWaves * 64) void kv_keep_q4_0(KeepArgs a) {
  struct Move {
    const uint8_t *source;  // the head's part of the page; nullptr: stays
    uint8_t *target;
    uint32_t from, to;  // tokens there
  };
  __shared__ Move s_move[kKeepTokens];
  constexpr int kTurns = kKeepTokens / kKeepWaves, kRounds = (kKeepUnits + 63) / 64;
  const uint32_t request = blockIdx.x, head = blockIdx.y;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int32_t *const path = a.path + request * a.path_stride;
  const int stride = static_cast<int>(min(a.path_stride, static_cast<size_t>(a.max_added)));
  int node = threadIdx.x < kKeepTokens && static_cast<int>(threadIdx.x) < stride ? path[threadIdx.x] : -1;
  const Nodes nodes(a.first, a.length, request, 0x7fffffffu);
  const int most = min(nodes.count, static_cast<int>(a.max_added));
  const int count = min(a.count[request], min(most, stride));
  const PageHead lay(a.page_size, a.head_dim);
  const RowUnits units(a.head_dim);
  const int32_t *const table = a.block_table + request * a.table_stride;
  // the head's part of the page of the request's token t, and its place there; nullptr where there is none
  const auto place = [&](int64_t t, uint32_t &token) -> uint8_t * {
    if (t < 0 || static_cast<size_t>(t) / a.page_size >= a.table_stride)
      return nullptr;
    const uint32_t column = static_cast<uint32_t>(t) / a.page_size;
    token = static_cast<uint32_t>(t) - column * a.page_size;
    const uint32_t page = static_cast<uint32_t>(table[column]);
    return page < a.pages ? a.cache + (static_cast<size_t>(page) * a.kv_heads + head) * lay.bytes()
                          : nullptr;
  };
  for (int k0 = 0; k0 < count; k0 += kKeepTokens) {
    if (threadIdx.x < kKeepTokens) {
      const int k = k0 + static_cast<int>(threadIdx.x);
      if (k0)
        node = k < count ? path[k] : -1;
      Move move{nullptr, nullptr, 0, 0};
      if (k < count && node != k && node >= 0 && node < most) {
        move.source = place(static_cast<int64_t>(nodes.cached) + node, move.from);
        move.target = place(static_cast<int64_t>(nodes.cached) + k, move.to);
        if (!move.target)
          move.source = nullptr;
      }
      s_move[threadIdx.x] = move;
    }
    __syncthreads();
    uint16_t row[kTurns][kRounds];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const Move &move = s_move[wave + i * kKeepWaves];
#pragma unroll
      for (int j = 0; j < kRounds; ++j)
        if (move.source && lane + 64u * j < units.all)
          row[i][j] = *reinterpret_cast<const uint16_t *>(
              move.source + units.at(lay, move.from, lane + 64 * j));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      const Move &move = s_move[wave + i * kKeepWaves];
#pragma unroll
      for (int j = 0; j < kRounds; ++j)
        if (move.source && lane + 64u * j < units.all)
          *reinterpret_cast<uint16_t *>(move.target + units.at(lay, move.to, lane + 64 * j)) =
              row[i][j];
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace tcrv

extern "C" {

int tcrv_hip_tree_tables(const int32_t *parents, const int32_t *first, const int32_t *length,
                         size_t requests, uint64_t *ancestors, size_t words, int32_t *positions,
                         size_t max_tokens, void *stream) {
  using namespace tcrv_host;
  if (max_tokens == 0)
    return TCRV_HIP_OK;
  if (max_tokens > 0x7fffffffu || requests >= kMostGroups || words > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (words == 0)
    return TCRV_HIP_ERR_BAD_SIZE;
  if (!ancestors || !positions || (requests && (!parents || !first || !length)))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(ancestors, 8) || !aligned4(positions) || !aligned4(parents) || !aligned4(first) ||
      !aligned4(length))
    return TCRV_HIP_ERR_MISALIGNED;
  // what may lie past the last token: a pass of up to 256 work-groups
  const size_t fill = std::min({(max_tokens - 1) / tcrv::kTreeThreads + 1, size_t{256}, kMostGroups - requests});
  tcrv::tree_tables<<<dim3(static_cast<unsigned>(requests + fill)), dim3(tcrv::kTreeThreads), 0,
                      as_stream(stream)>>>(parents, first, length, static_cast<uint32_t>(requests),
                                           ancestors, words, positions,
                                           static_cast<uint32_t>(max_tokens));
  return launch_status();
}

int tcrv_hip_kv_keep_q4_0(uint8_t *cache, size_t pages, size_t page_size, const int32_t *block_table,
                          size_t table_stride, const int32_t *first, const int32_t *length,
                          const int32_t *path, size_t path_stride, const int32_t *count,
                          size_t requests, size_t max_added, size_t kv_heads, size_t head_dim,
                          void *stream) {
  using namespace tcrv_host;
  if (!cache_sizes_ok(page_size, kv_heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (requests == 0 || max_added == 0 || path_stride == 0 || pages == 0 || table_stride == 0)
    return TCRV_HIP_OK;
  if (requests > kMostGroups || max_added > 0x7fffffffu || pages > 0x7fffffffu ||
      table_stride > 0x7fffffffu)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (!cache || !block_table || !first || !length || !path || !count)
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned16(cache) || !aligned4(block_table) || !aligned4(first) || !aligned4(length) ||
      !aligned4(path) || !aligned4(count))
    return TCRV_HIP_ERR_MISALIGNED;
  const tcrv::KeepArgs a{cache,
                         block_table,
                         first,
                         length,
                         path,
                         count,
                         table_stride,
                         path_stride,
                         static_cast<uint32_t>(pages),
                         static_cast<uint32_t>(page_size),
                         static_cast<uint32_t>(max_added),
                         static_cast<uint32_t>(kv_heads),
                         static_cast<uint32_t>(head_dim)};
  tcrv::kv_keep_q4_0<<<dim3(static_cast<unsigned>(requests), static_cast<unsigned>(kv_heads)),
                       dim3(tcrv::kKeepWaves * 64), 0, as_stream(stream)>>>(a);
  return launch_status();
}

}  // extern "C"

// rope.hip -- rotary positions: the table of cosines and sines, and the turn.
#include "kv_cache.h"

namespace tcrv {
namespace {

// ---------------------------------------------------------------------------
// The table.  Angles of a position past 2^17 need more than f32's 24 bits, so they are formed in
// f64 and reduced there.  A thread makes kTableRows rows of one pair, so that the power is taken
// once for all of them.  131072 rows of 64 pairs 34 us (67 MB, 14 us at a copy's rate), of 32 pairs 31, 4096
// rows 5.9: a thread's 16 sines in turn, on one of a work-group's four waves up to 64 pairs.  It runs once, or
// as contexts grow.
// ---------------------------------------------------------------------------
constexpr int kTableThreads = 256;
constexpr int kTableRows = 16;

struct TableForm {
  double log2_base, low, inverse_span, inverse_factor, amplitude;
  int ramp;  // whether pairs past `low` go over to the stretched positions
};

__global__ __launch_bounds__(kTableThreads) void rope_table(float2 *table, const float *divisors,
                                                            uint32_t pairs, uint64_t first,
                                                            uint64_t count, TableForm form) {
  const uint32_t i = blockIdx.y * kTableThreads + threadIdx.x;
  if (i >= pairs)
    return;
  double f = exp2(-form.log2_base * (static_cast<double>(i) / pairs));
  if (divisors)
    f /= static_cast<double>(divisors[i]);
  double r = 1.0;
  if (form.ramp)
    r = fmin(fmax((i - form.low) * form.inverse_span, 0.0), 1.0);
  f = f * (1.0 - r) + f * form.inverse_factor * r;
  for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * kTableRows, k = 0;
       k < kTableRows && row < count; ++k, ++row) {
    double s, c;
    sincos(static_cast<double>(first + row) * f, &s, &c);
    table[row * pairs + i] = make_float2(static_cast<float>(c * form.amplitude),
                                         static_cast<float>(s * form.amplitude));
  }
}

// ---------------------------------------------------------------------------
// The turn.  Bound by memory: x is read and y written once, and a token's table row (8 bytes a
// pair, against 8 to 16 a pair and head) is read once a thread for all heads that the thread turns.
// A thread holds kPairs pairs of one place in the head and walks the heads of its work-group.
// 4096 tokens x 32 heads x 128, f32, 64 elements turned: 23 us with the operands in the last-level
// cache, 29 from memory (135 MB, 4.6 TB/s); 7 tokens: 2.9, a launch.
// ---------------------------------------------------------------------------
struct RopeArgs {
  const void *x;
  void *y;
  const int32_t *positions;
  const float *table;
  size_t x_token, x_head, y_token, y_head;
  size_t table_rows;
  uint32_t heads, heads_a_group, head_dim, n_dims;
  float sign;  // of the sines
};

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
  const float ya = a * c - b * s;
  b = a * s + b * c;
  a = ya;
}

// kPairs pairs at a time where all is aligned and whole, else one.
template <typename T, bool kHalf, int kPairs>
__global__ __launch_bounds__(256) void rope(RopeArgs a) {
  constexpr bool kWide = kPairs > 1;
  const uint32_t turned = a.n_dims / (2 * kPairs);
  // copied: the elements past n_dims, as many at once as a turn holds, or one by one
  constexpr uint32_t kCopy = kPairs == 1 ? 1 : 2 * kPairs;
  const uint32_t units = turned + (a.head_dim - a.n_dims) / kCopy;
  const size_t token = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + token * a.x_token;
  T *y = static_cast<T *>(a.y) + token * a.y_token;
  const int32_t p = a.positions[token];
  const bool known = p >= 0 && static_cast<size_t>(p) < a.table_rows;
  const float *row = a.table + (known ? static_cast<size_t>(p) : 0) * a.n_dims;
  const uint32_t head0 = blockIdx.y * a.heads_a_group;
  const uint32_t head1 = min(a.heads, head0 + a.heads_a_group);
  const uint32_t side = blockDim.x / units ? blockDim.x / units : 1;  // heads beside one another
  for (uint32_t at = threadIdx.x; at < units * side; at += blockDim.x) {
    const uint32_t u = at % units;
    const bool turns = u < turned;
    float c[kPairs] = {}, s[kPairs] = {};
    if (turns && known) {
      float cs[2 * kPairs];
      load_values<2 * kPairs>(cs, row + u * 2 * kPairs, kWide);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        c[i] = cs[2 * i];
        s[i] = cs[2 * i + 1] * a.sign;
      }
    }
    for (uint32_t h = head0 + at / units; h < head1; h += side) {
      const T *xh = x + h * a.x_head;
      T *yh = y + h * a.y_head;
      if (!turns) {
        const uint32_t e = a.n_dims + (u - turned) * kCopy;
        float v[kCopy];
        load_values<kCopy>(v, xh + e, kWide);
        store_values<kCopy>(yh + e, v, kWide);
      } else if constexpr (kHalf) {
        const uint32_t e = u * kPairs, f = e + a.n_dims / 2;
        float v[kPairs], w[kPairs];
        load_values<kPairs>(v, xh + e, kWide);
        load_values<kPairs>(w, xh + f, kWide);
        if (known) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            turn(v[i], w[i], c[i], s[i]);
        }
        store_values<kPairs>(yh + e, v, kWide);
        store_values<kPairs>(yh + f, w, kWide);
      } else {
        const uint32_t e = u * 2 * kPairs;
        float v[2 * kPairs];
        load_values<2 * kPairs>(v, xh + e, kWide);
        if (known) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i)
            turn(v[2 * i], v[2 * i + 1], c[i], s[i]);
        }
        store_values<2 * kPairs>(yh + e, v, kWide);
      }
    }
  }
}

}  // namespace
}  // namespace tcrv

namespace {

bool positive(double x) { return x > 0.0 && x <= 1.0e300; }  // not NaN, not infinite

template <typename T>
void launch_rope(const tcrv::RopeArgs &a, bool half, bool wide, dim3 grid, uint32_t threads,
                 hipStream_t st) {
  if (half && wide)
    tcrv::rope<T, true, 4><<<grid, dim3(threads), 0, st>>>(a);
  else if (half)
    tcrv::rope<T, true, 1><<<grid, dim3(threads), 0, st>>>(a);
  else if (wide)
    tcrv::rope<T, false, 4><<<grid, dim3(threads), 0, st>>>(a);
  else
    tcrv::rope<T, false, 1><<<grid, dim3(threads), 0, st>>>(a);
}

}  // namespace

extern "C" {

int tcrv_hip_rope_table(int scaling, size_t n_dims, double base, double factor,
                        double trained_context, double beta_fast, double beta_slow,
                        double amplitude, const float *divisors, size_t first, size_t count,
                        float *table, void *stream) {
  using namespace tcrv_host;
  if (scaling < TCRV_HIP_ROPE_SCALE_NONE || scaling > TCRV_HIP_ROPE_SCALE_YARN)
    return TCRV_HIP_ERR_UNSUPPORTED;
  const bool yarn = scaling == TCRV_HIP_ROPE_SCALE_YARN;
  if (n_dims == 0 || n_dims % 2 || !positive(base) || !(amplitude >= 0.0 && amplitude <= 1.0e30))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (scaling != TCRV_HIP_ROPE_SCALE_NONE && !positive(factor))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (scaling == TCRV_HIP_ROPE_SCALE_NTK && n_dims == 2)
    return TCRV_HIP_ERR_BAD_SIZE;
  if (yarn && (!positive(trained_context) || !positive(beta_fast) || !positive(beta_slow) ||
               beta_fast < beta_slow || !(base > 1.0)))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (count == 0)
    return TCRV_HIP_OK;
  if (!table)
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(table, 8) || !aligned4(divisors))
    return TCRV_HIP_ERR_MISALIGNED;
  const size_t pairs = n_dims / 2;
  const size_t gx = (count - 1) / tcrv::kTableRows + 1;
  const size_t gy = (pairs + tcrv::kTableThreads - 1) / tcrv::kTableThreads;
  if (gx > kMostGroups || gy > 65535u || first > (1ull << 52) || count > (1ull << 52))
    return TCRV_HIP_ERR_TOO_LARGE;
  const double n = static_cast<double>(n_dims);
  tcrv::TableForm form{log2(base), 0.0, 0.0, 1.0, amplitude > 0.0 ? amplitude : 1.0, 0};
  if (scaling == TCRV_HIP_ROPE_SCALE_LINEAR || yarn)
    form.inverse_factor = 1.0 / factor;
  if (scaling == TCRV_HIP_ROPE_SCALE_NTK)
    form.log2_base += log2(factor) * n / (n - 2.0);
  if (yarn) {
    // the pair that turns beta times over the trained context: base^(2 i / n) 2 pi beta = context
    const auto place = [&](double beta) {
      return n * log(trained_context / (beta * 2.0 * M_PI)) / (2.0 * log(base));
    };
    const double low = fmax(floor(place(beta_fast)), 0.0);
    const double high = fmin(ceil(place(beta_slow)), n - 1.0);
    form.ramp = 1;
    form.low = low;
    form.inverse_span = 1.0 / fmax(high - low, 0.001);
    if (!(amplitude > 0.0))
      form.amplitude = 0.1 * log(factor) + 1.0;
  }
  tcrv::rope_table<<<dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)),
                     dim3(tcrv::kTableThreads), 0, as_stream(stream)>>>(
      reinterpret_cast<float2 *>(table), divisors, static_cast<uint32_t>(pairs), first, count,
      form);
  return launch_status();
}

int tcrv_hip_rope(int elem, int layout, const void *x, size_t x_token, size_t x_head, void *y,
                  size_t y_token, size_t y_head, const int32_t *positions, const float *table,
                  size_t table_rows, size_t tokens, size_t heads, size_t head_dim, size_t n_dims,
                  int inverse, void *stream) {
  using namespace tcrv_host;
  const size_t size = float_elem_bytes(elem);
  if (!size || (layout != TCRV_HIP_ROPE_INTERLEAVED && layout != TCRV_HIP_ROPE_HALF))
    return TCRV_HIP_ERR_UNSUPPORTED;
  if (n_dims % 2 || n_dims > head_dim || !strides_ok(x_token, x_head, tokens, heads, head_dim) ||
      !strides_ok(y_token, y_head, tokens, heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  if (tokens == 0 || heads == 0 || head_dim == 0)
    return TCRV_HIP_OK;
  if (!x || !y || !positions || (!table && n_dims && table_rows))
    return TCRV_HIP_ERR_NULL_POINTER;
  if (!aligned_to(x, size) || !aligned_to(y, size) || !aligned4(positions) || !aligned4(table))
    return TCRV_HIP_ERR_MISALIGNED;
  if (tokens > kMostTokens || heads > 0xffffu || head_dim > 65536u)
    return TCRV_HIP_ERR_TOO_LARGE;
  if (!rows_apart(y_token, y_head, tokens, heads, head_dim))
    return TCRV_HIP_ERR_BAD_SIZE;
  const auto whole = [&](const void *p, size_t token, size_t head) {
    // the loads of 4 or 8 elements: 16 bytes of f32, 8 or 16 of 16-bit types
    return aligned16(p) && token * size % 16 == 0 && head * size % 16 == 0;
  };
  const bool half = layout == TCRV_HIP_ROPE_HALF;
  const bool wide = n_dims % 8 == 0 && head_dim % 8 == 0 && whole(x, x_token, x_head) &&
                    whole(y, y_token, y_head) && aligned16(table);
  const size_t units = wide ? head_dim / 8 : n_dims / 2 + (head_dim - n_dims);
  // A work-group turns a token's heads in runs: as many as leave 1024 work-groups.
  const size_t beside = units < 256 ? 256 / units : 1;
  size_t runs = (heads + beside - 1) / beside;
  const size_t wanted = (1024 + tokens - 1) / tokens;
  if (runs > wanted)
    runs = wanted;
  const size_t a_group = (heads + runs - 1) / runs;
  runs = (heads + a_group - 1) / a_group;
  tcrv::RopeArgs a{x,      y,          positions, table, x_token, x_head, y_token,
                   y_head, table_rows, static_cast<uint32_t>(heads),
                   static_cast<uint32_t>(a_group), static_cast<uint32_t>(head_dim),
                   static_cast<uint32_t>(n_dims), inverse ? -1.0f : 1.0f};
  if (!table)
    a.table_rows = 0;
  const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>(runs));
  hipStream_t st = as_stream(stream);
  switch (elem) {
  case TCRV_HIP_ELEM_F32:
    launch_rope<float>(a, half, wide, grid, 256, st);
    break;
  case TCRV_HIP_ELEM_F16:
    launch_rope<_Float16>(a, half, wide, grid, 256, st);
    break;
  default:
    launch_rope<tcrv::Bf16>(a, half, wide, grid, 256, st);
    break;
  }
  return launch_status();
}

}  // extern "C"

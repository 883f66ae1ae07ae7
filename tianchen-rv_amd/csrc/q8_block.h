// q8_block.h -- what the kernels that write Q8_0 blocks share: eight lanes own a block, four of its
// values each.
#pragma once

#include "tcrv_hip_internal.h"

namespace tcrv {

// Branch-free: the clamp to the i16 range (v_med3_f32) commutes with the
// rounding, as both bounds are integers; NaN is selected afterwards, since the
// clamp would map it to a bound.  (Written with branches the compiler gave
// every element its own exec-mask block: 340 instructions against 271.)
__device__ __forceinline__ uint32_t quant_byte(float x, float id) {
  const float v = x * id;
  const float r = fminf(fmaxf(__builtin_rintf(v), -32768.0f), 32767.0f);  // rint: nearest-even
  // RVV float->int conversion of NaN gives the largest value
  const int w = v != v ? 32767 : static_cast<int>(r);
  return static_cast<uint32_t>(w) & 0xffu;  // narrowing keeps the low byte
}

// max of v over the 8 lanes of its group: quad_perm [1,0,3,2] and [2,3,0,1]
// give each quad's max, row_half_mirror pairs lane i with lane 7-i of the
// other quad (fmaxf is exact and order-free)
__device__ __forceinline__ float max8(float v) {
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v),
                                                                  0xB1, 0xf, 0xf, false)));
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v),
                                                                  0x4E, 0xf, 0xf, false)));
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v),
                                                                  0x141, 0xf, 0xf, false)));
  return v;
}

// The same over the 4 lanes of a quad.
__device__ __forceinline__ float max4(float v) {
  v = fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v),
                                                                  0xB1, 0xf, 0xf, false)));
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v),
                                                                     0x4E, 0xf, 0xf, false)));
}

// Four of a block's values as this lane's part of it; every lane of the group takes part.
__device__ __forceinline__ void store_q8_part(uint8_t *block, int part, const float (&v)[4]) {
  using u32a2 = uint32_t __attribute__((aligned(2)));
  const float top = fmaxf(
      max8(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))), 0.0f);
  const float d = __fdiv_rn(top, 127.0f);
  const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
  *reinterpret_cast<u32a2 *>(block + 2 + 4 * part) =
      quant_byte(v[0], id) | quant_byte(v[1], id) << 8 | quant_byte(v[2], id) << 16 |
      quant_byte(v[3], id) << 24;
  if (part == 0)
    *reinterpret_cast<uint16_t *>(block) = __builtin_bit_cast(uint16_t, static_cast<_Float16>(d));
}

}  // namespace tcrv

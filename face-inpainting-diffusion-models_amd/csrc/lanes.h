// Exchanges between lanes without LDS: data-parallel primitives within rows of 16, swaps of rows and halves of the wave.
#pragma once
#include "common.h"

namespace ifd {

// A value of another lane of this lane's group of 2^(STEP + 1), whose members of one half hold the same (or mirrored) values:
// steps 0..5 after one another combine 2, 4, 8, 16, 32, 64 lanes. A pair (x, y): combining x with y is the step's result.
template <int STEP>
__device__ __forceinline__ void lane_step(unsigned v, unsigned& x, unsigned& y) {
  if constexpr (STEP < 4) {
    // quad_perm [1,0,3,2], quad_perm [2,3,0,1], half-row mirror, row mirror
    constexpr int ctrl = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;
    x = v;
    y = (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);
  } else if constexpr (STEP == 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    x = r[0];
    y = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    x = r[0];
    y = r[1];
  }
}
template <int STEP>
__device__ __forceinline__ float lane_add(float v) {
  unsigned x, y;
  lane_step<STEP>(__float_as_uint(v), x, y);
  return __uint_as_float(x) + __uint_as_float(y);
}
// sum over groups of 2^k lanes, n = 2^k (the same for the whole wave)
__device__ __forceinline__ float group_sum(float v, int n) {
  if (n > 1) v = lane_add<0>(v);
  if (n > 2) v = lane_add<1>(v);
  if (n > 4) v = lane_add<2>(v);
  if (n > 8) v = lane_add<3>(v);
  if (n > 16) v = lane_add<4>(v);
  if (n > 32) v = lane_add<5>(v);
  return v;
}
template <int STEP>
__device__ __forceinline__ unsigned lane_max(unsigned v) {
  unsigned x, y;
  lane_step<STEP>(v, x, y);
  return max(x, y);
}
// the wave's largest of values that are not negative (their bits keep their order; a NaN comes out on top)
__device__ __forceinline__ float wave_max_nonneg(float v) {
  unsigned u = __float_as_uint(v);
  u = lane_max<0>(u);
  u = lane_max<1>(u);
  u = lane_max<2>(u);
  u = lane_max<3>(u);
  u = lane_max<4>(u);
  u = lane_max<5>(u);
  return __uint_as_float(u);
}

}  // namespace ifd

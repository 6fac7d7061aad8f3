// Reductions over groups of consecutive lanes, by exchanges of the vector unit.
#pragma once
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace momoe {

template <int CTRL>
__device__ __forceinline__ float lane_moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// op over the lanes of each group of LANES (1, 2, 4 .. 64), in every lane of it.  Four and eight apart the mirrored lane will
// do: the quads, and then the groups of eight, hold the same in every lane by then.
template <int LANES, class Op>
__device__ __forceinline__ float over_lanes(float v, Op op) {
  static_assert(LANES >= 1 && LANES <= 64 && (LANES & (LANES - 1)) == 0, "groups that halve");
  if constexpr (LANES >= 2) v = op(v, lane_moved<0xB1>(v));   // quad_perm: lane ^ 1
  if constexpr (LANES >= 4) v = op(v, lane_moved<0x4E>(v));   // quad_perm: lane ^ 2
  if constexpr (LANES >= 8) v = op(v, lane_moved<0x141>(v));  // row_half_mirror
  if constexpr (LANES >= 16) v = op(v, lane_moved<0x140>(v)); // row_mirror
  const auto swap = [&](auto pair) { return op(__uint_as_float(pair[0]), __uint_as_float(pair[1])); };
  if constexpr (LANES >= 32) v = swap(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  if constexpr (LANES >= 64) v = swap(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return v;
}
template <int LANES>
__device__ __forceinline__ float max_over_lanes(float v) {
  return over_lanes<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int LANES>
__device__ __forceinline__ float sum_over_lanes(float v) {
  return over_lanes<LANES>(v, [](float a, float b) { return a + b; });
}
// the sum over the lanes that are equal modulo STEP (a power of two), in every lane
template <int STEP>
__device__ __forceinline__ float sum_over_strides(float v) {
  if constexpr (STEP <= 4) v += lane_moved<0x124>(v);   // row_ror:4 -- with 8 below, all quads of a row of 16
  if constexpr (STEP <= 8) v += lane_moved<0x128>(v);   // row_ror:8
  const auto swap = [](auto pair) { return __uint_as_float(pair[0]) + __uint_as_float(pair[1]); };
  if constexpr (STEP <= 16) v = swap(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  if constexpr (STEP <= 32) v = swap(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return v;
}

}  // namespace momoe

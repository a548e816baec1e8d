// Reductions over the 64 lanes of a wave by lane permutes (no LDS): within 4, 8 and 16 lanes, then across the rows of 16.
#pragma once
#include <hip/hip_runtime.h>

namespace kans {

template <int CTRL, int ROWS>
__device__ __forceinline__ float lane_permute(float v, float other) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, other), __builtin_bit_cast(int, v), CTRL,
                                                               ROWS, 0xf, false));
}

// op over a wave, in every lane; `none` is its neutral element.
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, float none, F op) {
  v = op(v, lane_permute<0xb1, 0xf>(v, none));   // lane ^ 1
  v = op(v, lane_permute<0x4e, 0xf>(v, none));   // lane ^ 2
  v = op(v, lane_permute<0x141, 0xf>(v, none));  // mirrored in 8
  v = op(v, lane_permute<0x140, 0xf>(v, none));  // mirrored in 16
  v = op(v, lane_permute<0x142, 0xa>(v, none));  // lane 15 of a row into the next
  v = op(v, lane_permute<0x143, 0xc>(v, none));  // lane 31 into the upper half
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {  // of values >= 0
  return wave_reduce(v, 0.0f, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace kans

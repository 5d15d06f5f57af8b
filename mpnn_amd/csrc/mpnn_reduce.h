// Reductions of fp64 values over groups of g = 1, 2, 4 .. 64 neighbouring lanes, the result in every lane.  DPP moves (quad
// permutations, mirrors of 8 and 16 lanes: the lanes they pair hold different parts of the sum) take a few cycles each, a
// shuffle through the LDS crossbar a hundred, and every step of a reduction waits for the one before.
#pragma once
#include <hip/hip_runtime.h>

namespace {

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, false));
}
template <typename Op>
__device__ __forceinline__ double group_reduce(double v, int g, Op op) {
  if (g > 1) v = op(v, dpp_d<0xB1>(v));      // lane ^ 1
  if (g > 2) v = op(v, dpp_d<0x4E>(v));      // lane ^ 2
  if (g > 4) v = op(v, dpp_d<0x141>(v));     // mirrored in 8 lanes
  if (g > 8) v = op(v, dpp_d<0x140>(v));     // mirrored in 16 lanes
  if (g > 16) v = op(v, __shfl_xor(v, 16));
  if (g > 32) v = op(v, __shfl_xor(v, 32));
  return v;
}
__device__ __forceinline__ double group_max(double v, int g) {
  return group_reduce(v, g, [](double a, double b) { return fmax(a, b); });
}
__device__ __forceinline__ double group_sum(double v, int g) {
  return group_reduce(v, g, [](double a, double b) { return a + b; });
}

}  // namespace

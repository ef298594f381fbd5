// The arithmetic of activations kept in 8 bits, for the kernels that write and read them.
#ifndef ARBORETUM_AMD_CHECKPOINT_H_
#define ARBORETUM_AMD_CHECKPOINT_H_
#include "operators_device.h"

namespace arb {
namespace {

constexpr int kCodeVec = 8;  // values a lane codes at a time

// max that hands a NaN on
__device__ __forceinline__ float Larger(float a, float b) { return a > b || a != a ? a : b; }

template <int N>
__device__ __forceinline__ float MostOf(const float (&v)[N]) {
  float most = fabsf(v[0]);
#pragma unroll
  for (int c = 1; c < N; ++c) most = Larger(most, fabsf(v[c]));
  return most;
}

// The scale of a group whose greatest magnitude is `most`.  Steps are no smaller than 2^-100, so that their reciprocal is a
// number; an infinity or a NaN in a group makes the scale a NaN, and with it all that is read back of the group.
__device__ __forceinline__ float ScaleOf(float most) {
  const float scale = most / 127.0f;
  return most < __builtin_inff() ? fmaxf(scale, 0x1p-100f) : __builtin_nanf("");
}

// (a NaN becomes 0: the scale tells of it)
template <int N>
__device__ __forceinline__ Pack<signed char, N> CodesOf(const float (&v)[N], float scale) {
  Pack<signed char, N> codes;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const float code = rintf(v[c] / scale);
    codes.v[c] = (signed char)(int)(code == code ? fminf(fmaxf(code, -127.0f), 127.0f) : 0.0f);
  }
  return codes;
}

// (127 steps of the greatest float may round to more than it)
__device__ __forceinline__ float Restored(signed char code, float scale) {
  const float v = (float)code * scale;
  return fabsf(v) == __builtin_inff() ? copysignf(3.402823466e38f, v) : v;
}

}  // namespace
}  // namespace arb
#endif  // ARBORETUM_AMD_CHECKPOINT_H_

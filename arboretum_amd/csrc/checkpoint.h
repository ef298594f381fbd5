// The arithmetic of activations kept in 8 bits, for the kernels that write and read them.
#ifndef ARBORETUM_AMD_CHECKPOINT_H_
#define ARBORETUM_AMD_CHECKPOINT_H_
#include "operators_device.h"

namespace arb {
namespace {

constexpr int kCodeVec = 8;  // values a lane codes at a time

// Magnitudes as whole numbers: their order is that of the floats, with NaN above infinity.
__device__ __forceinline__ unsigned Magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

template <int N>
__device__ __forceinline__ unsigned MostOf(const float (&v)[N]) {
  unsigned most = Magnitude(v[0]);
#pragma unroll
  for (int c = 1; c < N; ++c) most = max(most, Magnitude(v[c]));
  return most;
}

// The scale of a group whose greatest magnitude is `most`.  Steps are no smaller than 2^-100, so that their reciprocal is a
// number; an infinity or a NaN in a group makes the scale a NaN, and with it all that is read back of the group.
__device__ __forceinline__ float ScaleOf(unsigned most) {
  return most < 0x7F800000u ? fmaxf(__uint_as_float(most) / 127.0f, 0x1p-100f) : __builtin_nanf("");
}

// rint(v / scale).  With y = 1 / scale correctly rounded, q = v y is off by no more than a rounding or two and v - q scale is exact,
// so that q + (v - q scale) y, rounded, is the quotient correctly rounded (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000"): three operations, where a division takes about ten and bound the kernel (297 us for 65,536 x 4096, now 190).
// (What a NaN becomes does not matter: the scale tells of it.)
template <int N>
__device__ __forceinline__ Pack<signed char, N> CodesOf(const float (&v)[N], float scale) {
  Pack<signed char, N> codes;
  const float y = 1.0f / scale;
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const float q = v[c] * y;
    const float quotient = fmaf(fmaf(-q, scale, v[c]), y, q);
    codes.v[c] = (signed char)(int)rintf(__builtin_amdgcn_fmed3f(quotient, -127.0f, 127.0f));
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

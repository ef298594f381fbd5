// The arithmetic of activations kept in 8 bits, for the kernels that write and read them.
#ifndef ARBORETUM_AMD_CHECKPOINT_H_
#define ARBORETUM_AMD_CHECKPOINT_H_
#include "operators_device.h"

namespace arb {
namespace {

constexpr int kCodeVec = 8;  // values a lane codes at a time

// The greater of `most` and the magnitude of v; a NaN where either is one.
__device__ __forceinline__ float MostOf(float most, float v) { return __builtin_elementwise_maximum(most, fabsf(v)); }

// The scale of a group whose greatest magnitude is `most`.  Steps are no smaller than 2^-100, so that their reciprocal is a
// number; an infinity or a NaN in a group makes the scale a NaN, and with it all that is read back of the group.
__device__ __forceinline__ float ScaleOf(float most) { return most < __builtin_inff() ? fmaxf(most / 127.0f, 0x1p-100f) : __builtin_nanf(""); }

// rint(v / scale).  With y = 1 / scale correctly rounded, q = v y is off by no more than a rounding or two and v - q scale is exact,
// so that q + (v - q scale) y, rounded, is the quotient correctly rounded (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000"): three operations, where a division takes about ten and bound the kernel (65,536 x 4096: 297 us, and 190 with nothing else changed).  Quotients are within
// 127 and a rounding: the sum with 1.5 2^23, whose last bit is worth 1, rounds them to nearest, ties to even, with the code in its low eight bits.
// (What a NaN becomes does not matter: the scale tells of it.)
template <int N>
__device__ __forceinline__ Pack<signed char, N> CodesOf(const float (&v)[N], float scale) {
  Pack<signed char, N> codes;
  const float y = 1.0f / scale;
  unsigned sum[N];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const float q = v[c] * y;
    sum[c] = __float_as_uint(fmaf(fmaf(-q, scale, v[c]), y, q) + 12582912.0f);
  }
  if constexpr (N % 4 == 0) {
    struct Words {
      unsigned w[N / 4];
    } words;
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      const unsigned low = __builtin_amdgcn_perm(sum[4 * w + 1], sum[4 * w], 0x0C0C0400), high = __builtin_amdgcn_perm(sum[4 * w + 3], sum[4 * w + 2], 0x0C0C0400);
      words.w[w] = high << 16 | low;
    }
    codes = __builtin_bit_cast(Pack<signed char, N>, words);
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) codes.v[c] = (signed char)(sum[c] & 0xFF);
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

// What the gated layer's checks (gated.hip) hand to its kernels, which are compiled type by type (gated_float32.hip,
// gated_bfloat16.hip, gated_float16.hip).
#ifndef ARBORETUM_AMD_GATED_LAUNCH_H_
#define ARBORETUM_AMD_GATED_LAUNCH_H_
#include "operators.h"

namespace arb {

constexpr int kLineBytes = 128;           // of k's in a block: 64 of 16 bits, 32 of 32
constexpr int kWaveI = 64, kWaveJ = 128;  // a wave's part of a tile: 4 x 8 fragments of 16 x 16

// A workgroup's tile: kWavesI x kWavesJ waves.
template <int kWavesI, int kWavesJ>
struct TileShape {
  static constexpr int kThreads = 64 * kWavesI * kWavesJ, kI = kWaveI * kWavesI, kJ = kWaveJ * kWavesJ;
  static constexpr int kLdsBytes = (2 * kI + 3 * kJ) * kLineBytes;  // two blocks of A, three of B
  static constexpr int kEach = 160 * 1024 / kLdsBytes;              // workgroups of a CU
  static constexpr int kWavesEach = (kWavesI * kWavesJ * kEach + 3) / 4;  // waves of a SIMD
};
typedef TileShape<4, 2> LargeTile;
typedef TileShape<2, 1> SmallTile;

// How a product is cut up: into which tiles, and how many shares of its k's (blocks of kLineBytes of them).
struct ProductCut {
  bool large;
  long long splits, split_blocks;
};
// Where in the work memory (bytes from its start) copies of x and the weights lie whose rows begin at multiples of 64 elements;
// stride 0: there are none.
struct LayerPad {
  long long stride;
  size_t x, w_gate, w_up;
};
struct GatedPlan {
  bool few;
  ProductCut out;
  LayerPad pad;
  size_t partial, bytes;
};
struct GatedGradPlan {
  long long d_stride;  // elements between rows of d_gate and of d_up
  ProductCut x, w;     // of grad_x, of the weights' gradients
  LayerPad pad;
  size_t d_gate, d_up, partial, bytes;
};

inline long long Pieces(long long n, long long of) { return (n + of - 1) / of; }

// (arguments that have passed the checks)
template <typename T>
void RunGated(const GatedArgs &a, const GatedPlan &plan);
template <typename T>
void RunGatedGrad(const GatedGradArgs &a, const GatedGradPlan &plan);

}  // namespace arb
#endif  // ARBORETUM_AMD_GATED_LAUNCH_H_

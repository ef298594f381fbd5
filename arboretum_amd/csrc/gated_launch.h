// What the gated layer's checks (gated.hip) hand to its kernels, which are compiled type by type (gated_float32.hip,
// gated_bfloat16.hip, gated_float16.hip).
#ifndef ARBORETUM_AMD_GATED_LAUNCH_H_
#define ARBORETUM_AMD_GATED_LAUNCH_H_
#include "operators.h"

namespace arb {

constexpr int kLineBytes = 128;  // of k's in a block: 64 of 16 bits, 32 of 32
constexpr int kWaveJ = 128;      // columns of a wave's part of a tile
constexpr int kFewRows = 16;     // up to here a product's sixteen rows hold all of x
constexpr int kRangeGroups = 2048;  // workgroups that form d_gate and d_up in float16: each of the second pass reads what all of the first have found

// A workgroup's tile: kWavesI x kWavesJ waves, kWaveI rows by kWaveJ columns each.  The LDS holds kBlocksA blocks of A and kBlocksB of B: one that is multiplied, the
// others on their way.
template <int kWavesI, int kWavesJ, int kWaveI_, int kBlocksA_, int kBlocksB_>
struct TileShape {
  static constexpr int kWaveI = kWaveI_, kThreads = 64 * kWavesI * kWavesJ, kI = kWaveI * kWavesI, kJ = kWaveJ * kWavesJ;
  static constexpr int kBlocksA = kBlocksA_, kBlocksB = kBlocksB_;
  static constexpr int kLdsBytes = (kBlocksA * kI + kBlocksB * kJ) * kLineBytes;
  static constexpr int kEach = 160 * 1024 / kLdsBytes;              // workgroups of a CU
  static constexpr int kWavesEach = kWavesI * kWavesJ * kEach / 4;  // waves of a SIMD
};
typedef TileShape<4, 2, 64, 2, 3> LargeTile;  // 256 x 256
typedef TileShape<4, 1, 32, 2, 3> SmallTile;  // 128 x 128, two to a CU.  Four waves, one for each SIMD where a CU has only one tile, read 1.7 times as much of
                                              // the LDS as two of 64 rows did, and took 20.4 us for 1003 x 771 x 2055 (22.3), 15.7 for 200000 x 16 x 64 (21.0)

// How a product is cut up: into which tiles, and how many shares of its k's (blocks of kLineBytes of them).
struct ProductCut {
  bool large;
  long long splits, split_blocks, tiles;  // tiles: of all shares
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
  bool together;       // all tiles of both have a place on the chip at once
  LayerPad pad;
  size_t d_gate, d_up, range, x_partial, w_partial, bytes;
};

inline long long Pieces(long long n, long long of) { return (n + of - 1) / of; }

// (arguments that have passed the checks)
template <typename T>
void RunGated(const GatedArgs &a, const GatedPlan &plan);
template <typename T>
void RunGatedGrad(const GatedGradArgs &a, const GatedGradPlan &plan);

}  // namespace arb
#endif  // ARBORETUM_AMD_GATED_LAUNCH_H_

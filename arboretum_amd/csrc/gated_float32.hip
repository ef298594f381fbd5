// The gated layer's kernels in float32.
#include "gated_kernels.h"

namespace arb {
template void RunGated<float>(const GatedArgs &a, bool large);
template void RunGatedGrad<float>(const GatedGradArgs &a, const GatedPlan &plan);
}  // namespace arb

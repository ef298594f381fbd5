// The gated layer's kernels in float32.
#include "gated_kernels.h"

namespace arb {
template void RunGated<float>(const GatedArgs &a, const GatedPlan &plan);
template void RunGatedGrad<float>(const GatedGradArgs &a, const GatedGradPlan &plan);
}  // namespace arb

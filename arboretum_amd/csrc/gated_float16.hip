// The gated layer's kernels in float16.
#include "gated_kernels.h"

namespace arb {
template void RunGated<_Float16>(const GatedArgs &a, const GatedPlan &plan);
template void RunGatedGrad<_Float16>(const GatedGradArgs &a, const GatedGradPlan &plan);
}  // namespace arb

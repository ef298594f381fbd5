// The gated layer's kernels in bfloat16.
#include "gated_kernels.h"

namespace arb {
template void RunGated<__bf16>(const GatedArgs &a, bool large);
template void RunGatedGrad<__bf16>(const GatedGradArgs &a, const GatedPlan &plan);
}  // namespace arb

// The gated layer's kernels in bfloat16.
#include "gated_kernels.h"

namespace arb {
template void RunGated<__bf16>(const GatedArgs &a, const GatedPlan &plan);
template void RunGatedGrad<__bf16>(const GatedGradArgs &a, const GatedGradPlan &plan);
}  // namespace arb

// Experts' products, FP8 weights.
#include "experts_kernel.h"

namespace paia {

int launch_experts_fp8(const ExpertsParams& p, bool gated, hipStream_t st) { return launch_experts_format<kFP8>(p, gated, st); }

}  // namespace paia

// Experts' products, BF16 weights.
#include "experts_kernel.h"

namespace paia {

int launch_experts_bf16(const ExpertsParams& p, bool gated, hipStream_t st) { return launch_experts_format<kBF16>(p, gated, st); }

}  // namespace paia

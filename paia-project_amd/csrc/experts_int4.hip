// Experts' products, INT4 weights.
#include "experts_kernel.h"

namespace paia {

int launch_experts_int4(const ExpertsParams& p, bool gated, hipStream_t st) { return launch_experts_format<kI4>(p, gated, st); }

}  // namespace paia

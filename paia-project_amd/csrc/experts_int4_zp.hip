// Experts' products, INT4 asymmetric weights.
#include "experts_kernel.h"

namespace paia {

int launch_experts_int4_zp(const ExpertsParams& p, bool gated, hipStream_t st) { return launch_experts_format<kI4ZP>(p, gated, st); }

}  // namespace paia

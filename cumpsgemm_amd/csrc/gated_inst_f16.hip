// Gated blocks and their gradients: kernels of FP16 operands.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(f16, Elem::F16)
} // namespace cumpsgemm_amd

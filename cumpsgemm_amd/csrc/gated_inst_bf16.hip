// Gated blocks and their gradients: kernels of BF16 operands.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(bf16, Elem::BF16)
} // namespace cumpsgemm_amd

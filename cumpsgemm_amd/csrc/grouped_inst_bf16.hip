// Experts' products: kernels of BF16 operands.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_16(g_grouped_bf16, Elem::BF16)
} // namespace cumpsgemm_amd

// Experts' products: kernels of FP16 operands.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_16(g_grouped_f16, Elem::F16)
} // namespace cumpsgemm_amd

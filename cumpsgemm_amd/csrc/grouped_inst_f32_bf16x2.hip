// Experts' products: kernels of FP32 operands in two BF16 terms.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_F32(g_grouped_f32_bf16x2, Elem::F32_BF16X2)
} // namespace cumpsgemm_amd

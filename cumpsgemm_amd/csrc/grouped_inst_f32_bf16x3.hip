// Experts' products: kernels of FP32 operands in three BF16 terms.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_F32(g_grouped_f32_bf16x3, Elem::F32_BF16X3)
} // namespace cumpsgemm_amd

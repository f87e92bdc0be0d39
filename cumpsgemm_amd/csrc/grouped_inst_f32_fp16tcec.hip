// Experts' products: kernels of FP32 operands in FP16 hi / lo terms.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_F32(g_grouped_f32_fp16tcec, Elem::F32_FP16TCEC)
} // namespace cumpsgemm_amd

// Experts' products: kernels of FP32 operands rounded to FP16.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_F32(g_grouped_f32_fp16tc, Elem::F32_FP16TC)
} // namespace cumpsgemm_amd

// Gated blocks and their gradients: kernels of FP32 operands, TF32TCEC (bf16x3).
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(f32_bf16x3, Elem::F32_BF16X3)
} // namespace cumpsgemm_amd

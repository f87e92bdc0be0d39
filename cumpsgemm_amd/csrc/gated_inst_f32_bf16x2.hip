// Gated blocks and their gradients: kernels of FP32 operands, TF32TC (bf16x2).
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(f32_bf16x2, Elem::F32_BF16X2)
} // namespace cumpsgemm_amd

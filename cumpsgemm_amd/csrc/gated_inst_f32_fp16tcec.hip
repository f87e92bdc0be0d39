// Gated blocks and their gradients: kernels of FP32 operands, FP16TCEC.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(f32_fp16tcec, Elem::F32_FP16TCEC)
} // namespace cumpsgemm_amd

// Gated blocks and their gradients: kernels of FP32 operands, FP16TC.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GATED(f32_fp16tc, Elem::F32_FP16TC)
} // namespace cumpsgemm_amd

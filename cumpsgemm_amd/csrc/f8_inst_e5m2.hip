// Products of 8-bit floating point: kernels of tokens in E5M2.
#include "f8_kernel.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_F8(e5m2, Elem::E5M2)
} // namespace cumpsgemm_amd

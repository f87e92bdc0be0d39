// Products of 8-bit floating point: kernels of tokens in E4M3.
#include "f8_kernel.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_F8(e4m3, Elem::E4M3)
} // namespace cumpsgemm_amd

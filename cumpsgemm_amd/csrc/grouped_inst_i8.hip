// Experts' products: kernels of 8-bit integers.
#include "grouped_table.hpp"

namespace cumpsgemm_amd {
CUMPSGEMM_GROUPED_I8(g_grouped_i8, Elem::I8)
} // namespace cumpsgemm_amd

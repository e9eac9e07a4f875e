// q4k_attn_f16.hip -- the shared-prefix attention kernels of F16 queries, keys and values
#include "q4k_attn.h"

namespace q4k {
void attn_kernel_f16(AttnPlan &pl) { attn_kernel_of<_Float16, _Float16, 1>(pl); }
}  // namespace q4k

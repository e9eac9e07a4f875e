// q4k_attn_f16_f32.hip -- the shared-prefix attention kernels of F32 queries, F16 keys and values
#include "q4k_attn.h"

namespace q4k {
void attn_kernel_f16_f32(AttnPlan &pl) { attn_kernel_of<_Float16, float, 2>(pl); }
}  // namespace q4k

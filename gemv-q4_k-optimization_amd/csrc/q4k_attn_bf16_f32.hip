// q4k_attn_bf16_f32.hip -- the shared-prefix attention kernels of F32 queries, BF16 keys and values
#include "q4k_attn.h"

namespace q4k {
void attn_kernel_bf16_f32(AttnPlan &pl) { attn_kernel_of<__bf16, float, 3>(pl); }
}  // namespace q4k

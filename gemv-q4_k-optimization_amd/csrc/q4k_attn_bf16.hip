// q4k_attn_bf16.hip -- the shared-prefix attention kernels of BF16 queries, keys and values
#include "q4k_attn.h"

namespace q4k {
void attn_kernel_bf16(AttnPlan &pl) { attn_kernel_of<__bf16, __bf16, 1>(pl); }
}  // namespace q4k

// q4k_kv8_attn_f16.hip -- the attention kernels over caches of 8 bits for F16 queries
#include "q4k_kv8_attn.h"

namespace q4k {
void kv8_attn_f16(Kv8AttnPlan &pl) { kv8_attn_kernel_of<_Float16>(pl); }
}  // namespace q4k

// q4k_kv8_attn_f32.hip -- the attention kernels over caches of 8 bits for F32 queries
#include "q4k_kv8_attn.h"

namespace q4k {
void kv8_attn_f32(Kv8AttnPlan &pl) { kv8_attn_kernel_of<float>(pl); }
}  // namespace q4k

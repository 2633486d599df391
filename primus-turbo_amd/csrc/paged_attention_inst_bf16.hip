// Attention kernels of bf16 queries (paged_attention.h).
#include "paged_attention_launch.h"

namespace pta {
template void attn_launch<PTA_BF16>(const AttnCall &, int, hipStream_t);
} // namespace pta

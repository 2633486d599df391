// Attention kernels of f16 queries (paged_attention.h).
#include "paged_attention_launch.h"

namespace pta {
template void attn_launch<PTA_F16>(const AttnCall &, int, hipStream_t);
} // namespace pta

// Attention of tiles of tokens through their pages, fp16 queries.
#include "paged_attention_launch.h"

namespace pta {
template void attn_launch_tiles<PTA_F16>(const AttnArgs &, int, hipStream_t);
}

// Attention over caches of bf16.
#include "attn_tiles.h"

namespace hoard {

hipError_t launch_attn_bf16(const AttnCall &p, hipStream_t s) { return launch_attn_cache<bf16>(p, s); }

}  // namespace hoard

// Attention over caches of 8-bit codes.
#include "attn_tiles.h"

namespace hoard {

hipError_t launch_attn_i8(const AttnCall &p, hipStream_t s) { return launch_attn_cache<int8_t>(p, s); }

}  // namespace hoard

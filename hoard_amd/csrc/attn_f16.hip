// Attention over caches of f16.
#include "attn_tiles.h"

namespace hoard {

hipError_t launch_attn_f16(const AttnCall &p, hipStream_t s) { return launch_attn_cache<f16>(p, s); }

}  // namespace hoard

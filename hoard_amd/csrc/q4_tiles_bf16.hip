// Matrix tiles of the 4-bit products for bf16 activations.
#include "q4_tiles.h"

namespace hoard {

hipError_t launch_q4_tiles_bf16(const Q4Args &a, hipStream_t s) { return launch_tiles_typed<bf16>(a, s); }

}  // namespace hoard

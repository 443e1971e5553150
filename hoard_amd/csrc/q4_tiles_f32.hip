// Matrix tiles of the 4-bit products for f32 activations.
#include "q4_tiles.h"

namespace hoard {

hipError_t launch_q4_tiles_f32(const Q4Args &a, hipStream_t s) { return launch_tiles_typed<float>(a, s); }

}  // namespace hoard

// How the attention over a cache is split over its length: shared by the kernel of the
// tiles, that of the join and the host.
#pragma once

#include <hip/hip_runtime.h>

#include "attn.h"

namespace hoard {

struct AttnCall {
    hoard_kv_cache c;
    hoard_attn_args a;
    int splits;      // parts that a sequence may be split into, at most
    int row_waves;   // 1, 2 or 4: waves of a workgroup side by side over the rows
    int row_blocks;  // workgroups over the rows
    float *part_out, *part_lse;  // [rows][splits][head_dim] and [rows][splits], with splits > 1
};

constexpr int kKeyTile = 32;
constexpr int kMaxSplits = 256;
constexpr int kAttnGroups = 512;

// The parts of a sequence of which `keys` keys are seen: as many as there may be, but of a
// tile a wave at least.
struct AttnParts {
    int tiles, per, used;
};
__device__ __forceinline__ AttnParts attn_parts(int keys, int splits, int waves) {
    AttnParts p;
    p.tiles = (keys + kKeyTile - 1) / kKeyTile;
    p.per = max((p.tiles + splits - 1) / splits, waves);
    p.used = (p.tiles + p.per - 1) / p.per;
    return p;
}

hipError_t launch_attn_f16(const AttnCall &p, hipStream_t s);
hipError_t launch_attn_bf16(const AttnCall &p, hipStream_t s);
hipError_t launch_attn_i8(const AttnCall &p, hipStream_t s);

}  // namespace hoard

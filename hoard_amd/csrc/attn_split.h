// How the attention over a cache is split over its length: shared by the kernel of the
// tiles, that of the join and the host.
//
// A lane of work is one sequence's for one key head and block of rows: its tiles of 32 keys,
// at least one (a row that sees nothing has its zeros to write).  Where there are fewer lanes
// than keep the chip busy and level, the tiles of all of them are one row, as the lengths
// are found on the device, and every workgroup takes an equal run of it: the end of one lane,
// some whole ones, the beginning of another.  A lane that no run holds whole goes to the
// workspace in its parts, and a second launch joins them.  The parts in the order of the row are
// numbered by workgroup + lane, as one of the two grows from each to the next.  Where the runs
// are short a second part costs a workgroup more than an even share gains: there every lane
// begins a run of its own, and the parts are numbered by workgroup (a call with 1025 tokens by
// 4 lanes takes 11 us, 13.3 with runs over lanes; with 2048 tokens 11).  Their runs are so long
// that there are no more of them than CUs, where the lanes leave room for that: at 256 columns
// a CU holds one workgroup, and the rest would come second (16 sequences of 5 new tokens, 28000
// keys in all: 43 us with runs of a 256th of the tiles, 30 so).
//
// One workgroup a CU: 64 equal sequences of 4352 tokens by 4 lanes, 8-bit codes, take 55 us in
// 256 runs, 62 in 512, 64 in 1024 (the join of the parts included); 16 of some 1600 by 2 lanes of
// 256 columns 20, 28 and 28.  Equal runs, as a CU reads no more than twice its share of the
// memory's rate: 64 sequences of 512 to 8192 tokens 70 us (the two launches), 78 where each lane is cut by itself
// into parts of up to the same length, 82 into two.
#pragma once

#include <hip/hip_runtime.h>

#include "attn.h"
#include "wave.h"

namespace hoard {

constexpr int kKeyTile = 32;
constexpr int kRuns = 256;     // a workgroup a CU
constexpr int kOwnRun = 16;    // where even runs would be shorter each holds one lane's tiles only
constexpr int kMaxSplitSeqs = 256;

// Waves of the tiles' workgroup.  Eight read no faster (one sequence of 32768 tokens in bf16
// 19.3 us against 18.4), and take longer to start (256 tokens, the kernel: 6.9 against 6.1).
constexpr int kAttnWaves = 4;

struct AttnCall {
    hoard_kv_cache c;
    hoard_attn_args a;
    int split;       // whether lanes may be cut
    int row_waves;   // 1, 2 or 4: waves of a workgroup side by side over the rows
    int row_blocks;  // workgroups over the rows
    int block_rows;  // rows of a workgroup
    int min_run;     // tiles of a run, at least: one a wave
    float *part_out, *part_stat;  // [parts][block_rows][head_dim], and [parts][block_rows] of the largest score
                                  // and the weights' sum by it, with split
    int32_t *sums;   // [n_seq + 2]: tiles of all lanes of the sequences up to each, a run's, whether
                     // runs hold one lane's tiles only; with split
};

// The keys that each new token of a sequence sees, a lane each, and the most of them.
__device__ __forceinline__ int attn_seen(const hoard_attn_args &a, int limit, int seq) {
    const int lane = threadIdx.x & 63;
    return lane < a.n_new ? min(max(a.lens[(int64_t)seq * a.n_new + lane], 0), limit) : 0;
}
__device__ __forceinline__ int attn_most(int v) {
    v = max(v, dpp_i<kDppQuadXor1>(v));
    v = max(v, dpp_i<kDppQuadXor2>(v));
    v = max(v, dpp_i<kDppRowHalfMirror>(v));
    v = max(v, dpp_i<kDppRowMirror>(v));
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
// The running sum over the wave's lanes: within rows of 16, then the rows before.
__device__ __forceinline__ int attn_running(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, kDppRowBcast15, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, kDppRowBcast31, 0xc, 0xf, false);
    return v;
}
// A lane's tiles.
__device__ __forceinline__ int attn_tiles(int keys) {
    return max((int)(((uint32_t)keys + kKeyTile - 1) / kKeyTile), 1);
}

// Where in the row of tiles a sequence lies: its keys, its first tile and what a run holds.
struct AttnPlace {
    int seq, keys, first, run, total;
    bool own;
};
// A lane's tiles in the row: whole runs where they hold one lane's only.
__device__ __forceinline__ int attn_row_tiles(int tiles, int run, bool own) {
    return own ? (tiles + run - 1) / run * run : tiles;
}
// The sequence that holds tile (blockIdx.x * run) of the row; seq -1 where the row is shorter.  By
// all lanes of a wave.  The first workgroup leaves the sums for the join.
__device__ __forceinline__ AttnPlace attn_place(const AttnCall &p) {
    constexpr int STEPS = kMaxSplitSeqs / 64;
    const hoard_attn_args &a = p.a;
    const int limit = a.max_pages * p.c.page, lanes = p.c.n_kv_heads * p.row_blocks, lane = threadIdx.x & 63;
    int keys[STEPS], sums[STEPS], all = 0, before = 0;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        keys[i] = 0;
        if (i * 64 + lane < a.n_seq) {
            const int32_t *lens = a.lens + (int64_t)(i * 64 + lane) * a.n_new;
#pragma unroll 4
            for (int t = 0; t < a.n_new; t++) keys[i] = max(keys[i], lens[t]);
            keys[i] = min(keys[i], limit);
        }
    }
#pragma unroll
    for (int i = 0; i < STEPS; i++)
        if (i * 64 < a.n_seq)
            all += __builtin_amdgcn_readlane(attn_running(i * 64 + lane < a.n_seq ? attn_tiles(keys[i]) : 0), 63);
    AttnPlace r{-1, 0, 0, 0, 0, false};
    r.run = (all * lanes + kRuns - 1) / kRuns;
    r.own = r.run < kOwnRun;
    if (r.own) {
        const int runs = max(kRuns - a.n_seq * lanes, kRuns / 2);
        r.run = max((all * lanes + runs - 1) / runs, p.min_run);
    }
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        sums[i] = before;
        if (i * 64 >= a.n_seq) continue;
        // of this sequence and those before it
        sums[i] += attn_running(i * 64 + lane < a.n_seq ? attn_row_tiles(attn_tiles(keys[i]), r.run, r.own) * lanes : 0);
        before = __builtin_amdgcn_readlane(sums[i], 63);
        if (blockIdx.x == 0 && threadIdx.x < 64 && i * 64 + lane < a.n_seq) p.sums[i * 64 + lane] = sums[i];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.sums[a.n_seq] = r.run;
        p.sums[a.n_seq + 1] = r.own;
    }
    r.total = before;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        if (i * 64 >= a.n_seq || r.seq >= 0) continue;
        const int at = __popcll(__ballot(sums[i] <= (int)blockIdx.x * r.run));
        if (at >= 64 || i * 64 + at >= a.n_seq) continue;
        r.seq = i * 64 + at;
        r.keys = __builtin_amdgcn_readlane(keys[i], at);
        r.first = __builtin_amdgcn_readlane(sums[i], at) - attn_row_tiles(attn_tiles(r.keys), r.run, r.own) * lanes;
    }
    // one value for the wave, which the addresses of its buffers have to be seen to be
    r.seq = __builtin_amdgcn_readfirstlane(r.seq);
    r.keys = __builtin_amdgcn_readfirstlane(r.keys);
    r.first = __builtin_amdgcn_readfirstlane(r.first);
    return r;
}

hipError_t launch_attn_f16(const AttnCall &p, hipStream_t s);
hipError_t launch_attn_bf16(const AttnCall &p, hipStream_t s);
hipError_t launch_attn_i8(const AttnCall &p, hipStream_t s);

// Lanes of work, workgroups of the tiles' kernel, and parts in the workspace.
inline int64_t attn_lanes(const AttnCall &p) { return (int64_t)p.a.n_seq * p.c.n_kv_heads * p.row_blocks; }
inline int attn_grid(const AttnCall &p) { return (int)attn_lanes(p) + (p.split ? kRuns : 0); }
inline int64_t attn_parts(const AttnCall &p) { return p.split ? kRuns - 1 + attn_lanes(p) : 0; }

}  // namespace hoard

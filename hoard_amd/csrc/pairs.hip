// Pairs sorted by expert, their rows laid out and taken back (hoard_sort_*).
//
// The sort is a stable counting sort.  A block of kBlockPairs consecutive pairs
// counts its experts; a pair's sorted row is the number of pairs of lower
// experts, plus those of its own expert in earlier blocks, plus its rank among
// its own block's.  The rank within a wave comes from ballots over the bits of
// the expert id, the one across the block's waves from their counts in LDS.
// One block of pairs is one launch; above it a launch of counts comes first.  Up to
// kAddBlocks each block adds up what precedes it, which is one launch less; above, the
// counts are summed along the blocks by a launch between the two.
#include "ops.h"
#include "opsdev.h"

namespace hoard {

namespace {

constexpr int kBlockPairs = 1024;
constexpr int kMaxExperts = 1024;
constexpr int kWaves = kBlockPairs / 64;
constexpr int kAddBlocks = 64;

// The lanes of the wave that hold the same key (of `bits` bits), as a mask.
__device__ __forceinline__ uint64_t same_key(int key, int bits) {
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; b++) {
        const bool one = (key >> b) & 1;
        const uint64_t ones = __ballot(one);
        same &= one ? ones : ~ones;
    }
    return same;
}

// Pair p's expert; n_expert for a dropped pair and behind the last one.
__device__ __forceinline__ int key_of(const PairsArgs &a, int64_t p, int64_t pairs) {
    if (p >= pairs) return a.n_expert;
    const int e = a.ids[p];
    return e < 0 || e >= a.n_expert ? a.n_expert : e;
}

// counts[block][expert]
__global__ __launch_bounds__(kBlockPairs) void count_kernel(PairsArgs a, int64_t pairs) {
    __shared__ int cnt[kMaxExperts + 1];
    for (int e = threadIdx.x; e <= a.n_expert; e += kBlockPairs) cnt[e] = 0;
    __syncthreads();
    atomicAdd(&cnt[key_of(a, (int64_t)blockIdx.x * kBlockPairs + threadIdx.x, pairs)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < a.n_expert; e += kBlockPairs) a.work[(size_t)blockIdx.x * a.n_expert + e] = cnt[e];
}

// a.work[b][e]: the counts of blocks 0..b.  A workgroup takes 64 experts, its 16 waves
// a sixteenth of the blocks each: their sums first, then the running ones.
__global__ __launch_bounds__(1024) void scan_kernel(PairsArgs a, int blocks) {
    __shared__ int sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
    const int per = (blocks + 15) / 16, b0 = min(blocks, wave * per), b1 = min(blocks, b0 + per);
    int s = 0;
    if (e < a.n_expert) {
#pragma unroll 8
        for (int b = b0; b < b1; b++) s += a.work[(size_t)b * a.n_expert + e];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (e >= a.n_expert) return;
    s = 0;
    for (int w = 0; w < wave; w++) s += sums[w][lane];
#pragma unroll 8
    for (int b = b0; b < b1; b++) {
        s += a.work[(size_t)b * a.n_expert + e];
        a.work[(size_t)b * a.n_expert + e] = s;
    }
}

// blocks > 1: a.work holds every block's counts, or their running sums (above kAddBlocks).
__global__ __launch_bounds__(kBlockPairs) void place_kernel(PairsArgs a, int64_t pairs, int bits) {
    __shared__ uint16_t of_wave[kWaves][kMaxExperts + 1];  // pairs of each expert in each wave, then before it
    __shared__ int base[kMaxExperts + 1];                  // the block's first row of each expert
    __shared__ int sums[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.n_expert, blocks = gridDim.x;
    const int64_t p = (int64_t)blockIdx.x * kBlockPairs + tid;
    const int key = key_of(a, p, pairs);
    for (int e = tid; e <= E; e += kBlockPairs)
#pragma unroll
        for (int w = 0; w < kWaves; w++) of_wave[w][e] = 0;
    __syncthreads();
    const uint64_t same = same_key(key, bits), before = same & ((1ull << lane) - 1ull);
    const int rank = __popcll(before);
    if (before == 0) of_wave[wave][key] = (uint16_t)__popcll(same);
    __syncthreads();
    // thread e: its expert's pairs over the waves, over the blocks before, over all
    int mine = 0, earlier = 0, total = 0;
    if (tid < E) {
        for (int w = 0; w < kWaves; w++) {
            const int c = of_wave[w][tid];
            of_wave[w][tid] = (uint16_t)mine;
            mine += c;
        }
        if (blocks == 1) {
            total = mine;
        } else if (blocks > kAddBlocks) {
            total = a.work[(size_t)(blocks - 1) * E + tid];
            earlier = blockIdx.x ? a.work[(size_t)(blockIdx.x - 1) * E + tid] : 0;
        } else {
#pragma unroll 8
            for (int b = 0; b < blocks; b++) {
                const int c = a.work[(size_t)b * E + tid];
                if (b < (int)blockIdx.x) earlier += c;
                total += c;
            }
        }
    }
    // exclusive sum of the totals over the experts
    int incl = total;
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int first = incl - total, all = 0;
    for (int w = 0; w < kWaves; w++) {
        if (w < wave) first += sums[w];
        all += sums[w];
    }
    if (tid < E) {
        base[tid] = first + earlier;
        if (blockIdx.x == 0) a.offsets[tid] = first;
    }
    if (blockIdx.x == 0 && tid == 0) a.offsets[E] = all;
    __syncthreads();
    if (p < pairs) {
        int row = -1;
        if (key < E) {
            row = base[key] + of_wave[wave][key] + rank;
            a.order[row] = (int)p;
        }
        a.place[p] = row;
        if (p >= all) a.order[p] = -1;
    }
}

// -- rows ---------------------------------------------------------------------

// Gather and combine are bound by memory: an item is 8 columns of a token, a wave's
// items are consecutive, and an item's places and rows are fetched kAhead slots at a
// time, so that their latencies overlap.
constexpr int kAhead = 8;

__device__ __forceinline__ bool item_of(const RowsArgs &a, int64_t i, int per_row, int64_t &t, Cols &c) {
    t = i / per_row;
    c = cols_of((int)(i - t * per_row) * 8, a.n);
    return t < a.n_tokens;
}
// The sorted rows of slots j0 .. j0 + kAhead - 1 of token t, -1 for a dropped pair.
__device__ __forceinline__ void rows_of(const RowsArgs &a, int64_t t, int j0, int64_t pairs, int row[kAhead],
                                        float w[kAhead]) {
    const int32_t *const place = a.place + t * a.k;
    const float *const weight = a.w + t * a.k;
#pragma unroll
    for (int u = 0; u < kAhead; u++) {
        const int j = min(j0 + u, a.k - 1);
        row[u] = place[j];
        w[u] = a.w ? weight[j] : 1.0f;
    }
#pragma unroll
    for (int u = 0; u < kAhead; u++)
        if (j0 + u >= a.k || row[u] >= pairs) row[u] = -1;
}

template <typename T, bool NT>
__global__ __launch_bounds__(256) void gather_kernel(RowsArgs a) {
    const int per_row = (a.n + 7) / 8;
    const int64_t pairs = (int64_t)a.n_tokens * a.k;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;; i += (int64_t)gridDim.x * 256) {
        int64_t t;
        Cols c;
        if (!item_of(a, i, per_row, t, c)) return;
        float x[8], o[8], w[kAhead];
        int row[kAhead];
        widen(fetch(static_cast<const T *>(a.x) + t * a.n, c, a.n), x);
        for (int j = 0; j < a.k; j += kAhead) {
            rows_of(a, t, j, pairs, row, w);
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (row[u] < 0) continue;
#pragma unroll
                for (int v = 0; v < 8; v++) o[v] = a.w ? w[u] * x[v] : x[v];
                put<NT>(static_cast<T *>(a.out) + (int64_t)row[u] * a.n, c, a.n, o);
            }
        }
    }
}

template <typename T, bool NT>
__global__ __launch_bounds__(256) void combine_kernel(RowsArgs a) {
    const int per_row = (a.n + 7) / 8;
    const int64_t pairs = (int64_t)a.n_tokens * a.k;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;; i += (int64_t)gridDim.x * 256) {
        int64_t t;
        Cols c;
        if (!item_of(a, i, per_row, t, c)) return;
        float s[8] = {}, w[kAhead], v[8];
        int row[kAhead];
        if (a.res) widen(fetch(static_cast<const T *>(a.res) + t * a.n, c, a.n), s);
        for (int j = 0; j < a.k; j += kAhead) {
            rows_of(a, t, j, pairs, row, w);
            Raw<T> y[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++)  // a dropped pair's place is row 0's, and not added
                y[u] = fetch<NT>(static_cast<const T *>(a.x) + (int64_t)max(row[u], 0) * a.n, c, a.n);
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                widen(y[u], v);
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] = row[u] >= 0 ? fmaf(w[u], v[i], s[i]) : s[i];
            }
        }
        put<NT>(static_cast<T *>(a.out) + t * a.n, c, a.n, s);
    }
}

// A wave takes a pair, kChunks * 512 columns at a time.
constexpr int kChunks = 4;
template <typename T, bool NT>
__device__ __forceinline__ float grad_row(const T *d, const T *y, T *dy, float w, int n) {
    const int lane = threadIdx.x & 63;
    float s = 0.0f;
    for (int at = lane * 8; at - lane * 8 < n; at += kChunks * 512) {
        Raw<T> dr[kChunks], yr[kChunks];
        Cols c[kChunks];
#pragma unroll
        for (int u = 0; u < kChunks; u++) {
            c[u] = cols_of(at + u * 512, n);
            dr[u] = fetch(d, c[u], n);
            yr[u] = fetch<NT>(y, c[u], n);
        }
#pragma unroll
        for (int u = 0; u < kChunks; u++) {
            float dv[8], yv[8];
            widen(dr[u], dv);
            widen(yr[u], yv);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                s = i >= c[u].lo ? fmaf(dv[i], yv[i], s) : s;
                dv[i] *= w;
            }
            if (dy && c[u].lo < 8) put<NT>(dy, c[u], n, dv);
        }
    }
    return s;
}

template <typename T, bool NT>
__global__ __launch_bounds__(256) void combine_grad_kernel(RowsArgs a) {
    const int64_t pairs = (int64_t)a.n_tokens * a.k;
    for (int64_t p = (int64_t)blockIdx.x * 4 + wave_index(); p < pairs; p += (int64_t)gridDim.x * 4) {
        const int row = a.place[p];
        float s = 0.0f;
        if (row >= 0 && row < pairs) {
            const T *const d = static_cast<const T *>(a.res) + p / a.k * a.n;
            const T *const y = static_cast<const T *>(a.x) + (int64_t)row * a.n;
            T *const dy = a.out ? static_cast<T *>(a.out) + (int64_t)row * a.n : nullptr;
            s = grad_row<T, NT>(d, y, dy, a.w[p], a.n);
        }
        s = wave_sum_f(s);
        if ((threadIdx.x & 63) == 0) a.dw[p] = s;
    }
}

int64_t rows_grid(const RowsArgs &a) {
    const int64_t items = (int64_t)a.n_tokens * ((a.n + 7) / 8), groups = (items + 255) / 256;
    return groups < (1 << 20) ? groups : (1 << 20);
}

// Sorted rows that the L2s (8 of 4 MB) would not hold until they are read, or hold
// since they were written, go past them: gather of 1021 tokens by 10 (28 MB written)
// 7.5 us against 12.5, combine of 4096 by 8 (134 MB read) 36.6 against 40.2, its
// gradient 102 against 111.  Smaller ones are left there for the call that follows.
bool past_caches(const RowsArgs &a) {
    const int64_t bytes = (int64_t)a.n_tokens * a.k * a.n * (a.type == HOARD_TYPE_F32 ? 4 : 2);
    return bytes >= (16 << 20);
}

#define HOARD_ROWS(KERNEL, GRID)                                                                             \
    do {                                                                                                     \
        const unsigned grid = (unsigned)(GRID);                                                              \
        const bool nt = past_caches(a);                                                                      \
        if (a.type == HOARD_TYPE_F32 && nt) KERNEL<float, true><<<grid, 256, 0, s>>>(a);                     \
        else if (a.type == HOARD_TYPE_F32) KERNEL<float, false><<<grid, 256, 0, s>>>(a);                     \
        else if (a.type == HOARD_TYPE_F16 && nt) KERNEL<f16, true><<<grid, 256, 0, s>>>(a);                  \
        else if (a.type == HOARD_TYPE_F16) KERNEL<f16, false><<<grid, 256, 0, s>>>(a);                       \
        else if (nt) KERNEL<bf16, true><<<grid, 256, 0, s>>>(a);                                             \
        else KERNEL<bf16, false><<<grid, 256, 0, s>>>(a);                                                    \
        return hipGetLastError();                                                                            \
    } while (0)

}  // namespace

size_t sort_work_bytes(int64_t pairs, int n_expert) {
    return pairs <= kBlockPairs ? 0 : sizeof(int32_t) * (size_t)((pairs + kBlockPairs - 1) / kBlockPairs) * n_expert;
}

hipError_t launch_sort_pairs(const PairsArgs &a, hipStream_t s) {
    const int64_t pairs = (int64_t)a.n_tokens * a.k;
    const int blocks = pairs ? (int)((pairs + kBlockPairs - 1) / kBlockPairs) : 1;
    int bits = 1;
    while ((1 << bits) <= a.n_expert) bits++;  // keys 0..n_expert
    if (blocks > 1) {
        count_kernel<<<blocks, kBlockPairs, 0, s>>>(a, pairs);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    if (blocks > kAddBlocks) {
        scan_kernel<<<(a.n_expert + 63) / 64, 1024, 0, s>>>(a, blocks);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    place_kernel<<<blocks, kBlockPairs, 0, s>>>(a, pairs, bits);
    return hipGetLastError();
}

hipError_t launch_gather(const RowsArgs &a, hipStream_t s) { HOARD_ROWS(gather_kernel, rows_grid(a)); }
hipError_t launch_combine(const RowsArgs &a, hipStream_t s) { HOARD_ROWS(combine_kernel, rows_grid(a)); }
hipError_t launch_combine_grad(const RowsArgs &a, hipStream_t s) {
    const int64_t groups = ((int64_t)a.n_tokens * a.k + 3) / 4;
    HOARD_ROWS(combine_grad_kernel, groups < (1 << 20) ? groups : (1 << 20));
}

}  // namespace hoard

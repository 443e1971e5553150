// Attention over a paged cache: how a call is split, and its parts joined
// (hoard_attn_decode).  The attention itself is in attn_tiles.h.
#include "attn.h"
#include "attn_split.h"
#include "opsdev.h"

namespace hoard {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

// A wave joins a row where there are many of them, of few parts each (64 sequences by 32 heads, two
// parts: 4.9 us, a workgroup a row 7.3; 80 tokens by 16 heads, 9 parts: 7.3 and 5.7).
constexpr int kJoinRows = 512, kJoinLanes = kRuns / 2;

// The parts of one row: their number, the first one's row in the workspace and the distance to
// the next one's.
struct RowParts {
    int parts, step;
    int64_t first;
};
__device__ __forceinline__ RowParts row_parts(const AttnCall &p, int token, int head) {
    const hoard_attn_args &a = p.a;
    const int seq = token / a.n_new, group = a.n_q_heads / p.c.n_kv_heads;
    const int row = token % a.n_new * group + head % group, block = row / p.block_rows;
    const int lanes = p.c.n_kv_heads * p.row_blocks, of = head / group * p.row_blocks + block;
    // the lane's tiles, and the workgroups whose runs they fall in
    const int before = seq ? p.sums[seq - 1] : 0, run = p.sums[a.n_seq], own = p.sums[a.n_seq + 1];
    const int tiles = (p.sums[seq] - before) / lanes, begin = before + of * tiles, from_run = begin / run;
    return RowParts{(begin + tiles - 1) / run - from_run + 1, p.block_rows,
                    (from_run + (own ? 0 : (int64_t)seq * lanes + of)) * p.block_rows + row % p.block_rows};
}

// out = sum_s w_s part_s,  w_s = l_s 2^(m_s - m) / sum: the parts of one row, each already
// divided by its own sum l_s of weights, formed by its own largest score m_s.  (Not by the
// logarithm of the two: far from zero it would have no digits left for the sum.)  The weights are
// divided before they meet the parts, so that no sum is larger than these are.
//
// A workgroup takes a row: four columns a thread, the parts dealt to the threads left over,
// which meet in LDS.  What a thread reads first it asks for before the weights are known: the
// launch is latency alone.
constexpr int kFetch = 8;
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnCall p) {
    __shared__ float weight[kRuns], stat[2][4];
    __shared__ v4f outs[256];
    const int token = blockIdx.x, head = blockIdx.y;
    const RowParts row = row_parts(p, token, head);
    if (row.parts == 1) return;
    const int lane = threadIdx.x & 63, dim = p.c.head_dim;
    const v2f none = {-INFINITY, 0.0f};
    const v2f mine = (int)threadIdx.x < row.parts ? reinterpret_cast<const v2f *>(p.part_stat)[row.first + (int64_t)threadIdx.x * row.step] : none;
    const int quads = dim / 4, deep = 256 / quads, quad = threadIdx.x % quads, from = threadIdx.x / quads;
    const float *part = p.part_out + row.first * dim + 4 * quad;
    v4f ahead[kFetch];
#pragma unroll
    for (int i = 0; i < kFetch; i++)
        ahead[i] = *reinterpret_cast<const v4f *>(part + (int64_t)min(from + i * deep, row.parts - 1) * row.step * dim);
    const float top = wave_max_f(mine[0]);
    if (lane == 0) stat[0][wave_index()] = top;
    __syncthreads();
    float m = fmaxf(fmaxf(stat[0][0], stat[0][1]), fmaxf(stat[0][2], stat[0][3]));
    m = m > -INFINITY ? m : 0.0f;
    const float w = exp2f(mine[0] - m) * mine[1], s = wave_sum_f(w);  // a NaN is everyone's
    if (lane == 0) stat[1][wave_index()] = s;
    weight[threadIdx.x] = w;
    __syncthreads();
    const float sum = (stat[1][0] + stat[1][1]) + (stat[1][2] + stat[1][3]), f = sum != 0.0f ? 1.0f / sum : 0.0f;
    v4f o = {0, 0, 0, 0};
    if (from < deep) {
#pragma unroll
        for (int i = 0; i < kFetch; i++)
            if (from + i * deep < row.parts) o += weight[from + i * deep] * f * ahead[i];
#pragma unroll 4
        for (int i = from + kFetch * deep; i < row.parts; i += deep)
            o += weight[i] * f * *reinterpret_cast<const v4f *>(part + (int64_t)i * row.step * dim);
    }
    outs[threadIdx.x] = o;
    __syncthreads();
    const int64_t out = (int64_t)token * p.a.n_q_heads + head;
    if (from == 0) {
        for (int i = 1; i < deep; i++) o += outs[i * quads + quad];
        T *to = static_cast<T *>(p.a.out) + out * dim + 4 * quad;
#pragma unroll
        for (int k = 0; k < 4; k++) to[k] = (T)o[k];
    }
    if (threadIdx.x == 0 && p.a.lse) p.a.lse[out] = (m + log2f(sum)) * 0.6931471805599453f;
}

// Many rows of few parts: a wave takes one, its lanes four columns each.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_rows_kernel(AttnCall p) {
    const int64_t out = (int64_t)blockIdx.x * 4 + wave_index();
    if (out >= (int64_t)p.a.n_seq * p.a.n_new * p.a.n_q_heads) return;
    const RowParts row = row_parts(p, (int)(out / p.a.n_q_heads), (int)(out % p.a.n_q_heads));
    if (row.parts == 1) return;
    const int lane = threadIdx.x & 63, dim = p.c.head_dim, quad = min(lane, dim / 4 - 1);
    const float *part = p.part_out + row.first * dim + 4 * quad;
    const v4f first = *reinterpret_cast<const v4f *>(part), second = *reinterpret_cast<const v4f *>(part + (int64_t)row.step * dim);
    const v2f none = {-INFINITY, 0.0f};
    v2f stat[kRuns / 64];
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kRuns / 64; i++) {
        stat[i] = i * 64 + lane < row.parts ? reinterpret_cast<const v2f *>(p.part_stat)[row.first + (int64_t)(i * 64 + lane) * row.step] : none;
        m = fmaxf(m, stat[i][0]);
    }
    m = wave_max_f(m);
    m = m > -INFINITY ? m : 0.0f;
    float weight[kRuns / 64];
#pragma unroll
    for (int i = 0; i < kRuns / 64; i++) {
        weight[i] = exp2f(stat[i][0] - m) * stat[i][1];
        sum += weight[i];
    }
    sum = wave_sum_f(sum);
    const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
    v4f o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kRuns / 64; i++) {
        const float w = weight[i] * f;
#pragma unroll 4
        for (int j = 0; j < min(row.parts - i * 64, 64); j++) {
            const float wj = readlane_f(w, j);
            o += wj * (i == 0 && j < 2 ? (j ? second : first) : *reinterpret_cast<const v4f *>(part + (int64_t)(i * 64 + j) * row.step * dim));
        }
    }
    if (lane < dim / 4) {
        T *to = static_cast<T *>(p.a.out) + out * dim + 4 * quad;
#pragma unroll
        for (int k = 0; k < 4; k++) to[k] = (T)o[k];
    }
    if (lane == 0 && p.a.lse) p.a.lse[out] = (m + log2f(sum)) * 0.6931471805599453f;
}

template <typename T>
void join(const AttnCall &p, hipStream_t s) {
    const int64_t rows = (int64_t)p.a.n_seq * p.a.n_new * p.a.n_q_heads;
    if (rows >= kJoinRows && attn_lanes(p) >= kJoinLanes) attn_join_rows_kernel<T><<<(int)((rows + 3) / 4), 256, 0, s>>>(p);
    else attn_join_kernel<T><<<dim3(p.a.n_seq * p.a.n_new, p.a.n_q_heads), 256, 0, s>>>(p);
}

// Lanes of so many tiles are not cut: the join takes longer than it gains (512 tokens by 4 lanes
// 8.3 us in the kernel, some 10 with a join; 1024 tokens 12.5 and 10.3).
constexpr int kWholeTiles = 16;

// Waves side by side over the rows where there are more than 16, which so read a tile at about
// the same time; of three tiles of rows the fourth wave has none.  (Two tiles of rows a wave, that
// unpack keys and values once for both, took 38.5 us against 47 for 16 new tokens of one sequence
// over 32768 keys, but 30 to 36 against 27 to 33 for 16 sequences of 3 new tokens by 8 heads, 3000
// keys, and spilled in fp32 at 256 columns.)
AttnCall call_of(const hoard_kv_cache &c, const hoard_attn_args &a, float *work) {
    AttnCall p{};
    p.c = c;
    p.a = a;
    const int rows = a.n_new * (a.n_q_heads / c.n_kv_heads), tiles = (rows + 15) / 16;
    p.row_waves = tiles >= 3 ? 4 : tiles;
    p.row_blocks = (tiles + p.row_waves - 1) / p.row_waves;
    p.min_run = kAttnWaves / p.row_waves;
    p.block_rows = rows < 16 * p.row_waves ? rows : 16 * p.row_waves;
    // cut where the lanes alone would leave the chip half empty, and there is something to cut (by
    // the table's width: how uneven the lengths are only the device knows, so one long sequence
    // among 512 lanes is not cut: 100000 tokens among 127 sequences of 500 by 4 key heads 752 us, 62
    // among 126); the row of tiles, three times (runs behind its end have numbers too), in 32 bits
    const int64_t tiles_most = ((int64_t)a.max_pages * c.page + kKeyTile - 1) / kKeyTile;
    p.split = attn_lanes(p) < 2 * kRuns && a.n_seq <= kMaxSplitSeqs && tiles_most > kWholeTiles && attn_lanes(p) * tiles_most < 1 << 28;
    if (p.split) {
        p.part_out = work;
        p.part_stat = work ? work + attn_parts(p) * p.block_rows * c.head_dim : nullptr;
        p.sums = work ? reinterpret_cast<int32_t *>(p.part_stat + 2 * attn_parts(p) * p.block_rows) : nullptr;
    }
    return p;
}

constexpr int64_t kMaxGrid = 1 << 23;

}  // namespace

size_t attn_work_bytes(const hoard_kv_cache &c, const hoard_attn_args &a) {
    const AttnCall p = call_of(c, a, nullptr);
    return p.split ? sizeof(float) * ((size_t)(c.head_dim + 2) * attn_parts(p) * p.block_rows + a.n_seq + 2) : 0;
}

hipError_t launch_attn(const hoard_kv_cache &c, const hoard_attn_args &a, float *work, hipStream_t s) {
    AttnCall p = call_of(c, a, work);
    // as many sequences at a time as a grid takes
    const int64_t lanes = (int64_t)c.n_kv_heads * p.row_blocks, at_once = kMaxGrid / lanes > 1 ? kMaxGrid / lanes : 1;
    const size_t z = a.type == HOARD_TYPE_F32 ? 4 : 2;
    for (int64_t seq = 0; seq < a.n_seq; seq += at_once) {
        const int64_t token = seq * a.n_new;
        p.a.n_seq = (int)(a.n_seq - seq < at_once ? a.n_seq - seq : at_once);
        p.a.q = static_cast<const char *>(a.q) + token * a.q_stride * z;
        p.a.pages = a.pages + seq * a.max_pages;
        p.a.lens = a.lens + token;
        p.a.out = static_cast<char *>(a.out) + token * a.n_q_heads * c.head_dim * z;
        p.a.lse = a.lse ? a.lse + token * a.n_q_heads : nullptr;
        const hipError_t rc = c.type == HOARD_TYPE_F16    ? launch_attn_f16(p, s)
                              : c.type == HOARD_TYPE_BF16 ? launch_attn_bf16(p, s)
                                                          : launch_attn_i8(p, s);
        if (rc != hipSuccess) return rc;
    }
    if (!p.split) return hipSuccess;
    if (a.type == HOARD_TYPE_F32) join<float>(p, s);
    else if (a.type == HOARD_TYPE_F16) join<f16>(p, s);
    else join<bf16>(p, s);
    return hipGetLastError();
}

}  // namespace hoard

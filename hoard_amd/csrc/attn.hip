// Attention over a paged cache: how a call is split, and its parts joined
// (hoard_attn_decode).  The attention itself is in attn_tiles.h.
#include "attn.h"
#include "attn_split.h"
#include "opsdev.h"

namespace hoard {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

// out = sum_s w_s part_s,  w_s = 2^(lse_s - m) / sum: the parts of one row, each already
// divided by its own sum.  A workgroup takes a row: four columns a thread, the parts dealt
// to the threads left over, which meet in LDS.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnCall p) {
    __shared__ float weight[kMaxSplits], stat[2][4];
    __shared__ v4f outs[256];
    const hoard_attn_args &a = p.a;
    const int64_t token = blockIdx.x, row = token * a.n_q_heads + blockIdx.y, seq = token / a.n_new;
    const int lane = threadIdx.x & 63, dim = p.c.head_dim;
    const int limit = a.max_pages * p.c.page;
    int most = 0;
    for (int t = 0; t < a.n_new; t++) most = max(most, min(max(a.lens[seq * a.n_new + t], 0), limit));
    const AttnParts parts = attn_parts(most, p.splits, 4 / p.row_waves);
    if (parts.used <= 1) return;
    const float *lse = p.part_lse + row * p.splits;
    const float mine = (int)threadIdx.x < parts.used ? lse[threadIdx.x] : -INFINITY;
    // a NaN of one part is everyone's
    const float top = wave_max_f(mine);
    if (lane == 0) stat[0][wave_index()] = top;
    __syncthreads();
    float m = fmaxf(fmaxf(stat[0][0], stat[0][1]), fmaxf(stat[0][2], stat[0][3]));
    m = m > -INFINITY ? m : 0.0f;
    const float w = exp2f(mine - m), s = wave_sum_f(w);
    if (lane == 0) stat[1][wave_index()] = s;
    if ((int)threadIdx.x < kMaxSplits) weight[threadIdx.x] = w;
    __syncthreads();
    const float sum = (stat[1][0] + stat[1][1]) + (stat[1][2] + stat[1][3]), f = sum != 0.0f ? 1.0f / sum : 0.0f;
    const int quads = dim / 4, deep = 256 / quads, quad = threadIdx.x % quads, from = threadIdx.x / quads;
    v4f o = {0, 0, 0, 0};
    if (from < deep) {
        const float *part = p.part_out + row * p.splits * dim + 4 * quad;
#pragma unroll 4
        for (int i = from; i < parts.used; i += deep) {
            const float wi = weight[i];
            // a part of which the row sees nothing holds zeros
            o += wi * *reinterpret_cast<const v4f *>(part + (int64_t)i * dim);
        }
    }
    outs[threadIdx.x] = o;
    __syncthreads();
    if (from == 0) {
        for (int i = 1; i < deep; i++) o += outs[i * quads + quad];
        T *to = static_cast<T *>(a.out) + row * dim + 4 * quad;
#pragma unroll
        for (int k = 0; k < 4; k++) to[k] = (T)(o[k] * f);
    }
    if (threadIdx.x == 0 && a.lse) a.lse[row] = (m + log2f(sum)) * 0.6931471805599453f;
}

// Waves side by side over the rows where there are more than 16; workgroups for about two
// a CU, a sequence split into as many parts as that leaves.
AttnCall call_of(const hoard_kv_cache &c, const hoard_attn_args &a, float *work) {
    AttnCall p{};
    p.c = c;
    p.a = a;
    const int rows = a.n_new * (a.n_q_heads / c.n_kv_heads), tiles = (rows + 15) / 16;
    p.row_waves = tiles >= 4 ? 4 : tiles >= 2 ? 2 : 1;
    p.row_blocks = (tiles + p.row_waves - 1) / p.row_waves;
    const int64_t groups = (int64_t)a.n_seq * c.n_kv_heads * p.row_blocks;
    const int64_t keys = (int64_t)a.max_pages * c.page, deep = 4 / p.row_waves;
    const int64_t most = (keys + kKeyTile * deep - 1) / (kKeyTile * deep);
    int64_t splits = groups ? kAttnGroups / groups : 1;
    splits = splits > most ? most : splits;
    p.splits = (int)(splits < 1 ? 1 : splits > kMaxSplits ? kMaxSplits : splits);
    const int64_t all = (int64_t)a.n_seq * a.n_new * a.n_q_heads * p.splits;
    p.part_out = work;
    p.part_lse = work ? work + all * c.head_dim : nullptr;
    return p;
}

}  // namespace

size_t attn_work_bytes(const hoard_kv_cache &c, const hoard_attn_args &a) {
    const AttnCall p = call_of(c, a, nullptr);
    if (p.splits == 1) return 0;
    return sizeof(float) * (size_t)(c.head_dim + 1) * a.n_seq * a.n_new * a.n_q_heads * p.splits;
}

hipError_t launch_attn(const hoard_kv_cache &c, const hoard_attn_args &a, float *work, hipStream_t s) {
    const AttnCall p = call_of(c, a, work);
    const hipError_t rc = c.type == HOARD_TYPE_F16    ? launch_attn_f16(p, s)
                          : c.type == HOARD_TYPE_BF16 ? launch_attn_bf16(p, s)
                                                      : launch_attn_i8(p, s);
    if (rc != hipSuccess || p.splits == 1) return rc;
    const dim3 grid(a.n_seq * a.n_new, a.n_q_heads);
    if (a.type == HOARD_TYPE_F32) attn_join_kernel<float><<<grid, 256, 0, s>>>(p);
    else if (a.type == HOARD_TYPE_F16) attn_join_kernel<f16><<<grid, 256, 0, s>>>(p);
    else attn_join_kernel<bf16><<<grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

}  // namespace hoard

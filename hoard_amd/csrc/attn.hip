// Attention of a few new tokens a sequence over a paged cache (hoard_attn_decode).
//
//   S_j = scale <q, k_j>,  out = sum_j exp(S_j - m) v_j / sum_j exp(S_j - m),  m = max_j S_j,
// over the keys that the row sees; lse = m + log sum_j exp(S_j - m).
//
// A workgroup takes one query head of one new token, its four waves every fourth run of 64
// keys: a lane forms its key's score, then the lanes take the columns of the values.  Sums
// and maxima of what a wave has seen run along and are joined at the end.
#include "attn.h"
#include "opsdev.h"

namespace hoard {

namespace {

// The cache's row of key j; -1 where its page is none.
__device__ __forceinline__ int64_t row_of(const hoard_kv_cache &c, const int32_t *pages, int head, int j) {
    const int page = pages[j / c.page];
    if (page < 0 || page >= c.n_pages) return -1;
    return ((int64_t)page * c.n_kv_heads + head) * c.page + j % c.page;
}

template <typename T, typename C>
__global__ __launch_bounds__(256) void attn_kernel(hoard_kv_cache c, hoard_attn_args a) {
    __shared__ float q[256], part[4][256], top[4], sum[4];
    const int64_t token = blockIdx.x;
    const int head = blockIdx.y, kv = head / (a.n_q_heads / c.n_kv_heads), dim = c.head_dim;
    const int lane = threadIdx.x & 63, wave = wave_index();
    const int n = (int)min((int64_t)a.lens[token], (int64_t)a.max_pages * c.page);
    const int32_t *pages = a.pages + token / a.n_new * a.max_pages;
    if ((int)threadIdx.x < dim) q[threadIdx.x] = (float)(static_cast<const T *>(a.q) + token * a.q_stride + head * dim)[threadIdx.x];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[4] = {};
    for (int at = wave * 64; at < n; at += 256) {
        const int j = at + lane;
        const int64_t row = j < n ? row_of(c, pages, kv, j) : -1;
        float s = -INFINITY;
        if (row >= 0) {
            const C *k = static_cast<const C *>(c.k) + row * dim;
            s = 0.0f;
            for (int d = 0; d < dim; d++) s = fmaf(q[d], (float)k[d], s);
            s *= a.scale;
            if (sizeof(C) == 1) s *= c.k_scale[row];
        }
        const uint64_t seen = __ballot(row >= 0);
        if (!seen) continue;
        float most = row >= 0 ? s : -INFINITY;
        for (int off = 1; off < 64; off *= 2) most = fmaxf(most, __shfl_xor(most, off));
        most = fmaxf(m, most);
        const float base = most > -INFINITY ? most : 0.0f, old = expf(m - base);
        const float e = row >= 0 ? expf(s - base) : 0.0f;
        m = most;
        l = l * old + wave_sum_f(e);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] *= old;
        for (int i = 0; i < 64; i++) {
            if (!(seen >> i & 1)) continue;
            const int64_t r = __shfl(row, i);
            float w = __shfl(e, i);
            if (sizeof(C) == 1) w *= c.v_scale[r];
            const C *v = static_cast<const C *>(c.v) + r * dim;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (lane + 64 * k < dim) acc[k] = fmaf(w, (float)v[lane + 64 * k], acc[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++) part[wave][lane + 64 * k] = acc[k];
    if (lane == 0) {
        top[wave] = m;
        sum[wave] = l;
    }
    __syncthreads();
    m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    const float base = m > -INFINITY ? m : 0.0f;
    float o = 0.0f;
    l = 0.0f;
    for (int w = 0; w < 4; w++) {
        const float f = expf(top[w] - base);
        l += f * sum[w];
        o += f * part[w][threadIdx.x];
    }
    if ((int)threadIdx.x < dim)
        (static_cast<T *>(a.out) + (token * a.n_q_heads + head) * dim)[threadIdx.x] = (T)(l != 0.0f ? o / l : 0.0f);
    if (threadIdx.x == 0 && a.lse) a.lse[token * a.n_q_heads + head] = base + logf(l);
}

template <typename T>
void attn_type(const hoard_kv_cache &c, const hoard_attn_args &a, hipStream_t s) {
    const dim3 grid(a.n_seq * a.n_new, a.n_q_heads);
    if (c.type == HOARD_TYPE_F16) attn_kernel<T, f16><<<grid, 256, 0, s>>>(c, a);
    else if (c.type == HOARD_TYPE_BF16) attn_kernel<T, bf16><<<grid, 256, 0, s>>>(c, a);
    else attn_kernel<T, int8_t><<<grid, 256, 0, s>>>(c, a);
}

}  // namespace

size_t attn_work_bytes(const hoard_kv_cache &, const hoard_attn_args &) { return 0; }

hipError_t launch_attn(const hoard_kv_cache &c, const hoard_attn_args &a, float *, hipStream_t s) {
    if (a.type == HOARD_TYPE_F32) attn_type<float>(c, a, s);
    else if (a.type == HOARD_TYPE_F16) attn_type<f16>(c, a, s);
    else attn_type<bf16>(c, a, s);
    return hipGetLastError();
}

}  // namespace hoard

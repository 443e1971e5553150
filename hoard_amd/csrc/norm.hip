// Norms around a block (hoard_norm_forward, hoard_norm_backward).
//
// Forward, per row of n values:  c = b rho_b (o + w_post),  v = r + s g c,
// h = v rho_v (o + w_pre),  rho_x = (mean x^2 + eps)^(-1/2).
// Backward, with u = dh (o + w_pre):
//   dv     = dr_out + rho_v (u - v rho_v^2 mean(u v)),      dr = dv
//   dgate  = s dv c (times g (1 - g) behind a sigmoid; summed over the rows for
//            a channel's gate, over the columns for a row's)
//   u2     = s g dv (o + w_post),  db = rho_b (u2 - b rho_b^2 mean(u2 b))
//   dw_pre = sum over rows of dh v rho_v,  dw_post = sum over rows of s g dv b rho_b.
//
// Both are bound by memory: a row's inputs are read once into registers (8
// values a thread and chunk), both norms' sums are formed from there, and the
// outputs are written from there.
#include "ops.h"
#include "opsdev.h"

namespace hoard {

namespace {

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// The gate of eight values as it is stored.
template <typename T>
__device__ __forceinline__ void load_gate(const hoard_norm_args &a, size_t row, int at, int some, float g[8]) {
    if (a.gate_kind == HOARD_GATE_CHANNEL) {
        load_some(static_cast<const float *>(a.gate) + at, some, g);
    } else if (a.gate_kind == HOARD_GATE_FULL) {
        load_some(static_cast<const T *>(a.gate) + row * a.n + at, some, g);
    } else {
        const float t = a.gate_kind == HOARD_GATE_TOKEN ? static_cast<const float *>(a.gate)[row] : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = t;
    }
}

// A workgroup of BS threads takes a row at a time; NV chunks of BS * 8 values cover it.
template <typename T, typename R, int BS, int NV>
__global__ __launch_bounds__(BS) void norm_kernel(hoard_norm_args a) {
    __shared__ float part[2][2][BS / 64];
    const float inv_n = 1.0f / (float)a.n;
    int at[NV], some[NV];
#pragma unroll
    for (int c = 0; c < NV; c++) {
        at[c] = (c * BS + (int)threadIdx.x) * 8;
        some[c] = max(0, min(8, a.n - at[c]));
    }
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)a.n_rows; row += gridDim.x, turn ^= 1) {
        const size_t base = row * a.n;
        float v[NV][8], b[NV][8];
#pragma unroll
        for (int c = 0; c < NV; c++) {
            load_some(static_cast<const R *>(a.r) + base + at[c], some[c], v[c]);
            if (a.b) load_some(static_cast<const T *>(a.b) + base + at[c], some[c], b[c]);
        }
        float rho_b = 1.0f, rho_v = 1.0f;
        if (a.b) {
            if (a.w_post) {
                float s = 0.0f;
#pragma unroll
                for (int c = 0; c < NV; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) s = fmaf(b[c][i], b[c][i], s);
                s = group_sum<BS / 64>(s, part[turn][0]);
                rho_b = 1.0f / sqrtf(fmaf(s, inv_n, a.eps));
            }
#pragma unroll
            for (int c = 0; c < NV; c++) {
                float g[8], w[8] = {};
                load_gate<T>(a, row, at[c], some[c], g);
                if (a.w_post) load_some(a.w_post + at[c], some[c], w);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (a.gate_sigmoid) g[i] = sigmoid(g[i]);
                    const float cc = a.w_post ? b[c][i] * rho_b * (a.w_offset + w[i]) : b[c][i];
                    // rounded here: the norm that follows is the stored stream's, as whoever reads it
                    // (the gradient, the next layer) sees it
                    v[c][i] = i < some[c] ? (float)(R)fmaf(a.scale * g[i], cc, v[c][i]) : 0.0f;
                }
                store_some(static_cast<R *>(a.r_out) + base + at[c], some[c], v[c]);
            }
        }
        if (a.h) {
            float s = 0.0f;
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(v[c][i], v[c][i], s);
            s = group_sum<BS / 64>(s, part[turn][1]);
            rho_v = 1.0f / sqrtf(fmaf(s, inv_n, a.eps));
#pragma unroll
            for (int c = 0; c < NV; c++) {
                float w[8];
                load_some(a.w_pre + at[c], some[c], w);
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = v[c][i] * rho_v * (a.w_offset + w[i]);
                store_some(static_cast<T *>(a.h) + base + at[c], some[c], w);
            }
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * row] = rho_b;
            a.stats[2 * row + 1] = rho_v;
        }
    }
}

// Group blockIdx.x takes the rows blockIdx.x, + gridDim.x, ...: the sums over its
// rows stay in registers and go to its rows of the workspace, one per wanted
// parameter ([parameter][group][n]).
template <typename T, typename R, int BS, int NV>
__global__ __launch_bounds__(BS) void norm_grad_kernel(hoard_norm_args a, hoard_norm_grads g, float *work) {
    __shared__ float part[2][3][BS / 64];
    const float inv_n = 1.0f / (float)a.n;
    float s_pre[NV][8] = {}, s_post[NV][8] = {}, s_gate[NV][8] = {};
    int at[NV], some[NV];
#pragma unroll
    for (int c = 0; c < NV; c++) {
        at[c] = (c * BS + (int)threadIdx.x) * 8;
        some[c] = max(0, min(8, a.n - at[c]));
    }
    const bool block = g.db || g.dgate || g.dw_post;
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)a.n_rows; row += gridDim.x, turn ^= 1) {
        const size_t base = row * a.n;
        const float rho_b = a.stats[2 * row], rho_v = a.stats[2 * row + 1];
        float dv[NV][8];
        if (g.dh) {
            float v[NV][8], u[NV][8], s = 0.0f;
#pragma unroll
            for (int c = 0; c < NV; c++) {
                float w[8];
                load_some(static_cast<const R *>(a.r_out) + base + at[c], some[c], v[c]);
                load_some(static_cast<const T *>(g.dh) + base + at[c], some[c], u[c]);
                load_some(a.w_pre + at[c], some[c], w);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    s_pre[c][i] = fmaf(u[c][i], v[c][i] * rho_v, s_pre[c][i]);
                    u[c][i] *= a.w_offset + w[i];
                    s = fmaf(u[c][i], v[c][i], s);
                }
            }
            s = group_sum<BS / 64>(s, part[turn][0]) * inv_n * rho_v * rho_v;
#pragma unroll
            for (int c = 0; c < NV; c++) {
                if (g.dr_out) {
                    load_some(static_cast<const R *>(g.dr_out) + base + at[c], some[c], dv[c]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) dv[c][i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) dv[c][i] += rho_v * (u[c][i] - v[c][i] * s);
            }
        } else {
#pragma unroll
            for (int c = 0; c < NV; c++) load_some(static_cast<const R *>(g.dr_out) + base + at[c], some[c], dv[c]);
        }
        if (g.dr) {
#pragma unroll
            for (int c = 0; c < NV; c++) store_some(static_cast<R *>(g.dr) + base + at[c], some[c], dv[c]);
        }
        if (!block) continue;
        float b[NV][8], s_b = 0.0f, s_g = 0.0f;
#pragma unroll
        for (int c = 0; c < NV; c++) {
            float q[8], w[8], dg[8];
            load_some(static_cast<const T *>(a.b) + base + at[c], some[c], b[c]);
            load_gate<T>(a, row, at[c], some[c], q);
            if (a.w_post) load_some(a.w_post + at[c], some[c], w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float t = a.gate_sigmoid ? sigmoid(q[i]) : q[i];
                const float slope = a.gate_sigmoid ? t * (1.0f - t) : 1.0f;
                const float wp = a.w_post ? a.w_offset + w[i] : 1.0f;
                const float d = a.scale * dv[c][i];  // of g c
                const float nb = b[c][i] * rho_b;    // rho_b is 1 without a norm
                dg[i] = d * nb * wp * slope;
                s_gate[c][i] += dg[i];
                s_g += dg[i];
                s_post[c][i] = fmaf(d * t, nb, s_post[c][i]);
                dv[c][i] = d * t * wp;  // u2 from here on
                s_b = fmaf(dv[c][i], b[c][i], s_b);
            }
            if (a.gate_kind == HOARD_GATE_FULL && g.dgate)
                store_some(static_cast<T *>(g.dgate) + base + at[c], some[c], dg);
        }
        if (a.gate_kind == HOARD_GATE_TOKEN && g.dgate) {
            s_g = group_sum<BS / 64>(s_g, part[turn][2]);
            if (threadIdx.x == 0) static_cast<float *>(g.dgate)[row] = s_g;
        }
        if (!g.db) continue;
        if (a.w_post) {
            s_b = group_sum<BS / 64>(s_b, part[turn][1]) * inv_n * rho_b * rho_b;
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) dv[c][i] = rho_b * (dv[c][i] - b[c][i] * s_b);
        }
#pragma unroll
        for (int c = 0; c < NV; c++) store_some(static_cast<T *>(g.db) + base + at[c], some[c], dv[c]);
    }
    const size_t mine = (size_t)blockIdx.x * a.n, all = (size_t)gridDim.x * a.n;
    float *to = work;
#pragma unroll
    for (int c = 0; c < NV; c++) {
        float *p = to;
        if (g.dw_pre) {
            store_some(p + mine + at[c], some[c], s_pre[c]);
            p += all;
        }
        if (g.dw_post) {
            store_some(p + mine + at[c], some[c], s_post[c]);
            p += all;
        }
        if (g.dgate && a.gate_kind == HOARD_GATE_CHANNEL) store_some(p + mine + at[c], some[c], s_gate[c]);
    }
}

// The groups' partial sums [parameter][groups][n] added: a workgroup takes 64
// columns, its 16 waves a sixteenth of the groups each, in ascending order.
struct SumOut {
    float *out[3];
};
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float *work, int groups, int n, SumOut o) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    const int per = (groups + 15) / 16, g0 = wave * per, g1 = min(groups, g0 + per);
    float s = 0.0f;
    if (col < n) {
        const float *p = work + (size_t)blockIdx.y * groups * n + col;
#pragma unroll 8
        for (int g = g0; g < g1; g++) s += p[(size_t)g * n];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += part[i][lane];
    if (col < n) o.out[blockIdx.y][col] = s;
}

template <typename T, typename R, int BS, int NV>
void forward_of(const hoard_norm_args &a, hipStream_t s) {
    norm_kernel<T, R, BS, NV><<<min(a.n_rows, 1 << 20), BS, 0, s>>>(a);
}
template <typename T, typename R, int BS, int NV>
void grad_of(const hoard_norm_args &a, const hoard_norm_grads &g, float *work, hipStream_t s) {
    norm_grad_kernel<T, R, BS, NV><<<norm_groups(a.n_rows, a.n), BS, 0, s>>>(a, g, work);
}

// f(T, R, BS, NV) for the types and the row length: BS * 8 * NV >= n.
#define HOARD_NORM_SIZES(F, T, R, ...)                  \
    do {                                                \
        if (a.n <= 512) F<T, R, 64, 1>(__VA_ARGS__);        \
        else if (a.n <= 1024) F<T, R, 64, 2>(__VA_ARGS__);  \
        else if (a.n <= 2048) F<T, R, 256, 1>(__VA_ARGS__); \
        else if (a.n <= 4096) F<T, R, 256, 2>(__VA_ARGS__); \
        else if (a.n <= 8192) F<T, R, 1024, 1>(__VA_ARGS__);\
        else F<T, R, 1024, 2>(__VA_ARGS__);                 \
    } while (0)
#define HOARD_NORM_TYPES(F, ...)                                                                         \
    do {                                                                                                 \
        if (a.type == HOARD_TYPE_F32) HOARD_NORM_SIZES(F, float, float, __VA_ARGS__);                    \
        else if (a.type == HOARD_TYPE_F16 && a.res_type == HOARD_TYPE_F32) HOARD_NORM_SIZES(F, f16, float, __VA_ARGS__); \
        else if (a.type == HOARD_TYPE_F16) HOARD_NORM_SIZES(F, f16, f16, __VA_ARGS__);                   \
        else if (a.res_type == HOARD_TYPE_F32) HOARD_NORM_SIZES(F, bf16, float, __VA_ARGS__);            \
        else HOARD_NORM_SIZES(F, bf16, bf16, __VA_ARGS__);                                               \
    } while (0)

}  // namespace

int norm_groups(int n_rows, int n) {
    (void)n;
    return n_rows < 512 ? n_rows : 512;
}

hipError_t launch_norm(const hoard_norm_args &a, hipStream_t s) {
    if (!a.n_rows) return hipSuccess;
    HOARD_NORM_TYPES(forward_of, a, s);
    return hipGetLastError();
}

hipError_t launch_norm_grad(const hoard_norm_args &a, const hoard_norm_grads &g, float *work, hipStream_t s) {
    if (a.n_rows) {
        HOARD_NORM_TYPES(grad_of, a, g, work, s);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    SumOut o{};
    int params = 0;
    if (g.dw_pre) o.out[params++] = g.dw_pre;
    if (g.dw_post) o.out[params++] = g.dw_post;
    if (g.dgate && a.gate_kind == HOARD_GATE_CHANNEL) o.out[params++] = static_cast<float *>(g.dgate);
    if (!params) return hipSuccess;
    norm_sum_kernel<<<dim3((a.n + 63) / 64, params), 1024, 0, s>>>(work, norm_groups(a.n_rows, a.n), a.n, o);
    return hipGetLastError();
}

}  // namespace hoard

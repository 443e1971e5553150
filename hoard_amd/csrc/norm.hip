// Norms around a block (hoard_norm_forward, hoard_norm_backward).
//
// Forward, per row of n values:  c = b rho_b (o + w_post),  v = r + s g c,
// h = v rho_v (o + w_pre),  rho_x = (mean x^2 + eps)^(-1/2).
// Backward, with u = dh (o + w_pre):
//   dv     = dr_out + rho_v (u - v rho_v^2 mean(u v)),      dr = dv
//   dgate  = s dv c (times the sigmoid's derivative behind one; summed over the rows for
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
// The sigmoid and its derivative e / (1 + e)^2, e = exp(-|x|): as s (1 - s) it would keep
// none of its digits where s is close to 1.
__device__ __forceinline__ float sigmoid_slope(float x, float &slope) {
    const float e = expf(-fabsf(x)), r = 1.0f / (1.0f + e);
    slope = e * r * r;
    return x < 0.0f ? e * r : r;
}

// The gate of eight columns as it is stored: 32-bit values of a channel gate, those of
// a full one, or the row's in the first word.
struct Gate {
    u128 w[2];
};
template <typename T>
__device__ __forceinline__ Gate fetch_gate(const hoard_norm_args &a, size_t row, Cols c) {
    Gate g;
    if (a.gate_kind == HOARD_GATE_CHANNEL) {
        const Raw<float> r = fetch(static_cast<const float *>(a.gate), c, a.n);
        __builtin_memcpy(&g, &r, sizeof r);
    } else if (a.gate_kind == HOARD_GATE_FULL) {
        const Raw<T> r = fetch(static_cast<const T *>(a.gate) + row * a.n, c, a.n);
        __builtin_memcpy(&g, &r, sizeof r);
    } else {
        g.w[0][0] = static_cast<const uint32_t *>(a.gate)[row];
    }
    return g;
}
template <typename T>
__device__ __forceinline__ void gate_of(const hoard_norm_args &a, const Gate &g, float o[8]) {
    if (a.gate_kind == HOARD_GATE_CHANNEL) {
        Raw<float> r;
        __builtin_memcpy(&r, &g, sizeof r);
        widen(r, o);
    } else if (a.gate_kind == HOARD_GATE_FULL) {
        Raw<T> r;
        __builtin_memcpy(&r, &g, sizeof r);
        widen(r, o);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = __uint_as_float(g.w[0][0]);
    }
}

// A workgroup of BS threads takes a row at a time; NV chunks of BS * 8 values cover it.
// Everything that the row needs is fetched before the first sum; in workgroups of 256
// and more, with more waves to hide them, the gate and the weights come late (4096 rows
// of 2048: 15.8 us against 17.6; of 4096: 51.7 against 53.6).
template <typename T, typename R, int BS, int NV, bool NT>
__global__ __launch_bounds__(BS) void norm_kernel(hoard_norm_args a) {
    constexpr bool EARLY = BS < 256;
    __shared__ float part[2][2][BS / 64];
    const float inv_n = 1.0f / (float)a.n;
    Cols c[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) c[k] = cols_of((k * BS + (int)threadIdx.x) * 8, a.n);
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)a.n_rows; row += gridDim.x, turn ^= 1) {
        const size_t base = row * a.n;
        Raw<R> r[NV];
        Raw<T> br[NV];
        Raw<float> wp[NV], wq[NV];
        Gate gate[NV];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (a.b) br[k] = fetch(static_cast<const T *>(a.b) + base, c[k], a.n);
            r[k] = fetch(static_cast<const R *>(a.r) + base, c[k], a.n);
        }
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (EARLY && a.w_post) wp[k] = fetch(a.w_post, c[k], a.n);
            if (EARLY && a.gate) gate[k] = fetch_gate<T>(a, row, c[k]);
            if (EARLY && a.h) wq[k] = fetch(a.w_pre, c[k], a.n);
        }
        float rho_b = 1.0f, rho_v = 1.0f, v[NV][8];
        if (a.b) {
            if (a.w_post) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < NV; k++) {
                    float b[8];
                    widen(br[k], b);
                    mask_cols(c[k], b);
#pragma unroll
                    for (int i = 0; i < 8; i++) s = fmaf(b[i], b[i], s);
                }
                s = group_sum<BS / 64>(s, part[turn][0]);
                rho_b = 1.0f / sqrtf(fmaf(s, inv_n, a.eps));
            }
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float b[8], g[8], w[8];
                widen(r[k], v[k]);
                widen(br[k], b);
                if (a.w_post) {
                    widen(EARLY ? wp[k] : fetch(a.w_post, c[k], a.n), w);
#pragma unroll
                    for (int i = 0; i < 8; i++) b[i] = b[i] * rho_b * (a.w_offset + w[i]);
                }
                if (a.gate) {
                    gate_of<T>(a, EARLY ? gate[k] : fetch_gate<T>(a, row, c[k]), g);
#pragma unroll
                    for (int i = 0; i < 8; i++) g[i] = a.scale * (a.gate_sigmoid ? sigmoid(g[i]) : g[i]);
                }
                // rounded here: the norm that follows is the stored stream's, as whoever reads it
                // (the gradient, the next layer) sees it
#pragma unroll
                for (int i = 0; i < 8; i++) v[k][i] = (float)(R)fmaf(a.gate ? g[i] : a.scale, b[i], v[k][i]);
                if (c[k].lo < 8) put<NT>(static_cast<R *>(a.r_out) + base, c[k], a.n, v[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < NV; k++) widen(r[k], v[k]);
        }
        if (a.h) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                mask_cols(c[k], v[k]);
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(v[k][i], v[k][i], s);
            }
            s = group_sum<BS / 64>(s, part[turn][1]);
            rho_v = 1.0f / sqrtf(fmaf(s, inv_n, a.eps));
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float w[8];
                widen(EARLY ? wq[k] : fetch(a.w_pre, c[k], a.n), w);
#pragma unroll
                for (int i = 0; i < 8; i++) w[i] = v[k][i] * rho_v * (a.w_offset + w[i]);
                if (c[k].lo < 8) put<NT>(static_cast<T *>(a.h) + base, c[k], a.n, w);
            }
        }
        if (a.stats && threadIdx.x == 0) {
            a.stats[2 * row] = rho_b;
            a.stats[2 * row + 1] = rho_v;
        }
    }
}

// Values in registers as they lie in memory, so that their widened forms, twice the
// registers for 16-bit types, are formed again after a sum rather than kept over it.
template <typename T>
__device__ __forceinline__ void keep(Raw<T> &r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) asm volatile("" : "+v"(r.w[i]));
}

// A row's inputs of the backward pass.
template <typename T, typename R, int NV>
struct GradIn {
    Raw<R> v[NV], dr[NV];
    Raw<T> dh[NV], b[NV];
    Gate gate[NV];
    float rho_b, rho_v;
};

// Group blockIdx.x takes the rows blockIdx.x, + gridDim.x, ...: the sums over its
// rows stay in registers and go to its rows of the workspace, one per wanted
// parameter ([parameter][group][n]).  Where the registers hold them (AHEAD) the next
// row's inputs are fetched before this row's sums, whose two barriers would leave the
// memory idle, and the weights stay.  Rows longer than 8192 (WIDE) would need 250
// registers of the 128 that 1024 threads leave: two of the three sums lie in LDS, each
// column in its thread's own words, and inputs are read again where they are used
// (512 x 16384 in bf16: 48 us, 116 with all of it in registers, 215 to 360 of which
// spilled; 1 row 12.3, 41.7).  6 registers a lane still do.
template <typename T, typename R, int BS, int NV, bool NT>
__global__ __launch_bounds__(BS) void norm_grad_kernel(hoard_norm_args a, hoard_norm_grads g, float *work) {
    constexpr bool AHEAD = BS <= 512 && NV * (2 * sizeof(R) + 2 * sizeof(T)) <= 16;
    constexpr bool WIDE = NV * BS * 8 > 8192;
    __shared__ float part[2][3][BS / 64];
    __shared__ float lds[WIDE ? 2 : 1][WIDE ? NV * 8 : 1][WIDE ? BS : 1];
    const float inv_n = 1.0f / (float)a.n;
    float s_pre[NV][8] = {}, s_post[NV][8] = {}, s_gate[NV][8] = {};
    auto add_to = [&](int which, float (&s)[NV][8], int k, int i, float x, float y) {
        if constexpr (WIDE) lds[which][k * 8 + i][threadIdx.x] = fmaf(x, y, lds[which][k * 8 + i][threadIdx.x]);
        else s[k][i] = fmaf(x, y, s[k][i]);
    };
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < NV * 8; i++) lds[0][i][threadIdx.x] = lds[1][i][threadIdx.x] = 0.0f;
    }
    Cols c[NV];
    Raw<float> wp[NV], wq[NV];
    auto fetch_weights = [&]() {
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (a.w_post) wp[k] = fetch(a.w_post, c[k], a.n);
            if (g.dh) wq[k] = fetch(a.w_pre, c[k], a.n);
        }
    };
#pragma unroll
    for (int k = 0; k < NV; k++) c[k] = cols_of((k * BS + (int)threadIdx.x) * 8, a.n);
    const bool block = g.db || g.dgate || g.dw_post;
    auto fetch_row = [&](GradIn<T, R, NV> &in, size_t row) {
        const size_t base = row * a.n;
        in.rho_b = a.stats[2 * row];
        in.rho_v = a.stats[2 * row + 1];
        if constexpr (WIDE) return;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (g.dh) {
                in.v[k] = fetch(static_cast<const R *>(a.r_out) + base, c[k], a.n);
                in.dh[k] = fetch(static_cast<const T *>(g.dh) + base, c[k], a.n);
            }
            if (g.dr_out) in.dr[k] = fetch(static_cast<const R *>(g.dr_out) + base, c[k], a.n);
            if (block) {
                in.b[k] = fetch(static_cast<const T *>(a.b) + base, c[k], a.n);
                if (AHEAD && a.gate) in.gate[k] = fetch_gate<T>(a, row, c[k]);
            }
        }
    };
    int turn = 0;
    auto one = [&](GradIn<T, R, NV> &in, size_t row) {
        const size_t base = row * a.n;
        auto v_of = [&](int k) {
            if constexpr (WIDE) return fetch(static_cast<const R *>(a.r_out) + base, c[k], a.n);
            else return in.v[k];
        };
        auto dh_of = [&](int k) {
            if constexpr (WIDE) return fetch(static_cast<const T *>(g.dh) + base, c[k], a.n);
            else return in.dh[k];
        };
        auto b_of = [&](int k) {
            if constexpr (WIDE) return fetch(static_cast<const T *>(a.b) + base, c[k], a.n);
            else return in.b[k];
        };
        auto in_turn = [] {  // one k after another, for their registers
            if constexpr (WIDE) asm volatile("" ::: "memory");
        };
        float dv[NV][8];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            if (g.dr_out) {
                widen(WIDE ? fetch(static_cast<const R *>(g.dr_out) + base, c[k], a.n) : in.dr[k], dv[k]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) dv[k][i] = 0.0f;
            }
        }
        if (g.dh) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float w[8], v[8], u[8];
                in_turn();
                widen(v_of(k), v);
                widen(dh_of(k), u);
                widen(AHEAD ? wq[k] : fetch(a.w_pre, c[k], a.n), w);
                mask_cols(c[k], u);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    add_to(0, s_pre, k, i, u[i], v[i] * in.rho_v);
                    s = fmaf(u[i] * (a.w_offset + w[i]), v[i], s);
                }
            }
            s = group_sum<BS / 64>(s, part[turn][0]) * inv_n * in.rho_v * in.rho_v;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float w[8], v[8], u[8];
                in_turn();
                if constexpr (!WIDE) {
                    keep(in.v[k]);
                    keep(in.dh[k]);
                }
                widen(v_of(k), v);
                widen(dh_of(k), u);
                widen(AHEAD ? wq[k] : fetch(a.w_pre, c[k], a.n), w);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    dv[k][i] += in.rho_v * (u[i] * (a.w_offset + w[i]) - v[i] * s);
            }
        }
        if (g.dr) {
#pragma unroll
            for (int k = 0; k < NV; k++)
                if (c[k].lo < 8) put<NT>(static_cast<R *>(g.dr) + base, c[k], a.n, dv[k]);
        }
        if (!block) return;
        float s_b = 0.0f, s_g = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float q[8], w[8], dg[8], b[8];
            in_turn();
            widen(b_of(k), b);
            mask_cols(c[k], dv[k]);
            if (a.gate) gate_of<T>(a, AHEAD ? in.gate[k] : fetch_gate<T>(a, row, c[k]), q);
            if (a.w_post) widen(AHEAD ? wp[k] : fetch(a.w_post, c[k], a.n), w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float slope = 1.0f;
                const float t = !a.gate ? 1.0f : a.gate_sigmoid ? sigmoid_slope(q[i], slope) : q[i];
                const float wo = a.w_post ? a.w_offset + w[i] : 1.0f;
                const float d = a.scale * dv[k][i];   // of g c
                const float nb = b[i] * in.rho_b;  // rho_b is 1 without a norm
                dg[i] = d * nb * wo * slope;
                s_gate[k][i] += dg[i];
                s_g += dg[i];
                add_to(1, s_post, k, i, d * t, nb);
                dv[k][i] = d * t * wo;  // u2 from here on
                s_b = fmaf(dv[k][i], b[i], s_b);
            }
            if (a.gate_kind == HOARD_GATE_FULL && g.dgate && c[k].lo < 8)
                put<NT>(static_cast<T *>(g.dgate) + base, c[k], a.n, dg);
        }
        if (a.gate_kind == HOARD_GATE_TOKEN && g.dgate) {
            s_g = group_sum<BS / 64>(s_g, part[turn][2]);
            if (threadIdx.x == 0) static_cast<float *>(g.dgate)[row] = s_g;
        }
        if (!g.db) return;
        if (a.w_post) {
            s_b = group_sum<BS / 64>(s_b, part[turn][1]) * inv_n * in.rho_b * in.rho_b;
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float b[8];
                if constexpr (!WIDE) keep(in.b[k]);
                widen(b_of(k), b);
#pragma unroll
                for (int i = 0; i < 8; i++) dv[k][i] = in.rho_b * (dv[k][i] - b[i] * s_b);
            }
        }
#pragma unroll
        for (int k = 0; k < NV; k++)
            if (c[k].lo < 8) put<NT>(static_cast<T *>(g.db) + base, c[k], a.n, dv[k]);
    };
    if constexpr (AHEAD) {
        GradIn<T, R, NV> in[2];
        const size_t rows = a.n_rows, by = gridDim.x;
        fetch_weights();
        fetch_row(in[0], blockIdx.x);  // there are no more groups than rows
        for (size_t row = blockIdx.x; row < rows; row += 2 * by, turn = 0) {
            fetch_row(in[1], min(row + by, rows - 1));
            one(in[0], row);
            if (row + by >= rows) break;
            turn = 1;
            fetch_row(in[0], min(row + 2 * by, rows - 1));
            one(in[1], row + by);
        }
    } else {
        for (size_t row = blockIdx.x; row < (size_t)a.n_rows; row += gridDim.x, turn ^= 1) {
            GradIn<T, R, NV> in;
            fetch_row(in, row);
            one(in, row);
        }
    }
    // the group's rows of the workspace, or the result itself where it is the only row
    const size_t mine = (size_t)blockIdx.x * a.n, all = (size_t)gridDim.x * a.n;
    const bool alone = a.n_rows == 1;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        float *p = work + mine;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                s_pre[k][i] = lds[0][k * 8 + i][threadIdx.x];
                s_post[k][i] = lds[1][k * 8 + i][threadIdx.x];
            }
        }
        if (c[k].lo == 8) continue;
        if (g.dw_pre) {
            put(alone ? g.dw_pre : p, c[k], a.n, s_pre[k]);
            p += all;
        }
        if (g.dw_post) {
            put(alone ? g.dw_post : p, c[k], a.n, s_post[k]);
            p += all;
        }
        if (g.dgate && a.gate_kind == HOARD_GATE_CHANNEL)
            put(alone ? static_cast<float *>(g.dgate) : p, c[k], a.n, s_gate[k]);
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

// Rows that the L2s (8 of 4 MB) would not hold until they are read go past them: 4096
// rows of 4096, bf16 and a 32-bit stream, 43.7 us against 51.7; gradients of 4096 x 2048
// 26.7 against 30.5.
template <typename T>
bool past_caches(const hoard_norm_args &a) {
    return (int64_t)a.n_rows * a.n * sizeof(T) >= (8 << 20);
}

template <typename T, typename R, int BS, int NV>
void forward_of(const hoard_norm_args &a, hipStream_t s) {
    if (past_caches<T>(a)) norm_kernel<T, R, BS, NV, true><<<min(a.n_rows, 1 << 20), BS, 0, s>>>(a);
    else norm_kernel<T, R, BS, NV, false><<<min(a.n_rows, 1 << 20), BS, 0, s>>>(a);
}
template <typename T, typename R, int BS, int NV>
void grad_of(const hoard_norm_args &a, const hoard_norm_grads &g, float *work, hipStream_t s) {
    const int groups = norm_groups(a.n_rows, a.n);
    if (past_caches<T>(a)) norm_grad_kernel<T, R, BS, NV, true><<<groups, BS, 0, s>>>(a, g, work);
    else norm_grad_kernel<T, R, BS, NV, false><<<groups, BS, 0, s>>>(a, g, work);
}

// f(T, R, BS, NV) for the types and the row length: BS * 8 * NV >= n.
#define HOARD_NORM_SIZES(F, T, R, ...)                      \
    do {                                                    \
        if (a.n <= 512) F<T, R, 64, 1>(__VA_ARGS__);        \
        else if (a.n <= 1024) F<T, R, 64, 2>(__VA_ARGS__);  \
        else if (a.n <= 2048) F<T, R, 256, 1>(__VA_ARGS__); \
        else if (a.n <= 4096) F<T, R, 512, 1>(__VA_ARGS__); \
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

// As many groups as the chip holds at once (by their registers 3 of 256 threads a CU,
// 1 of more; of 64 threads as many as the partial sums are worth), with equal shares
// of the rows.  4096 x 2048, bf16: 29.4 us with at most 768 groups (683 of 6 rows), 33.0
// with 512, 37.7 with 1024; 4096 x 4096: 62.5 with 256, 64.3 with 512, 74.0 with 683.
int norm_groups(int n_rows, int n) {
    const int most = n <= 1024 ? 1024 : n <= 2048 ? 768 : 256;
    if (n_rows <= most) return n_rows;
    const int64_t share = ((int64_t)n_rows + most - 1) / most;
    return (int)((n_rows + share - 1) / share);
}

hipError_t launch_norm(const hoard_norm_args &a, hipStream_t s) {
    if (!a.n_rows) return hipSuccess;
    HOARD_NORM_TYPES(forward_of, a, s);
    return hipGetLastError();
}

hipError_t launch_norm_grad(const hoard_norm_args &a, const hoard_norm_grads &g, float *work, hipStream_t s) {
    SumOut o{};
    int params = 0;
    if (g.dw_pre) o.out[params++] = g.dw_pre;
    if (g.dw_post) o.out[params++] = g.dw_post;
    if (g.dgate && a.gate_kind == HOARD_GATE_CHANNEL) o.out[params++] = static_cast<float *>(g.dgate);
    if (a.n_rows) {
        HOARD_NORM_TYPES(grad_of, a, g, work, s);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    if (!params || a.n_rows == 1) return hipSuccess;  // one row's sums were written in place
    norm_sum_kernel<<<dim3((a.n + 63) / 64, params), 1024, 0, s>>>(work, norm_groups(a.n_rows, a.n), a.n, o);
    return hipGetLastError();
}

}  // namespace hoard

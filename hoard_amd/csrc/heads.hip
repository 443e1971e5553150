// Heads normed, rotated and written to a paged cache, and their gradients
// (hoard_heads_forward, hoard_heads_backward, hoard_kv_write, hoard_kv_read).
//
// Forward, per head row x of D values:  y = x rho (o + w),  rho = (mean x^2 + eps)^(-1/2),
// z = R y, R turning pair i by pos * freq_i.
// Backward, with dy = R^T dz and u = dy (o + w):
//   dx = rho (u - x rho^2 mean(u x)),   dw = sum over tokens and heads of dy x rho.
//
// Both are bound by memory: a head is read once into registers, its sum formed across its
// lanes and the result written from there.  A head takes LANES lanes (a power of two) of
// eight values: two runs of four that turn with each other, so no value crosses lanes.
// The angles of a token are formed once for all of its heads that a wave takes.
#include "attn.h"
#include "opsdev.h"

namespace hoard {

namespace {

// Four values as they lie in memory, at any alignment of their type.
typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T>
struct Four {
    uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Four<T> fetch4(const T *p) {
    Four<T> r;
    if constexpr (sizeof(T) == 4) {
        const words4 v = *reinterpret_cast<const words4 *>(p);
        __builtin_memcpy(&r, &v, sizeof r);
    } else {
        const words2 v = *reinterpret_cast<const words2 *>(p);
        __builtin_memcpy(&r, &v, sizeof r);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void widen4(const Four<T> &r, float o[4]) {
    T v[4];
    __builtin_memcpy(v, &r, sizeof v);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = (float)v[i];
}
// Rounded to nearest, ties to even, once.
template <typename T>
__device__ __forceinline__ void put4(T *p, const float o[4]) {
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (T)o[i];
    if constexpr (sizeof(T) == 4) {
        words4 w;
        __builtin_memcpy(&w, v, sizeof w);
        *reinterpret_cast<words4 *>(p) = w;
    } else {
        words2 w;
        __builtin_memcpy(&w, v, sizeof w);
        *reinterpret_cast<words2 *>(p) = w;
    }
}

// Sum and maximum over each aligned group of LANES lanes, in all of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    if (LANES >= 2) v += dpp_f<kDppQuadXor1>(v);
    if (LANES >= 4) v += dpp_f<kDppQuadXor2>(v);
    if (LANES >= 8) v += dpp_f<kDppRowHalfMirror>(v);
    if (LANES >= 16) v += dpp_f<kDppRowMirror>(v);
    if (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ int lanes_max(int v) {
    if (LANES >= 2) v = max(v, dpp_i<kDppQuadXor1>(v));
    if (LANES >= 4) v = max(v, dpp_i<kDppQuadXor2>(v));
    if (LANES >= 8) v = max(v, dpp_i<kDppRowHalfMirror>(v));
    if (LANES >= 16) v = max(v, dpp_i<kDppRowMirror>(v));
    if (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((int)r[0], (int)r[1]);
    }
    return v;
}

// A lane's place in its head: the first values of its two runs of four.
struct Place {
    int li, a, b;
    bool on, turned;
};
template <int LANES>
__device__ __forceinline__ Place place_of(const hoard_heads_args &h) {
    Place p;
    p.li = (int)threadIdx.x & (LANES - 1);
    p.on = p.li * 8 < h.head_dim;
    const int li = p.on ? p.li : 0;
    p.turned = li * 8 < h.rot_dim;
    const bool halves = h.rope == HOARD_ROPE_HALVES && p.turned;
    p.a = halves ? 4 * li : 8 * li;
    p.b = halves ? h.rot_dim / 2 + 4 * li : 8 * li + 4;
    return p;
}

// Cosines and sines of the lane's four pairs.  A position times a frequency is taken in 64
// bits to its fraction of a turn, so far positions keep their digits.
struct Turn {
    float c[4], s[4];
};
__device__ __forceinline__ Turn turn_of(const hoard_heads_args &a, const Place &p, int64_t token) {
    Turn t;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        t.c[j] = 1.0f;
        t.s[j] = 0.0f;
    }
    if (!p.turned) return t;
    const int first = p.on ? 4 * p.li : 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int axis = a.axis ? min((int)a.axis[first + j], a.n_axes - 1) : 0;
        const double turns = (double)a.pos[(int64_t)axis * a.n_tokens + token] * a.freq[first + j] * 0.15915494309189535;
        sincospif(2.0f * (float)(turns - rint(turns)), &t.s[j], &t.c[j]);
    }
    return t;
}
// The lane's values v[0..3] (run a) and v[4..7] (run b) turned, by the negative angle with `back`.
__device__ __forceinline__ void rotate(int rope, const Place &p, const Turn &t, bool back, float v[8]) {
    if (!p.turned) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float s = back ? -t.s[j] : t.s[j];
        float &x = rope == HOARD_ROPE_HALVES ? v[j] : v[2 * j], &y = rope == HOARD_ROPE_HALVES ? v[4 + j] : v[2 * j + 1];
        const float nx = x * t.c[j] - y * s, ny = y * t.c[j] + x * s;
        x = nx;
        y = ny;
    }
}

// The weights of the lane's values, the offset added; ones without weights.
__device__ __forceinline__ void weights_of(const float *w, float offset, const Place &p, float o[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        o[i] = w ? offset + w[p.a + i] : 1.0f;
        o[4 + i] = w ? offset + w[p.b + i] : 1.0f;
    }
}

struct NoCache {};

// A head's values to its row of the cache.  8 bits: the largest magnitude as an integer, so
// that a NaN (and an infinity) is larger than every number.
template <typename C, int LANES>
__device__ __forceinline__ void put_row(C *rows, float *scales, int64_t row, int dim, const Place &p, const float v[8]) {
    if constexpr (sizeof(C) == 2) {
        if (p.on) {
            put4(rows + row * dim + p.a, v);
            put4(rows + row * dim + p.b, v + 4);
        }
    } else {
        int most = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) most = max(most, __float_as_int(v[i]) & 0x7fffffff);
        most = lanes_max<LANES>(p.on ? most : 0);
        const float step = most < 0x7f800000 ? __int_as_float(most) / 127.0f : __int_as_float(0x7fc00000);
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float code = step > 0.0f ? fminf(fmaxf(rintf(v[i] / step), -127.0f), 127.0f) : 0.0f;
            w[i / 4] |= (uint32_t)((int)code & 0xff) << (8 * (i & 3));
        }
        if (p.on) {
            int8_t *to = reinterpret_cast<int8_t *>(rows) + row * dim;
            *reinterpret_cast<uint32_t *>(to + p.a) = w[0];
            *reinterpret_cast<uint32_t *>(to + p.b) = w[1];
            if (p.li == 0) scales[row] = step;
        }
    }
}

// How the heads of the tokens are dealt to waves: a wave takes HEADS = 64 / LANES heads at a
// time and `per` such passes of a token, a token takes `chunks` waves.
struct Deal {
    int per, chunks;
    int64_t items;  // waves' worth of work
};

// Passes that a wave has in flight at once.
constexpr int kAhead = 2;

template <typename T, typename C, int LANES>
__global__ __launch_bounds__(256) void heads_kernel(hoard_heads_args a, hoard_kv_cache c, Deal d) {
    constexpr int HEADS = 64 / LANES;
    constexpr bool CACHE = !__is_same(C, NoCache);
    const Place p = place_of<LANES>(a);
    const int hi = (threadIdx.x & 63) / LANES, dim = a.head_dim;
    const int nq = a.q ? a.n_q_heads : 0, nk = a.k ? a.n_kv_heads : 0, nv = a.v ? a.n_kv_heads : 0;
    const int heads = nq + nk + nv, passes = (heads + HEADS - 1) / HEADS;
    const float inv_n = 1.0f / (float)dim;
    float wq[8], wk[8];
    weights_of(a.w_q, a.w_offset, p, wq);
    weights_of(a.w_k, a.w_offset, p, wk);
    for (int64_t item = (int64_t)blockIdx.x * 4 + wave_index(); item < d.items; item += (int64_t)gridDim.x * 4) {
        const int64_t token = item / d.chunks;
        const int first = (int)(item - token * d.chunks) * d.per, last = min(passes, first + d.per);
        const Turn turn = turn_of(a, p, token);
        int64_t slot = -1;
        if constexpr (CACHE) {
            slot = a.slots[token];
            if (slot >= (int64_t)c.n_pages * c.page) slot = -1;
        }
        for (int at = first; at < last; at += kAhead) {
            Four<T> raw[kAhead][2];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int h = min((at + u) * HEADS + hi, heads - 1);
                const T *row = h < nq        ? static_cast<const T *>(a.q) + token * a.q_stride + h * dim
                               : h < nq + nk ? static_cast<const T *>(a.k) + token * a.k_stride + (h - nq) * dim
                                             : static_cast<const T *>(a.v) + token * a.v_stride + (h - nq - nk) * dim;
                raw[u][0] = fetch4(row + p.a);
                raw[u][1] = fetch4(row + p.b);
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (at + u >= last) break;
                const int h = (at + u) * HEADS + hi;
                const bool on = p.on && h < heads, is_q = h < nq, is_k = !is_q && h < nq + nk;
                float v[8];
                widen4(raw[u][0], v);
                widen4(raw[u][1], v + 4);
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) s = fmaf(v[i], v[i], s);
                s = lanes_sum<LANES>(p.on ? s : 0.0f);
                const bool normed = is_q ? a.w_q != nullptr : is_k && a.w_k != nullptr;
                const float rho = normed ? 1.0f / sqrtf(fmaf(s, inv_n, a.eps)) : 1.0f;
                if (normed) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = v[i] * rho * (is_q ? wq[i] : wk[i]);
                }
                if (is_q || is_k) rotate(a.rope, p, turn, false, v);
                if (on && is_q) {
                    T *to = static_cast<T *>(a.q_out) + token * a.q_out_stride + h * dim;
                    put4(to + p.a, v);
                    put4(to + p.b, v + 4);
                }
                if (on && is_k && a.k_out) {
                    T *to = static_cast<T *>(a.k_out) + token * a.k_out_stride + (h - nq) * dim;
                    put4(to + p.a, v);
                    put4(to + p.b, v + 4);
                }
                if (on && a.stats && p.li == 0 && (is_q || is_k))
                    a.stats[token * (a.n_q_heads + a.n_kv_heads) + (is_q ? h : a.n_q_heads + h - nq)] = rho;
                if constexpr (CACHE) {
                    if (slot >= 0) {
                        const int head = is_k ? h - nq : h - nq - nk;
                        const int64_t row = (slot / c.page * c.n_kv_heads + head) * c.page + slot % c.page;
                        Place to = p;
                        to.on = on && !is_q;
                        put_row<C, LANES>(static_cast<C *>(is_k ? c.k : c.v), is_k ? c.k_scale : c.v_scale, row, dim, to, v);
                    }
                }
            }
        }
    }
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void heads_grad_kernel(hoard_heads_args a, hoard_heads_grads g, float *work, Deal d) {
    constexpr int HEADS = 64 / LANES;
    __shared__ float part[4][2][256];
    const Place p = place_of<LANES>(a);
    const int lane = threadIdx.x & 63, hi = lane / LANES, dim = a.head_dim;
    const int nq = g.dq || g.dw_q ? a.n_q_heads : 0, nk = g.dk || g.dw_k ? a.n_kv_heads : 0;
    const int heads = nq + nk, passes = (heads + HEADS - 1) / HEADS;
    const float inv_n = 1.0f / (float)dim;
    float wq[8], wk[8], sum_q[8] = {}, sum_k[8] = {};
    weights_of(a.w_q, a.w_offset, p, wq);
    weights_of(a.w_k, a.w_offset, p, wk);
    for (int64_t item = (int64_t)blockIdx.x * 4 + wave_index(); item < d.items; item += (int64_t)gridDim.x * 4) {
        const int64_t token = item / d.chunks;
        const int first = (int)(item - token * d.chunks) * d.per, last = min(passes, first + d.per);
        const Turn turn = turn_of(a, p, token);
        for (int at = first; at < last; at += kAhead) {
            Four<T> dz[kAhead][2], x[kAhead][2];
            float rho[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int h = min((at + u) * HEADS + hi, heads - 1);
                const bool is_q = h < nq;
                const T *from = is_q ? static_cast<const T *>(g.dq_out) + token * a.q_out_stride + h * dim
                                     : static_cast<const T *>(g.dk_out) + token * a.k_out_stride + (h - nq) * dim;
                dz[u][0] = fetch4(from + p.a);
                dz[u][1] = fetch4(from + p.b);
                rho[u] = 1.0f;
                if (is_q ? a.w_q != nullptr : a.w_k != nullptr) {
                    from = is_q ? static_cast<const T *>(a.q) + token * a.q_stride + h * dim
                                : static_cast<const T *>(a.k) + token * a.k_stride + (h - nq) * dim;
                    x[u][0] = fetch4(from + p.a);
                    x[u][1] = fetch4(from + p.b);
                    rho[u] = a.stats[token * (a.n_q_heads + a.n_kv_heads) + (is_q ? h : a.n_q_heads + h - nq)];
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                if (at + u >= last) break;
                const int h = (at + u) * HEADS + hi;
                const bool on = p.on && h < heads, is_q = h < nq;
                float v[8], xv[8] = {};
                widen4(dz[u][0], v);
                widen4(dz[u][1], v + 4);
                rotate(a.rope, p, turn, true, v);
                const bool normed = is_q ? a.w_q != nullptr : a.w_k != nullptr;
                if (normed) {
                    widen4(x[u][0], xv);
                    widen4(x[u][1], xv + 4);
                }
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (normed && on) {
                        const float t = v[i] * (xv[i] * rho[u]);
                        sum_q[i] += is_q ? t : 0.0f;
                        sum_k[i] += is_q ? 0.0f : t;
                    }
                    v[i] *= is_q ? wq[i] : wk[i];
                    s = fmaf(v[i], xv[i], s);
                }
                s = lanes_sum<LANES>(p.on ? s : 0.0f) * inv_n * rho[u] * rho[u];
                if (normed) {
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = rho[u] * (v[i] - xv[i] * s);
                }
                T *to = is_q ? static_cast<T *>(g.dq) : static_cast<T *>(g.dk);
                if (on && to) {
                    to += is_q ? token * g.dq_stride + h * dim : token * g.dk_stride + (h - nq) * dim;
                    put4(to + p.a, v);
                    put4(to + p.b, v + 4);
                }
            }
        }
    }
    if (!g.dw_q && !g.dw_k) return;
    // the wave's heads, then the workgroup's waves, in a fixed order
#pragma unroll
    for (int i = 0; i < 8; i++) {
#pragma unroll
        for (int off = LANES; off < 64; off *= 2) {
            sum_q[i] += __shfl_xor(sum_q[i], off);
            sum_k[i] += __shfl_xor(sum_k[i], off);
        }
    }
    if (lane < LANES && p.on) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int col = i < 4 ? p.a + i : p.b + i - 4;
            part[wave_index()][0][col] = sum_q[i];
            part[wave_index()][1][col] = sum_k[i];
        }
    }
    __syncthreads();
    const int col = threadIdx.x;
    if (col >= dim) return;
    const bool alone = gridDim.x == 1;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        float *out = w ? g.dw_k : g.dw_q;
        if (!out) continue;
        const float s = (part[0][w][col] + part[1][w][col]) + (part[2][w][col] + part[3][w][col]);
        if (alone) out[col] = s;
        else work[((size_t)w * gridDim.x + blockIdx.x) * dim + col] = s;
    }
}

// The groups' partial sums [q, k][groups][dim] added, as the norms' are: a workgroup takes
// 64 columns, its 16 waves a sixteenth of the groups each, in ascending order.
__global__ __launch_bounds__(1024) void heads_sum_kernel(const float *work, int groups, int dim, float *dw_q, float *dw_k) {
    __shared__ float part[16][64];
    float *out = blockIdx.y ? dw_k : dw_q;
    if (!out) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    const int per = (groups + 15) / 16, g0 = wave * per, g1 = min(groups, g0 + per);
    float s = 0.0f;
    if (col < dim) {
        const float *p = work + (size_t)blockIdx.y * groups * dim + col;
#pragma unroll 8
        for (int g = g0; g < g1; g++) s += p[(size_t)g * dim];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) s += part[i][lane];
    if (col < dim) out[col] = s;
}

template <typename T, typename C, int LANES>
__global__ __launch_bounds__(256) void kv_read_kernel(KvReadArgs a, Deal d) {
    constexpr int HEADS = 64 / LANES;
    const int li = threadIdx.x & (LANES - 1), hi = (threadIdx.x & 63) / LANES, dim = a.c.head_dim;
    const int nk = a.k ? a.c.n_kv_heads : 0, heads = nk + (a.v ? a.c.n_kv_heads : 0), passes = (heads + HEADS - 1) / HEADS;
    for (int64_t item = (int64_t)blockIdx.x * 4 + wave_index(); item < d.items; item += (int64_t)gridDim.x * 4) {
        const int64_t token = item / d.chunks, slot = a.slots[token];
        if (slot < 0 || slot >= (int64_t)a.c.n_pages * a.c.page) continue;
        const int first = (int)(item - token * d.chunks) * d.per, last = min(passes, first + d.per);
        for (int at = first; at < last; at++) {
            const int h = at * HEADS + hi;
            if (h >= heads || li * 8 >= dim) continue;
            const bool is_k = h < nk;
            const int head = is_k ? h : h - nk;
            const int64_t row = (slot / a.c.page * a.c.n_kv_heads + head) * a.c.page + slot % a.c.page;
            const C *from = static_cast<const C *>(is_k ? a.c.k : a.c.v) + row * dim + 8 * li;
            T *to = is_k ? static_cast<T *>(a.k) + token * a.k_stride : static_cast<T *>(a.v) + token * a.v_stride;
            to += head * dim + 8 * li;
            float v[8];
            if constexpr (sizeof(C) == 1) {
                const float step = (is_k ? a.c.k_scale : a.c.v_scale)[row];
                const words2 w = *reinterpret_cast<const words2 *>(from);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = step * (float)(int8_t)(w[i / 4] >> (8 * (i & 3)));
            } else {
                widen4(fetch4(from), v);
                widen4(fetch4(from + 4), v + 4);
            }
            put4(to, v);
            put4(to + 4, v + 4);
        }
    }
}

int lanes_of(int dim) {
    int lanes = 1;
    while (lanes * 8 < dim) lanes *= 2;
    return lanes;
}

// Few tokens: a pass a wave, for the latency of one.  Many: a token's passes together, for
// its angles are formed once a wave; at 4096 waves and more the chip is full.
Deal deal(int64_t tokens, int heads, int lanes) {
    const int passes = (heads * lanes + 63) / 64;
    Deal d;
    d.per = (int)(tokens * passes / 4096);
    d.per = d.per < 1 ? 1 : d.per > passes ? passes : d.per;
    d.chunks = (passes + d.per - 1) / d.per;
    d.items = tokens * d.chunks;
    return d;
}
int blocks_of(const Deal &d) { return (int)(d.items + 3 < (int64_t)4 << 20 ? (d.items + 3) / 4 : 1 << 20); }

// f<.., LANES>(...) for the head's length.
#define HOARD_LANES(DIM, CALL)              \
    switch (lanes_of(DIM)) {                \
        case 1: { CALL(1); } break;         \
        case 2: { CALL(2); } break;         \
        case 4: { CALL(4); } break;         \
        case 8: { CALL(8); } break;         \
        case 16: { CALL(16); } break;       \
        default: { CALL(32); } break;       \
    }

template <typename T, typename C>
void forward_of(const hoard_heads_args &a, const Deal &d, hipStream_t s) {
    const hoard_kv_cache c = a.cache ? *a.cache : hoard_kv_cache{};
#define HOARD_CALL(L) heads_kernel<T, C, L><<<blocks_of(d), 256, 0, s>>>(a, c, d)
    HOARD_LANES(a.head_dim, HOARD_CALL)
#undef HOARD_CALL
}
template <typename T>
void forward_type(const hoard_heads_args &a, const Deal &d, hipStream_t s) {
    if (!a.cache) forward_of<T, NoCache>(a, d, s);
    else if (a.cache->type == HOARD_TYPE_F16) forward_of<T, f16>(a, d, s);
    else if (a.cache->type == HOARD_TYPE_BF16) forward_of<T, bf16>(a, d, s);
    else forward_of<T, int8_t>(a, d, s);
}
template <typename T>
void grad_type(const hoard_heads_args &a, const hoard_heads_grads &g, float *work, int groups, const Deal &d, hipStream_t s) {
#define HOARD_CALL(L) heads_grad_kernel<T, L><<<groups, 256, 0, s>>>(a, g, work, d)
    HOARD_LANES(a.head_dim, HOARD_CALL)
#undef HOARD_CALL
}
template <typename T, typename C>
void read_of(const KvReadArgs &a, const Deal &d, hipStream_t s) {
#define HOARD_CALL(L) kv_read_kernel<T, C, L><<<blocks_of(d), 256, 0, s>>>(a, d)
    HOARD_LANES(a.c.head_dim, HOARD_CALL)
#undef HOARD_CALL
}
template <typename T>
void read_type(const KvReadArgs &a, const Deal &d, hipStream_t s) {
    if (a.c.type == HOARD_TYPE_F16) read_of<T, f16>(a, d, s);
    else if (a.c.type == HOARD_TYPE_BF16) read_of<T, bf16>(a, d, s);
    else read_of<T, int8_t>(a, d, s);
}

}  // namespace

int heads_groups(const hoard_heads_args &a) {
    const Deal d = deal(a.n_tokens, a.n_q_heads + a.n_kv_heads, lanes_of(a.head_dim));
    return (int)(d.items < 4 * 1024 ? (d.items + 3) / 4 : 1024);
}

hipError_t launch_heads(const hoard_heads_args &a, hipStream_t s) {
    const int heads = (a.q ? a.n_q_heads : 0) + (a.k ? a.n_kv_heads : 0) + (a.v ? a.n_kv_heads : 0);
    if (!heads) return hipSuccess;
    const Deal d = deal(a.n_tokens, heads, lanes_of(a.head_dim));
    if (a.type == HOARD_TYPE_F32) forward_type<float>(a, d, s);
    else if (a.type == HOARD_TYPE_F16) forward_type<f16>(a, d, s);
    else forward_type<bf16>(a, d, s);
    return hipGetLastError();
}

hipError_t launch_heads_grad(const hoard_heads_args &a, const hoard_heads_grads &g, float *work, hipStream_t s) {
    const int groups = heads_groups(a);
    const int heads = (g.dq || g.dw_q ? a.n_q_heads : 0) + (g.dk || g.dw_k ? a.n_kv_heads : 0);
    if (groups) {
        const Deal d = deal(a.n_tokens, heads, lanes_of(a.head_dim));
        if (a.type == HOARD_TYPE_F32) grad_type<float>(a, g, work, groups, d, s);
        else if (a.type == HOARD_TYPE_F16) grad_type<f16>(a, g, work, groups, d, s);
        else grad_type<bf16>(a, g, work, groups, d, s);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    if ((!g.dw_q && !g.dw_k) || groups == 1) return hipSuccess;  // one group's sums were written in place
    heads_sum_kernel<<<dim3((a.head_dim + 63) / 64, 2), 1024, 0, s>>>(work, groups, a.head_dim, g.dw_q, g.dw_k);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvReadArgs &a, hipStream_t s) {
    const int heads = (a.k ? a.c.n_kv_heads : 0) + (a.v ? a.c.n_kv_heads : 0);
    const Deal d = deal(a.n_tokens, heads, lanes_of(a.c.head_dim));
    if (a.type == HOARD_TYPE_F32) read_type<float>(a, d, s);
    else if (a.type == HOARD_TYPE_F16) read_type<f16>(a, d, s);
    else read_type<bf16>(a, d, s);
    return hipGetLastError();
}

}  // namespace hoard

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
#include <type_traits>

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
// NT: with the non-temporal policy, for what is read or written once and would only push
// other data out of the caches.
template <bool NT = false, typename T>
__device__ __forceinline__ Four<T> fetch4(const T *p) {
    typedef std::conditional_t<sizeof(T) == 4, words4, words2> words;
    const words *from = reinterpret_cast<const words *>(p);
    const words v = NT ? __builtin_nontemporal_load(from) : *from;
    Four<T> r;
    __builtin_memcpy(&r, &v, sizeof r);
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
template <bool NT = false, typename T>
__device__ __forceinline__ void put4(T *p, const float o[4]) {
    typedef std::conditional_t<sizeof(T) == 4, words4, words2> words;
    T v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = (T)o[i];
    words w, *to = reinterpret_cast<words *>(p);
    __builtin_memcpy(&w, v, sizeof w);
    if (NT) __builtin_nontemporal_store(w, to);
    else *to = w;
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

// sin and cos of x + q pi / 2, |x| <= pi / 4: their series up to x^9 and x^10, which leave 2e-9 and
// 5e-10.
__device__ __forceinline__ void sincos_quarter(float x, int q, float &s, float &c) {
    const float y = x * x;
    const float sx = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float cx = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const float a = q & 1 ? cx : sx, b = q & 1 ? sx : cx;
    s = q & 2 ? -a : a;
    c = (q + 1) & 2 ? -b : b;
}

// Cosines and sines of the lane's four pairs.  A position times a frequency is taken in 64
// bits to what is left of the nearest quarter turn, so far positions keep their digits and the
// angle rounds to 32 bits when it is small (errors of 1.2 roundings of 1 at most; 2.4 where the
// fraction of a whole turn is rounded).
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
        const double quarters = (double)a.pos[(int64_t)axis * a.n_tokens + token] * a.freq[first + j] * 0.63661977236758134;
        const double whole = rint(quarters);
        // its last two bits, as those of a double between 2^52 and 2^53 (quarters past 2^51 have no
        // digits to say which of four they are)
        const int q = __double2loint(whole + 0x1.8p52);
        sincos_quarter((float)((quarters - whole) * 1.5707963267948966), q, t.s[j], t.c[j]);
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
        const float nx = fmaf(x, t.c[j], -(y * s)), ny = fmaf(y, t.c[j], x * s);
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
// The cache's row of a head at a slot; pages are powers of two.
__device__ __forceinline__ int64_t cache_row(const hoard_kv_cache &c, int slot, int head) {
    return ((int64_t)(slot >> (31 - __builtin_clz(c.page))) * c.n_kv_heads + head) * c.page + (slot & (c.page - 1));
}

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
// time and `per` such passes of a token, a token takes `chunks` waves (blockIdx.y).
struct Deal {
    int per, chunks;
};

// A wave has the next pass in flight while it forms one (two or four at a time are no faster:
// 4096 tokens by 36 heads of 128 in bf16 18.9, 20.5, 20.4 us).
template <typename T, typename C, int LANES, bool NT>
__global__ __launch_bounds__(256) void heads_kernel(hoard_heads_args a, hoard_kv_cache c, Deal d) {
    constexpr int HEADS = 64 / LANES;
    constexpr bool CACHE = !__is_same(C, NoCache);
    const Place p = place_of<LANES>(a);
    const int hi = (threadIdx.x & 63) / LANES, dim = a.head_dim;
    const int nq = a.q ? a.n_q_heads : 0, nk = a.k ? a.n_kv_heads : 0, nv = a.v ? a.n_kv_heads : 0;
    const int heads = nq + nk + nv, passes = (heads + HEADS - 1) / HEADS;
    const float inv_n = 1.0f / (float)dim;
    const int first = blockIdx.y * d.per, last = min(passes, first + d.per);
    Four<T> raw[2];
    auto fetch_pass = [&](int64_t token, int at) {
        const int h = min(at * HEADS + hi, heads - 1);
        const T *row = h < nq        ? static_cast<const T *>(a.q) + token * a.q_stride + h * dim
                       : h < nq + nk ? static_cast<const T *>(a.k) + token * a.k_stride + (h - nq) * dim
                                     : static_cast<const T *>(a.v) + token * a.v_stride + (h - nq - nk) * dim;
        raw[0] = fetch4<NT>(row + p.a);
        raw[1] = fetch4<NT>(row + p.b);
    };
    const int64_t stride = (int64_t)gridDim.x * 4;
    int64_t token = (int64_t)blockIdx.x * 4 + wave_index();
    if (token >= a.n_tokens) return;
    // asked for before the angles and the weights, whose latencies it shares
    fetch_pass(token, first);
    float wq[8], wk[8];
    weights_of(a.w_q, a.w_offset, p, wq);
    weights_of(a.w_k, a.w_offset, p, wk);
    for (; token < a.n_tokens; token += stride) {
        const Turn turn = turn_of(a, p, token);
        int slot = -1;
        if constexpr (CACHE) {
            slot = a.slots[token];
            if (slot >= c.n_pages * c.page) slot = -1;
        }
        for (int at = first; at < last; at++) {
            float v[8];
            widen4(raw[0], v);
            widen4(raw[1], v + 4);
            if (at + 1 < last) fetch_pass(token, at + 1);
            else if (token + stride < a.n_tokens) fetch_pass(token + stride, first);
            const int h = at * HEADS + hi;
            const bool on = p.on && h < heads, is_q = h < nq, is_k = !is_q && h < nq + nk;
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
            T *to = is_q ? static_cast<T *>(a.q_out) : is_k ? static_cast<T *>(a.k_out) : nullptr;
            if (on && to) {
                to += is_q ? token * a.q_out_stride + h * dim : token * a.k_out_stride + (h - nq) * dim;
                put4<NT>(to + p.a, v);
                put4<NT>(to + p.b, v + 4);
            }
            if (on && a.stats && p.li == 0 && (is_q || is_k))
                a.stats[token * (a.n_q_heads + a.n_kv_heads) + (is_q ? h : a.n_q_heads + h - nq)] = rho;
            if constexpr (CACHE) {
                if (slot >= 0) {
                    Place of = p;
                    of.on = on && !is_q;
                    put_row<C, LANES>(static_cast<C *>(is_k ? c.k : c.v), is_k ? c.k_scale : c.v_scale,
                                      cache_row(c, slot, is_k ? h - nq : h - nq - nk), dim, of, v);
                }
            }
        }
    }
}

template <typename T, int LANES, bool NT>
__global__ __launch_bounds__(256) void heads_grad_kernel(hoard_heads_args a, hoard_heads_grads g, float *work, Deal d) {
    constexpr int HEADS = 64 / LANES;
    __shared__ float part[4][2][256];
    const Place p = place_of<LANES>(a);
    const int lane = threadIdx.x & 63, hi = lane / LANES, dim = a.head_dim;
    const int nq = g.dq || g.dw_q ? a.n_q_heads : 0, nk = g.dk || g.dw_k ? a.n_kv_heads : 0;
    const int heads = nq + nk, passes = (heads + HEADS - 1) / HEADS;
    const float inv_n = 1.0f / (float)dim;
    float sum_q[8] = {}, sum_k[8] = {};
    const int first = blockIdx.y * d.per, last = min(passes, first + d.per);
    Four<T> dz[2], x[2];
    float next_rho = 1.0f;
    auto fetch_pass = [&](int64_t token, int at) {
        const int h = min(at * HEADS + hi, heads - 1);
        const bool is_q = h < nq;
        const T *from = is_q ? static_cast<const T *>(g.dq_out) + token * a.q_out_stride + h * dim
                             : static_cast<const T *>(g.dk_out) + token * a.k_out_stride + (h - nq) * dim;
        dz[0] = fetch4<NT>(from + p.a);
        dz[1] = fetch4<NT>(from + p.b);
        if (is_q ? a.w_q != nullptr : a.w_k != nullptr) {
            from = is_q ? static_cast<const T *>(a.q) + token * a.q_stride + h * dim
                        : static_cast<const T *>(a.k) + token * a.k_stride + (h - nq) * dim;
            x[0] = fetch4<NT>(from + p.a);
            x[1] = fetch4<NT>(from + p.b);
            next_rho = a.stats[token * (a.n_q_heads + a.n_kv_heads) + (is_q ? h : a.n_q_heads + h - nq)];
        }
    };
    const int64_t stride = (int64_t)gridDim.x * 4, tokens = first < last ? a.n_tokens : 0;
    int64_t token = (int64_t)blockIdx.x * 4 + wave_index();
    if (token < tokens) fetch_pass(token, first);
    float wq[8], wk[8];
    weights_of(a.w_q, a.w_offset, p, wq);
    weights_of(a.w_k, a.w_offset, p, wk);
    for (; token < tokens; token += stride) {
        const Turn turn = turn_of(a, p, token);
        for (int at = first; at < last; at++) {
            const int h = at * HEADS + hi;
            const bool on = p.on && h < heads, is_q = h < nq, normed = is_q ? a.w_q != nullptr : a.w_k != nullptr;
            float v[8], xv[8] = {};
            widen4(dz[0], v);
            widen4(dz[1], v + 4);
            if (normed) {
                widen4(x[0], xv);
                widen4(x[1], xv + 4);
            }
            const float rho = normed ? next_rho : 1.0f;
            if (at + 1 < last) fetch_pass(token, at + 1);
            else if (token + stride < tokens) fetch_pass(token + stride, first);
            rotate(a.rope, p, turn, true, v);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (normed && on) {
                    const float t = v[i] * (xv[i] * rho);
                    sum_q[i] += is_q ? t : 0.0f;
                    sum_k[i] += is_q ? 0.0f : t;
                }
                v[i] *= is_q ? wq[i] : wk[i];
                s = fmaf(v[i], xv[i], s);
            }
            s = lanes_sum<LANES>(p.on ? s : 0.0f) * inv_n * rho * rho;
            if (normed) {
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = rho * (v[i] - xv[i] * s);
            }
            T *to = is_q ? static_cast<T *>(g.dq) : static_cast<T *>(g.dk);
            if (on && to) {
                to += is_q ? token * g.dq_stride + h * dim : token * g.dk_stride + (h - nq) * dim;
                put4<NT>(to + p.a, v);
                put4<NT>(to + p.b, v + 4);
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
    const int groups = gridDim.x * gridDim.y, group = blockIdx.y * gridDim.x + blockIdx.x;
    const bool alone = groups == 1;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        float *out = w ? g.dw_k : g.dw_q;
        if (!out) continue;
        const float s = (part[0][w][col] + part[1][w][col]) + (part[2][w][col] + part[3][w][col]);
        if (alone) out[col] = s;
        else work[((size_t)w * groups + group) * dim + col] = s;
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
    const int first = blockIdx.y * d.per, last = min(passes, first + d.per);
    for (int64_t token = (int64_t)blockIdx.x * 4 + wave_index(); token < a.n_tokens; token += (int64_t)gridDim.x * 4) {
        const int slot = a.slots[token];
        if (slot < 0 || slot >= a.c.n_pages * a.c.page) continue;
        for (int at = first; at < last; at++) {
            const int h = at * HEADS + hi;
            if (h >= heads || li * 8 >= dim) continue;
            const bool is_k = h < nk;
            const int head = is_k ? h : h - nk;
            const int64_t row = cache_row(a.c, slot, head);
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

// Waves that tokens are dealt to before each takes more than a pass: about the chip's waves, as
// one lives some 5 us whatever it has to do (1000 tokens in 8 bits 14.3 us, 16.3 with 4096, 22
// with 8192).
constexpr int kWaves = 2048, kGroups = 1024, kBlocks = 1536;

int lanes_of(int dim) {
    int lanes = 4;
    while (lanes * 8 < dim) lanes *= 2;
    return lanes;
}

// Few tokens: a pass a wave, for the latency of one.  Many: a token's passes together, for
// its angles are formed once a wave.
Deal deal(int64_t tokens, int heads, int lanes) {
    const int passes = (heads * lanes + 63) / 64;
    Deal d;
    d.per = (int)(tokens * passes / kWaves);
    d.per = d.per < 1 ? 1 : d.per > passes ? passes : d.per;
    d.chunks = (passes + d.per - 1) / d.per;
    return d;
}
// Past the caches from where these no longer hold them until they are read: gradients of 8192
// tokens by 36 heads of 128 in bf16 (75 MB) 56.3 us against 60.6; 4096 tokens forward (38 MB) 18.9
// through them, 20.4 past.
bool past_caches(const hoard_heads_args &a) {
    return (int64_t)a.n_tokens * (a.n_q_heads + a.n_kv_heads) * a.head_dim * (a.type == HOARD_TYPE_F32 ? 4 : 2) >= 64 << 20;
}
dim3 grid_of(int64_t tokens, const Deal &d) {
    // 16384 tokens by 36 heads of 128 in bf16: 64 us, 73 with a wave for every token
    return dim3((unsigned)((tokens + 3) / 4 < kBlocks ? (tokens + 3) / 4 : kBlocks), d.chunks);
}
// The gradient's groups: as many workgroups over the tokens as there may be partial sums of.
dim3 grad_grid(const hoard_heads_args &a) {
    const Deal d = deal(a.n_tokens, a.n_q_heads + a.n_kv_heads, lanes_of(a.head_dim));
    if (!a.n_tokens || !d.chunks) return dim3(0, 0);
    const int64_t most = kGroups / d.chunks > 1 ? kGroups / d.chunks : 1, all = ((int64_t)a.n_tokens + 3) / 4;
    return dim3((unsigned)(all < most ? all : most), d.chunks);
}

// f<.., LANES>(...) for the head's length.
#define HOARD_LANES(DIM, CALL)              \
    switch (lanes_of(DIM)) {                \
        case 4: { CALL(4); } break;         \
        case 8: { CALL(8); } break;         \
        case 16: { CALL(16); } break;       \
        default: { CALL(32); } break;       \
    }

template <typename T, typename C>
void forward_of(const hoard_heads_args &a, const Deal &d, hipStream_t s) {
    const hoard_kv_cache c = a.cache ? *a.cache : hoard_kv_cache{};
#define HOARD_CALL(L)                                                                  \
    if (past_caches(a)) heads_kernel<T, C, L, true><<<grid_of(a.n_tokens, d), 256, 0, s>>>(a, c, d); \
    else heads_kernel<T, C, L, false><<<grid_of(a.n_tokens, d), 256, 0, s>>>(a, c, d)
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
void grad_type(const hoard_heads_args &a, const hoard_heads_grads &g, float *work, dim3 groups, const Deal &d, hipStream_t s) {
#define HOARD_CALL(L)                                                                     \
    if (past_caches(a)) heads_grad_kernel<T, L, true><<<groups, 256, 0, s>>>(a, g, work, d); \
    else heads_grad_kernel<T, L, false><<<groups, 256, 0, s>>>(a, g, work, d)
    HOARD_LANES(a.head_dim, HOARD_CALL)
#undef HOARD_CALL
}
template <typename T, typename C>
void read_of(const KvReadArgs &a, const Deal &d, hipStream_t s) {
#define HOARD_CALL(L) kv_read_kernel<T, C, L><<<grid_of(a.n_tokens, d), 256, 0, s>>>(a, d)
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
    const dim3 g = grad_grid(a);
    return (int)(g.x * g.y);
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
    if (groups) {
        const Deal d = deal(a.n_tokens, a.n_q_heads + a.n_kv_heads, lanes_of(a.head_dim));
        if (a.type == HOARD_TYPE_F32) grad_type<float>(a, g, work, grad_grid(a), d, s);
        else if (a.type == HOARD_TYPE_F16) grad_type<f16>(a, g, work, grad_grid(a), d, s);
        else grad_type<bf16>(a, g, work, grad_grid(a), d, s);
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

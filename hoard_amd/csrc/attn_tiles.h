// Attention of a few new tokens a sequence over a paged cache, on matrix instructions
// (v_mfma_f32_16x16x32_{f16,bf16}).
//
//   S_j = scale <q, k_j>,  out = sum_j exp(S_j - m) v_j / sum_j exp(S_j - m),  m = max_j S_j
//
// The rows that share a key head, the query heads of its group for each new token, are
// taken 16 at a time; a wave takes 16 of them and every KW-th tile of 32 keys.  It needs no
// LDS and no other lane's data in its loop but two exchanges for the maximum:
//   S^T = K Q^T: a lane reads 16 bytes of one key (operand A) and gets 8 scores of one row
//   (column lane % 16; keys 4 (lane / 16) + 0..3 of either half of the tile).  Those are,
//   as they lie, operand B of
//   out^T = V^T P^T, whose order of keys is free as long as V's is the same: a lane reads 8
//   columns of those same 8 keys and transposes the 8 x 8 values in its registers.  It ends
//   with 32 consecutive columns of one row, and the row's maximum and factor are its own.
// The next tile's keys are fetched once this tile's scores are formed, its values once this
// tile's are used, so that half a tile or more is in flight all the time.
//
// Bound by memory from some 10 MB on: 131071 tokens of 8-bit codes by 4 key heads of 128 (138
// MB) take 29 us, 4.8 TB/s, and 4.8 for the join; 8 x 2048 tokens by 16 key heads in f16 (134 MB)
// 31 (28.2 at best, 4.8 TB/s); below, by the latencies one after the other (lengths, pages and queries, keys,
// joining the waves: 4 us) and a tile's 1 us a wave: 257 tokens 7.4 us.  A load of keys takes 64
// bytes of each of 16 rows: one CU reads 16-bit caches at 62 bytes a ns so (138 in whole rows),
// three times what it gets where all of them read.
//
// The matrix instructions have far less to do than they could meanwhile (4 rows * dim operations
// a key for 2 dim values).  So they take more of them where that keeps digits: weights as two
// 16-bit planes (f16: 22 bits, bf16: 16; three for fp32: 24), fp32 queries as two f16 planes of a
// row brought by a power of two to 2^14 or as three bf16 planes.  8-bit codes become f16
// exactly (the byte as a subnormal, times 2^15 less a quarter: code * 2^-9); a key's scale
// multiplies its score, a value's its weight.  Each row has a power of two of its own that its
// weighted sums are held by, that of the largest product of a weight and a scale that it has seen,
// so that the products stay in f16's range: no other row's keys and no scale that weighs nothing
// take digits from it.
#pragma once

#include <math.h>

#include <type_traits>

#include "attn.h"
#include "attn_split.h"
#include "opsdev.h"

namespace hoard {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));

namespace attn {

// The elements that products are formed in, and the planes of queries and weights.
template <typename T, typename C>
struct Core {
    typedef f16 E;
    static constexpr int qp = __is_same(T, float) ? 2 : 1, pp = 2;
};
template <typename T>
struct Core<T, bf16> {
    typedef bf16 E;
    static constexpr int qp = __is_same(T, float) ? 3 : __is_same(T, f16) ? 2 : 1, pp = __is_same(T, float) ? 3 : 2;
};

__device__ __forceinline__ v4f product(f16, v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f product(bf16, v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// Two values rounded to nearest, and what that leaves of them.
__device__ __forceinline__ uint32_t plane(f16, v2f &x) {
    const v2h h = __builtin_convertvector(x, v2h);
    x -= __builtin_convertvector(h, v2f);
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ uint32_t plane(bf16, v2f &x) {
    const v2bf h = __builtin_convertvector(x, v2bf);
    x -= __builtin_convertvector(h, v2f);
    return __builtin_bit_cast(uint32_t, h);
}

// Of 16-bit pairs those that are not finite, as masks of their halves: an exponent of ones carries
// into the sign's place.
__device__ __forceinline__ uint32_t carried(f16, uint32_t w) { return (w & 0x7c007c00u) + 0x04000400u; }
__device__ __forceinline__ uint32_t carried(bf16, uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }
template <typename E>
__device__ __forceinline__ uint32_t not_finite(E, uint32_t w) {
    const uint32_t c = carried(E(), w);
    return (c & 0x8000u ? 0xffffu : 0u) | (c >> 31 ? 0xffff0000u : 0u);
}
// Their signs: one, minus one or zero.
__device__ __forceinline__ uint32_t signs(uint32_t one, uint32_t w) {
    return (w & 0x80008000u) | ((((w & 0x7fff7fffu) + 0x7fff7fffu) >> 15 & 0x00010001u) * one);
}

// Waits out the last matrix instruction (16 states, more than any of its kind takes) before
// vector instructions read its result behind a branch, over which the compiler was seen not to
// count them.
__device__ __forceinline__ void settle(v4f &a, v4f &b) { asm volatile("s_nop 15" : "+v"(a), "+v"(b)); }
template <int N>
__device__ __forceinline__ void settle(v4f (&a)[N]) {
    static_assert(N % 4 == 0, "four at a time");
#pragma unroll
    for (int i = 0; i < N; i += 4) asm volatile("s_nop 15" : "+v"(a[i]), "+v"(a[i + 1]), "+v"(a[i + 2]), "+v"(a[i + 3]));
}

// Maximum and sum over the four lanes 16 apart, in all of them.
__device__ __forceinline__ float far_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float far_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int far_max_i(int v) {
    auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((int)r[0], (int)r[1]);
    r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return max((int)r[0], (int)r[1]);
}
__device__ __forceinline__ int row16_max_i(int v) {
    v = max(v, dpp_i<kDppQuadXor1>(v));
    v = max(v, dpp_i<kDppQuadXor2>(v));
    v = max(v, dpp_i<kDppRowHalfMirror>(v));
    return max(v, dpp_i<kDppRowMirror>(v));
}
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Two codes (plus 128), the low bytes of the halves of w, as f16: code * 2^-9.
constexpr int kCodeShift = 9;
__device__ __forceinline__ uint32_t codes_f16(uint32_t w) {
    const v2h up = {(f16)32768.0f, (f16)32768.0f}, less = {(f16)-0.25f, (f16)-0.25f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, w), up, less));
}
// Eight codes of a key, in their order.
__device__ __forceinline__ v4u codes_row(v2u w) {
    w ^= 0x80808080u;
    v4u o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        o[2 * i] = codes_f16(__builtin_amdgcn_perm(0, w[i], 0x0c010c00));
        o[2 * i + 1] = codes_f16(__builtin_amdgcn_perm(0, w[i], 0x0c030c02));
    }
    return o;
}

// `bytes` bytes from `at` on as a buffer, and W words of it; those behind its end are zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void *at, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(at), (short)0, bytes, 0x00020000);
}
template <int W>
__device__ __forceinline__ auto load(__amdgpu_buffer_rsrc_t from, int at) {
    if constexpr (W == 4) return __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
    else if constexpr (W == 2) return __builtin_amdgcn_raw_buffer_load_b64(from, at, 0, 0);
    else return __builtin_bit_cast(uint32_t __attribute__((ext_vector_type(1))), __builtin_amdgcn_raw_buffer_load_b32(from, at, 0, 0));
}

// A lane's part of a tile of 32 keys as it lies in memory: of the keys 16-byte pieces for
// the products' steps, of the values DV columns (a piece) of each of 8 keys.
template <typename C, int DP>
struct Shape {
    static constexpr int DV = DP == 64 ? 4 : 8;              // columns of a lane, and once more 128 further on
    static constexpr int H = DP / (16 * DV), NC = DV * H;    // products of a tile's values
    static constexpr int STEPS = DP / 32;                    // products of a tile's keys, each half
    static constexpr int KL = DP * (int)sizeof(C) / 64;      // pieces of a key
    static constexpr int VW = DV * (int)sizeof(C) / 4;       // words of a piece of a value
    typedef uint32_t piece __attribute__((ext_vector_type(VW)));
};

}  // namespace attn

// The tiles first .. last - 1 of a lane of work by one workgroup: `row_waves` of its waves
// side by side over the rows, kAttnWaves / row_waves deep over the tiles.  part: where the result goes in the
// workspace, or -1 for a lane that is whole.
template <typename T, typename C, int DP, bool WHOLE>
__device__ __forceinline__ void attn_part(const AttnCall &p, int seq, int lane_no, int seen, int keys, int first, int last, int64_t part) {
    using namespace attn;
    typedef Shape<C, DP> G;
    typedef Core<T, C> K;
    typedef typename K::E E;
    constexpr bool CODES = sizeof(C) == 1, HALF = __is_same(E, f16), SCALED = HALF && !__is_same(T, f16);
    constexpr int DV = G::DV, NC = G::NC, STEPS = G::STEPS;
    // f16 weights reach from 2^15 down (those of codes by their own power)
    constexpr float kLift = HALF && !CODES ? 32768.0f : 1.0f;
    __shared__ float stat[kAttnWaves][2][16];
    __shared__ v4f outs[kAttnWaves][16][16 * DV / 4 + 1];

    const hoard_kv_cache &c = p.c;
    const hoard_attn_args &a = p.a;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wave = wave_index();
    const int kv = lane_no / p.row_blocks, block = lane_no % p.row_blocks;
    const int group = a.n_q_heads / c.n_kv_heads, rows = a.n_new * group, dim = WHOLE ? DP : c.head_dim;
    const int rw = wave % p.row_waves, kw = wave / p.row_waves, kw_all = kAttnWaves / p.row_waves;
    const int row0 = (block * p.row_waves + rw) * 16, row = min(row0 + n, rows - 1);

    // page numbers of 64 pages from page0 on, a lane each
    const int shift = 31 - __builtin_clz(c.page), last_page = (max(keys, 1) - 1) >> shift;
    const int32_t *table = a.pages + (int64_t)seq * a.max_pages;
    const int first_page = (min(first + kw, last - 1) * kKeyTile) >> shift;
    int ti = first + kw, page0 = first_page, numbers = -1;
    if (keys) numbers = table[min(page0 + lane, a.max_pages - 1)];
    // the queries, asked for before the first keys and used behind them
    Raw<T> q_raw[STEPS];
    {
        const T *from = static_cast<const T *>(a.q) + ((int64_t)seq * a.n_new + row / group) * a.q_stride +
                        (kv * group + row % group) * dim;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = CODES ? (s / 2) * 64 + 16 * g + (s % 2) * 8 : s * 32 + 8 * g;
            q_raw[s] = fetch(from, Cols{d < dim ? d : 0, 0}, dim);
        }
    }
    // the keys that the wave's rows see: each its own, the most and the fewest
    const int mine = __shfl(seen, row / group);
    const int hi = row0 < rows ? __builtin_amdgcn_readfirstlane(row16_max_i(mine)) : 0;
    const int lo = -__builtin_amdgcn_readfirstlane(row16_max_i(-mine));
    const int end = min(last, (int)(((uint32_t)hi + kKeyTile - 1) / kKeyTile));
    asm volatile("" : "+v"(numbers));
    struct Where {
        int64_t at[2];  // the cache's rows of the tile's halves
        int n[2];       // of which the wave's rows see so many
    };
    auto where = [&](int tile) {
        Where w;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int j = tile * kKeyTile + 16 * t, page = min(j >> shift, last_page);
            if (page - page0 >= 64) {
                page0 = page;
                numbers = table[min(page + lane, a.max_pages - 1)];
                // waited for here, once in 64 pages: where the numbers are used the wait would be
                // for the keys and values in flight as well
                asm volatile("" : "+v"(numbers));
            }
            const int number = __builtin_amdgcn_readlane(numbers, page - page0);
            const bool ok = (uint32_t)number < (uint32_t)c.n_pages;
            w.n[t] = ok ? min(max(hi - j, 0), 16) : 0;
            w.at[t] = ((int64_t)(ok ? number : 0) * c.n_kv_heads + kv) * c.page + (j & (c.page - 1));
        }
        return w;
    };

    v4u key[2][G::KL];
    typename G::piece val[8][G::H];
    v4f key_scale[2], val_scale[2];
    // Through buffers that end behind the last key that is seen: what lies behind reads as
    // zeros, so no value there, whatever it is, meets a weight of zero.
    auto fetch_keys = [&](const Where &w) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const auto from = buffer(static_cast<const C *>(c.k) + w.at[t] * dim, w.n[t] * dim * (int)sizeof(C));
#pragma unroll
            for (int s = 0; s < G::KL; s++) {
                const int d = (s * 64 + 16 * g) / (int)sizeof(C);
                key[t][s] = load<4>(from, (n * dim + (WHOLE || d < dim ? d : 0)) * (int)sizeof(C));
            }
            if constexpr (CODES) key_scale[t] = __builtin_bit_cast(v4f, load<4>(buffer(c.k_scale + w.at[t], w.n[t] * 4), 16 * g));
        }
    };
    auto fetch_values = [&](const Where &w) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const auto from = buffer(static_cast<const C *>(c.v) + w.at[t] * dim, w.n[t] * dim * (int)sizeof(C));
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int h = 0; h < G::H; h++) {
                    const int d = DV * n + 16 * DV * h;
                    val[4 * t + r][h] = load<G::VW>(from, ((4 * g + r) * dim + (WHOLE || d < dim ? d : 0)) * (int)sizeof(C));
                }
            if constexpr (CODES) val_scale[t] = __builtin_bit_cast(v4f, load<4>(buffer(c.v_scale + w.at[t], w.n[t] * 4), 16 * g));
        }
    };

    float m = -INFINITY, l = 0.0f;
    v4f acc[NC] = {};
    // of codes acc is held times 2^-acc_up, a power of the row's own: kLowest while nothing counts
    constexpr int kLowest = -512;
    int acc_up = kLowest;
    // whether the tiles are gone through once more, with all that is not finite taken out of the
    // products, and the tiles whose values hold such
    bool careful = false;
    int odd_from = INT32_MAX, odd_to = -1;
    // without a condition (a wave without a tile fetches the last one, a lane without keys the
    // cache's first page), so that the queries' wait is not for these as well
    Where cur = where(min(ti, last - 1)), next{};
    fetch_keys(cur);
    fetch_values(cur);

    // queries, as planes: the k-th values of a product's step are those that the keys' pieces hold
    v4u q[K::qp][STEPS];
    int up = 0;  // q is held times 2^up
    {
        float x[STEPS][8];
        int top = 0;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const int d = CODES ? (s / 2) * 64 + 16 * g + (s % 2) * 8 : s * 32 + 8 * g;
            widen(q_raw[s], x[s]);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[s][i] = d < dim && row0 + n < rows ? x[s][i] : 0.0f;
                top = max(top, __float_as_int(x[s][i]) & 0x7fffffff);
            }
        }
        if constexpr (SCALED) {
            top = far_max_i(top);
            up = top ? 14 + 127 - (top >> 23) : 0;
        }
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v2f v = {x[s][2 * i], x[s][2 * i + 1]};
                if constexpr (K::qp == 1) v += v - v;  // an infinity is NaN, as its second plane is
                if constexpr (SCALED) v = v2f{ldexpf(v[0], up), ldexpf(v[1], up)};
#pragma unroll
                for (int pl = 0; pl < K::qp; pl++) q[pl][s][i] = plane(E(), v);
            }
    }
    const float to_log2 = a.scale * 1.4426950408889634f;
    const int down = (CODES ? kCodeShift : 0) - up;

    // The last tile is a copy of the loop without fetches: under a condition the compiler
    // could not count them, and would wait for all.
    auto step = [&](auto more) {
        const bool full = (ti + 1) * kKeyTile <= lo && cur.n[0] == 16 && cur.n[1] == 16;
        if constexpr (more.value) next = where(ti + kw_all);

        if constexpr (!WHOLE) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int s = 0; s < G::KL; s++)
                    if ((s * 64 + 16 * g) / (int)sizeof(C) >= dim) key[t][s] = v4u{0, 0, 0, 0};
        }
        v4f score[2] = {};
        // A key's infinity times the planes of a query would be NaN where they differ in sign or end
        // in zeros: it counts once, by the query's sign.
        if constexpr (!CODES && K::qp > 1)
            if (careful) {
#pragma unroll
                for (int s = 0; s < STEPS; s++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        v4u bad, sign;
#pragma unroll
                        for (int w = 0; w < 4; w++) {
                            const uint32_t mask = not_finite(E(), key[t][s][w]);
                            bad[w] = key[t][s][w] & mask;
                            key[t][s][w] &= ~mask;
                            sign[w] = signs(HALF ? 0x3c00u : 0x3f80u, q[0][s][w]);
                        }
                        score[t] = product(E(), bad, sign, score[t]);
                    }
                settle(score[0], score[1]);
            }
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                v4u k;
                if constexpr (CODES) {
                    const v4u w = key[t][s / 2];
                    k = codes_row(s % 2 ? v2u{w[2], w[3]} : v2u{w[0], w[1]});
                } else {
                    k = key[t][s];
                }
#pragma unroll
                for (int pl = 0; pl < K::qp; pl++) score[t] = product(E(), k, q[pl][s], score[t]);
            }
        settle(score[0], score[1]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = score[i / 4][i % 4] * to_log2;
            // the powers of two meet before the score, whose size they leave 32 bits by
            if constexpr (CODES) x[i] *= ldexpf(key_scale[i / 4][i % 4], down);
            else if constexpr (SCALED) x[i] = ldexpf(x[i], down);
        }
        if constexpr (more.value) fetch_keys(next);
        if (!full) {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (ti * kKeyTile + 16 * (i / 4) + 4 * g + i % 4 >= mine || 4 * g + i % 4 >= cur.n[i / 4]) {
                    x[i] = -INFINITY;
                    if constexpr (CODES) val_scale[i / 4][i % 4] = 0.0f;  // whatever it is
                }
        }
        const float top = far_max(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))));
        if (__any(top > m)) {
            if constexpr (CODES) {
                // a whole number, by which acc's power falls as the earlier weights do: acc stays as it is
                const float to = top > m ? ceilf(top) : m, rise = to > m ? to - m : 0.0f;
                acc_up = max(acc_up - (int)fminf(rise, 1024.0f), kLowest);
                l *= exp2_of(-rise);
                m = to;
            } else {
                const float f = top > m ? exp2_of(m - top) : 1.0f;
                settle(acc);
                m = fmaxf(m, top);
                l *= f;
#pragma unroll
                for (int i = 0; i < NC; i++) acc[i] *= f;
            }
        }
        const float base = m > -INFINITY ? m : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = exp2_of(x[i] - base);
            l += x[i];
        }

        // Values that are not finite count as zeros, and are added to the rows that see them after
        // the loop: zero times them is not zero, nor is a plane of a weight.  (Of codes only the
        // scale may be so, which each row has as its own.)
        if constexpr (!CODES)
            if (careful) {
                uint32_t any = 0;
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int h = 0; h < G::H; h++)
#pragma unroll
                        for (int w = 0; w < G::VW; w++) {
                            any |= carried(E(), val[i][h][w]);
                            val[i][h][w] &= ~not_finite(E(), val[i][h][w]);
                        }
                if (__any(any & 0x80008000u)) {
                    odd_from = min(odd_from, ti);
                    odd_to = ti;
                }
            }
        if constexpr (CODES) {
            float scaled[8];
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                scaled[i] = x[i] * ldexpf(val_scale[i / 4][i % 4], -acc_up);
                most = max(most, __float_as_uint(scaled[i]));
            }
            // near the end of f16's range (or a NaN, or below zero): exponents added, which no scale
            // leaves, and products below 2^14, so that it is not the next tile's turn at once (64
            // sequences of 512 to 8192 tokens 78.0 us, 80.7 with products below 2^15 and so checked)
            if (__any(most > __float_as_uint(65000.0f))) {
                int need = kLowest;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float scale = fabsf(val_scale[i / 4][i % 4]);
                    if (x[i] > 0.0f && scale > 0.0f && scale < INFINITY)
                        need = max(need, __builtin_amdgcn_frexp_expf(x[i]) + __builtin_amdgcn_frexp_expf(scale) - 14);
                }
                const int to = max(acc_up, far_max_i(need));
                settle(acc);
#pragma unroll
                for (int i = 0; i < NC; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[i][r] = ldexpf(acc[i][r], acc_up - to);
                acc_up = to;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float scale = val_scale[i / 4][i % 4];
                    scaled[i] = ldexpf(x[i] * __builtin_amdgcn_frexp_mantf(scale), __builtin_amdgcn_frexp_expf(scale) - acc_up);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = scaled[i];
        }
        // weights as planes: word w holds keys 2w and 2w + 1 of the lane's eight
        v4u weight[K::pp];
#pragma unroll
        for (int w = 0; w < 4; w++) {
            // lifted here, not in the exponent, which would lose digits and, from 2^24 on, the lift
            v2f v = {x[2 * w] * kLift, x[2 * w + 1] * kLift};
#pragma unroll
            for (int pl = 0; pl < K::pp; pl++) weight[pl][w] = plane(E(), v);
        }
        // the lane's keys of column i, in the weights' order
        auto column = [&](int i, int h) {
            v4u o;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if constexpr (CODES)
                    o[w] = codes_f16(__builtin_amdgcn_perm(val[2 * w + 1][h][i / 4] ^ 0x80808080u, val[2 * w][h][i / 4] ^ 0x80808080u,
                                                           0x0c040c00u + 0x00010001u * (i % 4)));
                else
                    o[w] = __builtin_amdgcn_perm(val[2 * w + 1][h][i / 2], val[2 * w][h][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
            }
            return o;
        };
#pragma unroll
        for (int h = 0; h < G::H; h++)
#pragma unroll
            for (int i = 0; i < DV; i++) {
                const v4u o = column(i, h);
#pragma unroll
                for (int pl = 0; pl < K::pp; pl++) acc[h * DV + i] = product(E(), o, weight[pl], acc[h * DV + i]);
            }
        if constexpr (more.value) fetch_values(next);
    };
    while (true) {
        for (; ti + kw_all < end; ti += kw_all, cur = next) step(std::true_type{});
        if (ti < end) step(std::false_type{});
        settle(acc);
        if constexpr (CODES) break;
        if (careful) break;
        // not finite: some key or value is not, that a row sees or that met a weight of zero
        v4f none = acc[0] * 0.0f;
#pragma unroll
        for (int i = 1; i < NC; i++) none += acc[i] * 0.0f;
        const float sum = (none[0] + none[1]) + (none[2] + none[3]) + l * 0.0f;
        if (!__any(sum != sum)) break;
        careful = true;
        ti = first + kw;
        page0 = first_page;
        numbers = table[min(page0 + lane, a.max_pages - 1)];
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; i++) acc[i] = v4f{0, 0, 0, 0};
        cur = where(min(ti, last - 1));
        fetch_keys(cur);
        fetch_values(cur);
    }
    l = far_sum(l);
    // what was not finite, to the rows that see it
    if constexpr (!CODES)
        for (int tile = odd_from; tile <= odd_to; tile += kw_all)
            for (int j = tile * kKeyTile; j < min(hi, (tile + 1) * kKeyTile); j++) {
                const int number = table[j >> shift];
                if (j >= mine || (uint32_t)number >= (uint32_t)c.n_pages) continue;
                const int64_t at = ((int64_t)number * c.n_kv_heads + kv) * c.page + (j & (c.page - 1));
                const C *from = static_cast<const C *>(c.v) + at * dim;
#pragma unroll
                for (int h = 0; h < G::H; h++)
#pragma unroll
                    for (int i = 0; i < DV; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const int d = 16 * DV * h + DV * (4 * g + r) + i;
                            const float v = d < dim ? (float)from[d] : 0.0f;
                            if (!(fabsf(v) <= 3.4028235e38f)) acc[h * DV + i][r] += v;
                        }
            }
    // the waves of the same rows joined: each scales its sums to the maximum of all
    if (g == 0) {
        stat[wave][0][n] = m;
        stat[wave][1][n] = l;
    }
    __syncthreads();
    float top = -INFINITY, total = 0.0f;
    for (int w = 0; w < kw_all; w++) top = fmaxf(top, stat[w * p.row_waves + rw][0][n]);
    const float base = top > -INFINITY ? top : 0.0f;
    for (int w = 0; w < kw_all; w++) total += exp2_of(stat[w * p.row_waves + rw][0][n] - base) * stat[w * p.row_waves + rw][1][n];
    // of codes the maxima are whole numbers, and the step between them goes with acc's power
    const float f = total == 0.0f ? 0.0f : CODES ? 1.0f / total : exp2_of(m - base) / total * (1.0f / kLift);
    const int out_up = CODES ? acc_up + kCodeShift + (int)fmaxf(m - base, -2048.0f) : 0;
    if (kw == 0 && g == 0 && row0 + n < rows) {
        const int64_t out = ((int64_t)seq * a.n_new + row / group) * a.n_q_heads + kv * group + row % group;
        if (part >= 0) reinterpret_cast<v2f *>(p.part_stat)[part * p.block_rows + rw * 16 + n] = v2f{top, total};
        else if (a.lse) a.lse[out] = (base + log2f(total)) * 0.6931471805599453f;
    }
#pragma unroll
    for (int h = 0; h < G::H; h++) {
        if (h) __syncthreads();
#pragma unroll
        for (int i = 0; i < DV; i += 4)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                v4f v;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    v[k] = acc[h * DV + i + k][r] * f;
                    if constexpr (CODES) v[k] = ldexpf(v[k], out_up);
                }
                outs[wave][n][(DV * (4 * g + r) + i) / 4] = v;
            }
        __syncthreads();
        for (int at = threadIdx.x; at < p.row_waves * 16 * 4 * DV; at += 64 * kAttnWaves) {
            const int quad = at % (4 * DV), r = at / (4 * DV) % 16, tile = at / (4 * DV * 16);
            const int d = 16 * DV * h + 4 * quad, of = (block * p.row_waves + tile) * 16 + r;
            if (of >= rows || d >= dim) continue;
            v4f v = outs[tile][r][quad];
            for (int w = 1; w < kw_all; w++) v += outs[w * p.row_waves + tile][r][quad];
            const int64_t out = ((int64_t)seq * a.n_new + of / group) * a.n_q_heads + kv * group + of % group;
            if (part < 0) {
                T o[4];
#pragma unroll
                for (int k = 0; k < 4; k++) o[k] = (T)v[k];
                T *to = static_cast<T *>(a.out) + out * dim + d;
#pragma unroll
                for (int k = 0; k < 4; k++) to[k] = o[k];
            } else {
                *reinterpret_cast<v4f *>(p.part_out + (part * p.block_rows + tile * 16 + r) * dim + d) = v;
            }
        }
    }
}

template <typename T, typename C, int DP, bool WHOLE>
__global__ __launch_bounds__(64 * kAttnWaves, DP > 128 ? 1 : 2) void attn_tile_kernel(AttnCall p) {
    const int lanes = p.c.n_kv_heads * p.row_blocks, limit = p.a.max_pages * p.c.page;
    if (!p.split) {
        const int seq = blockIdx.x / lanes, seen = attn_seen(p.a, limit, seq), keys = attn_most(seen);
        attn_part<T, C, DP, WHOLE>(p, seq, blockIdx.x % lanes, seen, keys, 0, attn_tiles(keys), -1);
        return;
    }
    const AttnPlace place = attn_place(p);
    if (place.seq < 0) return;
    int seq = place.seq, seen = attn_seen(p.a, limit, seq), keys = place.keys, tiles = attn_tiles(keys);
    const bool own = place.own;
    const int row_tiles = attn_row_tiles(tiles, place.run, own);
    int at = blockIdx.x * place.run - place.first, lane = at / row_tiles;
    at -= lane * row_tiles;
    int left = min(place.run, own ? tiles - at : place.total - (int)blockIdx.x * place.run);
    lane = __builtin_amdgcn_readfirstlane(lane);
    at = __builtin_amdgcn_readfirstlane(at);
    left = __builtin_amdgcn_readfirstlane(left);
    while (true) {
        const int last = min(tiles, at + left);
        const bool whole = at == 0 && last == tiles;
        const int64_t part = (int64_t)blockIdx.x + (own ? 0 : (int64_t)seq * lanes + lane);
        attn_part<T, C, DP, WHOLE>(p, seq, lane, seen, keys, at, last, whole ? -1 : part);
        left -= last - at;
        if (left <= 0) return;
        at = 0;
        if (++lane == lanes) {
            lane = 0;
            seen = attn_seen(p.a, limit, ++seq);
            keys = attn_most(seen);
            tiles = attn_tiles(keys);
        }
        __syncthreads();  // the LDS of the part before
    }
}

template <typename T, typename C, int DP>
void launch_attn_dim(const AttnCall &p, hipStream_t s) {
    const int grid = attn_grid(p);
    if (p.c.head_dim == DP) attn_tile_kernel<T, C, DP, true><<<grid, 64 * kAttnWaves, 0, s>>>(p);
    else attn_tile_kernel<T, C, DP, false><<<grid, 64 * kAttnWaves, 0, s>>>(p);
}
template <typename T, typename C>
hipError_t launch_attn_typed(const AttnCall &p, hipStream_t s) {
    if (p.c.head_dim <= 64) launch_attn_dim<T, C, 64>(p, s);
    else if (p.c.head_dim <= 128) launch_attn_dim<T, C, 128>(p, s);
    else launch_attn_dim<T, C, 256>(p, s);
    return hipGetLastError();
}
template <typename C>
hipError_t launch_attn_cache(const AttnCall &p, hipStream_t s) {
    if (p.a.type == HOARD_TYPE_F32) return launch_attn_typed<float, C>(p, s);
    if (p.a.type == HOARD_TYPE_F16) return launch_attn_typed<f16, C>(p, s);
    return launch_attn_typed<bf16, C>(p, s);
}

}  // namespace hoard

// 4-bit products on matrix instructions (v_mfma_f32_16x16x32_{bf16,f16}).
//
// A workgroup takes a tile of up to 16 MT rows of x (of one matrix) and NW * 16 P
// rows of W (NW * 16 of both matrices with a second one).  Its waves are NW wide
// over the rows of W and KS deep over the columns, 128 a step; the KS partial sums
// meet in LDS.  Codes go from memory to registers, each read by one wave, two steps
// ahead; x goes through LDS once per workgroup and step.
//
// x is the A operand and W the B operand: a lane then holds one row of W, its
// scale and zero point, and 4 rows of x in an accumulator.  A lane reads 32
// consecutive codes of its row (16 bytes) for four steps of 32 columns.  The order
// of the columns within a step is free as long as x is read in the same one, so
// the words are taken as they come for groups of 128; for 64 and 32 they are
// exchanged between the lanes of a row (v_permlane32_swap, v_permlane16_swap) so
// that a step never spans two groups.  A group's sum is scaled once it is whole.
//
// fp32 activations are two f16 planes: a group of a row is multiplied by the power of
// two that brings its largest value to 2^14, rounded, and what that leaves is rounded
// again.  Their sum is x to 2^-23 of it (the first leaves up to 2^12 steps of x's last
// place, of which the second's 11 bits hold no odd number above 2^11), or to 2^-39 of
// the group's largest value, whichever is more.  With f16's exact codes (below) the sums are
// of the terms themselves; three bf16 planes, exactly x, had to correct sums of 16 + code
// whose terms are five times the plain ones', and were four times further off.
#pragma once

#include <algorithm>
#include <type_traits>

#include "lds_dma.h"
#include "q4.h"

namespace hoard {

template <typename T>
struct Tiles {
    typedef T elem;
    static constexpr int planes = 1;
};
template <>
struct Tiles<float> {
    typedef f16 elem;
    static constexpr int planes = 2;
};

template <typename E>
__device__ __forceinline__ v4f mfma_16x16x32(v4u x, v4u w, v4f c);
template <>
__device__ __forceinline__ v4f mfma_16x16x32<bf16>(v4u x, v4u w, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, w), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ v4f mfma_16x16x32<f16>(v4u x, v4u w, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, w), c, 0, 0, 0);
}

// Waits out the last matrix instruction before its result is read (8 wait states).  The
// compiler counts them itself, but not over a branch: with the rows' early exit between
// the product and its use, it read accumulators that were not there yet.  In bf16 that
// costs 1 to 8 % (most with groups of 32), where the compiler puts other tiles' products
// between; there its order happens to be safe, which nothing guarantees.
// All accumulators go through one statement, which so follows all their products.
__device__ __forceinline__ void settle(v4f (&d)[1]) { asm volatile("s_nop 7" : "+v"(d[0])); }
__device__ __forceinline__ void settle(v4f (&d)[2]) { asm volatile("s_nop 7" : "+v"(d[0]), "+v"(d[1])); }
__device__ __forceinline__ void settle(v4f (&d)[2], v4f &xs) {
    asm volatile("s_nop 7" : "+v"(d[0]), "+v"(d[1]), "+v"(xs));
}

// f16 holds code - zero exactly (11 bits, the zero point being a byte), so there the
// offset is taken off in pairs and no sums of x are needed: 4 instructions for 8 codes
// in place of a product with ones, or of sums formed beside x (2000 rows of x by 8192
// x 4096 in groups of 32: 243 us against 284; 512 rows by 4096 x 4096: 29.8 against 32.2).
template <typename E>
constexpr bool kExact = __is_same(E, f16);
__device__ __forceinline__ v4u less(v4u w, float offset) {
    const f16 o = (f16)-offset;
    const v2h pair = {o, o};
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, (uint32_t)w[i]) + pair);
    return w;
}

// Four words of a lane rearranged among the four lanes (16 apart) of a row of W.
template <int G>
__device__ __forceinline__ v4u exchange(v4u c) {
    if (G <= 64) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const auto r = __builtin_amdgcn_permlane32_swap(c[i], c[i + 2], false, false);
            c[i] = r[0];
            c[i + 2] = r[1];
        }
    }
    if (G <= 32) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const auto r = __builtin_amdgcn_permlane16_swap(c[i], c[i + 1], false, false);
            c[i] = r[0];
            c[i + 1] = r[1];
        }
    }
    return c;
}
// The first of the 8 columns (of 128) that word `step` of lane group `q` holds then.
template <int G>
__device__ __forceinline__ int column_of(int step, int q) {
    if (G == 32) return step * 32 + q * 8;
    if (G == 64) return ((step & 2) + (q & 1)) * 32 + ((q & 2) + (step & 1)) * 8;
    return q * 32 + step * 8;
}

// N scales of a row from index `from` on, and its zero points plus `bias`, into LDS.
template <int N>
__device__ __forceinline__ void load_scales(const hoard_q4_matrix &m, size_t from, float *scale, float *zero, float bias) {
    if (m.scale_type == HOARD_TYPE_F32) {
        float v[N];
        __builtin_memcpy(v, static_cast<const float *>(m.scales) + from, sizeof v);
#pragma unroll
        for (int g = 0; g < N; g++) scale[g] = v[g];
    } else {
        uint16_t v[N];
        __builtin_memcpy(v, static_cast<const uint16_t *>(m.scales) + from, sizeof v);
        const bool half = m.scale_type == HOARD_TYPE_F16;
#pragma unroll
        for (int g = 0; g < N; g++)
            scale[g] = half ? (float)__builtin_bit_cast(f16, v[g]) : __uint_as_float((uint32_t)v[g] << 16);
    }
    uint8_t z[N];
    if (m.zeros) __builtin_memcpy(z, m.zeros + from, sizeof z);
#pragma unroll
    for (int g = 0; g < N; g++) zero[g] = bias + (m.zeros ? (float)z[g] : 8.0f);
}

// Eight values of a row of x as they are fetched.
template <typename T>
struct Piece {
    uint32_t w[2 * sizeof(T)];
};

// The tile of the workgroup: matrix, first row and row count.  Sorted rows: tile
// number `t` over the matrices' tiles in ascending order; each lane adds up a run
// of matrices.  False: no such tile.
__device__ __forceinline__ bool tile_of(const Q4Args &a, int64_t t, int tm, int &e, int &r0, int &rows) {
    if (a.mode != kQ4Sorted) {
        if (t * tm >= a.n_rows) return false;
        e = 0;
        r0 = (int)t * tm;
        rows = min(tm, a.n_rows - r0);
        return true;
    }
    const int lane = threadIdx.x & 63, n = a.w.n_mat, per = (n + 63) / 64, e0 = lane * per, e1 = min(n, e0 + per);
    auto at = [&](int i) { return max(0, min(a.n_rows, a.sel[i])); };
    // whole tiles and the rest of a matrix's rows: the whole ones of all matrices come
    // first, so that the launch does not end on the longest work
    int whole = 0, rest = 0;
    if (e0 < e1) {
        int lo = at(e0);
        for (int i = e0; i < e1; i++) {
            const int hi = at(i + 1), c = max(0, hi - lo);
            whole += c / tm;
            rest += c % tm != 0;
            lo = hi;
        }
    }
    int incl_w = whole, incl_r = rest;
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl_w, d), u = __shfl_up(incl_r, d);
        if (lane >= d) incl_w += v, incl_r += u;
    }
    const int all = __builtin_amdgcn_readlane(incl_w, 63);
    const bool first = t < all;
    if (!first) t -= all;
    const int incl = first ? incl_w : incl_r, mine = first ? whole : rest;
    const uint64_t past = __ballot(incl > t);
    if (!past) return false;
    const int who = __ffsll((unsigned long long)past) - 1;
    int left = (int)t - __builtin_amdgcn_readlane(incl - mine, who), lo = 0, hi = 0;
    for (e = who * per;; e++) {  // ends at the matrix whose tile it is, within the lane's run
        lo = at(e);
        hi = max(lo, at(e + 1));
        const int tiles = first ? (hi - lo) / tm : (hi - lo) % tm != 0;
        if (left < tiles || e + 1 >= n) break;
        left -= tiles;
    }
    const int from = first ? left * tm : (hi - lo) / tm * tm;
    e = __builtin_amdgcn_readfirstlane(e);
    r0 = __builtin_amdgcn_readfirstlane(lo + from);
    rows = __builtin_amdgcn_readfirstlane(min(tm, hi - r0));
    return rows > 0;
}

template <typename T, int G, bool UP, int P, int MT, int NW, int KS, int MW>
__global__ __launch_bounds__(64 * NW * KS, MW) void q4_tiles_kernel(Q4Args a) {
    typedef typename Tiles<T>::elem E;
    constexpr int PL = Tiles<T>::planes, TM = 16 * MT, THREADS = 64 * NW * KS;
    constexpr int NG = 128 / G, SP = 4 / NG;               // groups in a block of 128 columns, steps in a group
    constexpr int COLS = KS * 128;                         // columns of a step of the workgroup
    constexpr int RS = COLS * 2 + 16;                      // bytes of a row of x in LDS: 16 off the banks' period
    constexpr int XP = TM * (COLS / 8) / THREADS;          // pieces of 8 values a thread stages
    constexpr int XROWS = THREADS / (COLS / 8);            // rows of x between them
    constexpr int XS = KS * NG;                            // groups of a step
    constexpr int MEET = KS > 1 ? (KS - 1) * NW * P * MT * 1024 : 0;  // bytes of the partial sums
    static_assert(XROWS * (COLS / 8) == THREADS && XP * XROWS == TM, "whole pieces a thread, whole rows between them");
    static_assert(!UP || P == 2, "the second matrix is the second stream");
    constexpr int XBYTES = PL * TM * RS;
    constexpr int RW = 16 * NW * P;                        // rows of W, both matrices'
    // groups of a row whose scales lie in LDS at a time, a thread's share of them
    constexpr int MINSC = XS > 16 ? XS : 16, SC = MINSC * RW < THREADS ? THREADS / RW : MINSC;
    constexpr int SPC = SC / XS, SI = RW * SC / THREADS;
    static_assert(SC % XS == 0 && RW * SC % THREADS == 0 && SC % SI == 0, "whole steps, whole shares");
    __shared__ __align__(16) uint8_t lds[XBYTES > MEET ? XBYTES : MEET];
    // of a row of x and group: its sum in bf16; in fp32 what undoes its power of two
    constexpr bool SUMS = !kExact<E>, POWERS = PL == 2;
    __shared__ __align__(16) float beside[SUMS || POWERS ? XS : 1][SUMS || POWERS ? TM : 4];
    __shared__ float scale[RW][SC + 1], zero[RW][SC + 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const int nw = KS > 1 ? wave % NW : wave, ks = KS > 1 ? wave / NW : 0;
    const int col = lane & 15, q = lane >> 4;
    int e, r0, rows;
    // a tile of x in all its tiles of W: next to each other, or (a.spread) on one XCD,
    // whose L2 then fetches the rows of x once
    const int nt = (a.w.rows + NW * (UP ? 16 : 16 * P) - 1) / (NW * (UP ? 16 : 16 * P));
    const int id = blockIdx.x, run = a.spread ? id >> 3 : id;
    const int tn = run % nt;
    const int64_t tx = a.tile0 + (a.spread ? (run / nt) * 8 + (id & 7) : run / nt);
    if (!tile_of(a, tx, TM, e, r0, rows)) return;
    const int cols = a.w.cols, blocks = (cols + 127) / 128, steps = (blocks + KS - 1) / KS;
    constexpr int WIDE = UP ? 16 : 16 * P;  // rows of W of a wave
    const int first = (tn * NW + nw) * WIDE, n0 = first + col;

    // the streams: rows of W (clamped: what lies behind the last row is not stored),
    // as a base of the wave's and 32-bit offsets of the lanes'
    const int top = min(first, a.w.rows - 1), groups = cols / G;
    // the last block of a lane's 32 columns that lies inside
    const int last_block = (cols - 32 - q * 32) >= 0 ? (cols - 32 - q * 32) / 128 : 0;
    const size_t row0 = (size_t)e * a.w.rows + top;
    const uint8_t *const x0 = static_cast<const uint8_t *>(a.x) + (size_t)r0 * cols * sizeof(T);
    uint32_t code[P];
#pragma unroll
    for (int p = 0; p < P; p++) {
        const uint32_t row = min(n0 + (UP ? 0 : 16 * p), a.w.rows - 1) - top;
        code[p] = row * (cols / 2) + (q * 32 < cols ? q * 16 : 0);
    }

    // Codes two steps ahead, x one: the loads of a step are issued x first, so that
    // staging x waits for nothing behind it.  Nothing is loaded under a condition: what
    // lies behind the last column or row is read from a place inside instead, x is
    // zeroed behind the last column, and rows behind the last are not stored.
    v4u codes[2][P];
    Piece<T> xr[XP];
    auto fetch_w = [&](auto at, int step) {
        constexpr int B = decltype(at)::value;
        const int block = step * KS + ks;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const hoard_q4_matrix &m = UP && p == 1 ? a.up : a.w;
            const uint8_t *const from = static_cast<const uint8_t *>(m.codes) + row0 * (cols / 2);
            codes[B][p] = *reinterpret_cast<const v4u *>(from + (code[p] + min(block, last_block) * 64));
        }
    };
    // the scales of SC groups into LDS: read along the rows, as they lie in memory
    auto stage_scales = [&](int chunk) {
        const int row = tid / (SC / SI), g0 = (tid % (SC / SI)) * SI, p = row / (16 * NW), in = row % (16 * NW);
        const int n = tn * NW * WIDE + (UP ? in : (in / 16) * WIDE + p * 16 + in % 16);
        const hoard_q4_matrix &m = UP && p == 1 ? a.up : a.w;
        const size_t from = ((size_t)e * a.w.rows + min(n, a.w.rows - 1)) * groups;
        const int g1 = chunk * SC + g0;
        if (SI > 1 && g1 + SI <= groups) {
            load_scales<SI>(m, from + g1, scale[row] + g0, zero[row] + g0, 16.0f);
        } else {
#pragma unroll
            for (int g = 0; g < SI; g++)
                load_scales<1>(m, from + min(g1 + g, groups - 1), scale[row] + g0 + g, zero[row] + g0 + g, 16.0f);
        }
    };
    const int xrow = tid / (COLS / 8), xcol = (tid % (COLS / 8)) * 8;
    auto fetch_x = [&](int step) {
        const int k = min(step * COLS + xcol, cols - 8);
#pragma unroll
        for (int j = 0; j < XP; j++)
            if (j * XROWS < rows)
                xr[j] = *reinterpret_cast<const Piece<T> *>(x0 + (uint32_t)(min(xrow + j * XROWS, rows - 1) * cols + k) *
                                                                     (uint32_t)sizeof(T));
    };
    // x into LDS, and what stands beside it; a group's G / 8 pieces lie in consecutive lanes
    auto stage = [&](int step) {
        if ((step + 1) * COLS > cols) {
            const bool in = step * COLS + xcol < cols;
#pragma unroll
            for (int j = 0; j < XP; j++)
#pragma unroll
                for (int c = 0; c < (int)(2 * sizeof(T)); c++) xr[j].w[c] = in ? xr[j].w[c] : 0u;
        }
#pragma unroll
        for (int j = 0; j < XP; j++) {
            if (j * XROWS >= rows) break;
            const int row = xrow + j * XROWS, piece = xcol / 8;
            uint8_t *to = lds + row * RS + piece * 16;
            float value;
            if constexpr (PL == 1) {
                v4u w;
                __builtin_memcpy(&w, &xr[j], 16);
                *reinterpret_cast<v4u *>(to) = paired(w);
                if constexpr (!SUMS) continue;
                value = 0.0f;
#pragma unroll
                for (int c = 0; c < 4; c++) value = dot2<E>(w[c], kOnes<E>, value);
                value += dpp_f<kDppQuadXor1>(value);
                value += dpp_f<kDppQuadXor2>(value);
                if (G >= 64) value += dpp_f<kDppRowHalfMirror>(value);
                if (G >= 128) value += dpp_f<kDppRowMirror>(value);
            } else {
                // of magnitudes (a NaN's is above them all)
                uint32_t most = 0;
#pragma unroll
                for (int c = 0; c < 8; c++) most = max(most, xr[j].w[c] & 0x7fffffffu);
                most = max(most, __float_as_uint(dpp_f<kDppQuadXor1>(__uint_as_float(most))));
                most = max(most, __float_as_uint(dpp_f<kDppQuadXor2>(__uint_as_float(most))));
                if (G >= 64) most = max(most, __float_as_uint(dpp_f<kDppRowHalfMirror>(__uint_as_float(most))));
                if (G >= 128) most = max(most, __float_as_uint(dpp_f<kDppRowMirror>(__uint_as_float(most))));
                // 2^(141 - e) for the largest value's biased exponent e, and its inverse, both normal
                const uint32_t up = min(268u - (most >> 23), 253u);
                const float power = __uint_as_float(up << 23);
                value = __uint_as_float((254u - up) << 23);
                float x[8];
                v8h high, low;
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    x[c] = __uint_as_float(xr[j].w[c]) * power;
                    high[(c & 3) * 2 + (c >> 2)] = (f16)x[c];
                }
#pragma unroll
                for (int c = 0; c < 8; c++) low[(c & 3) * 2 + (c >> 2)] = (f16)(x[c] - (float)high[(c & 3) * 2 + (c >> 2)]);
                *reinterpret_cast<v8h *>(to) = high;
                *reinterpret_cast<v8h *>(to + TM * RS) = low;
            }
            if (piece % (G / 8) == 0) beside[piece / (G / 8)][row] = value;
        }
    };

    v4f acc[P][MT];
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
        for (int t = 0; t < MT; t++) acc[p][t] = (v4f)(0.0f);

    auto body = [&](auto at, int step) {
        constexpr int B = decltype(at)::value;
        if (step) __syncthreads();  // the last step's x has been read
        if (step % SPC == 0) stage_scales(step / SPC);
        stage(step);
        v4u now[P];
#pragma unroll
        for (int p = 0; p < P; p++) now[p] = exchange<G>(codes[B][p]);
        __syncthreads();
        if (step + 1 < steps) fetch_x(step + 1);
        if (step + 2 < steps) fetch_w(at, step + 2);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            v4u w[P][SP];
            float sc[P], zc[P];
#pragma unroll
            for (int p = 0; p < P; p++) {
                const int at = (step % SPC) * XS + ks * NG + g;
                sc[p] = scale[(p * NW + nw) * 16 + col][at];
                zc[p] = zero[(p * NW + nw) * 16 + col][at];
            }
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int i = 0; i < SP; i++) {
                    w[p][i] = biased<E>(now[p][g * SP + i]);
                    if (kExact<E>) w[p][i] = less(w[p][i], zc[p]);
                }
#pragma unroll
            for (int t = 0; t < MT; t++) {
                if (t * 16 >= rows) break;
                v4f d[P] = {}, xs = (v4f)(1.0f);
                if constexpr (SUMS || POWERS) xs = *reinterpret_cast<const v4f *>(&beside[ks * NG + g][t * 16 + 4 * q]);
                if constexpr (SUMS) {
#pragma unroll
                    for (int p = 0; p < P; p++)
#pragma unroll
                        for (int i = 0; i < 4; i++) d[p][i] = -zc[p] * xs[i];
                }
                const uint8_t *from = lds + (t * 16 + col) * RS + ks * 256;
#pragma unroll
                for (int i = 0; i < SP; i++)
#pragma unroll
                    for (int l = 0; l < PL; l++) {
                        const v4u x = *reinterpret_cast<const v4u *>(from + l * TM * RS + 2 * column_of<G>(g * SP + i, q));
#pragma unroll
                        for (int p = 0; p < P; p++) d[p] = mfma_16x16x32<E>(x, w[p][i], d[p]);
                    }
                settle(d);
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        acc[p][t][i] = fmaf(sc[p], POWERS ? d[p][i] * xs[i] : d[p][i], acc[p][t][i]);
            }
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch_w(even, 0);
    fetch_x(0);
    if (steps > 1) fetch_w(odd, 1);
    for (int step = 0; step < steps; step += 2) {
        body(even, step);
        if (step + 1 < steps) body(odd, step + 1);
    }
    if constexpr (KS > 1) {
        __syncthreads();
        v4f *meet = reinterpret_cast<v4f *>(lds);
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int t = 0; t < MT; t++)
                if (ks) meet[((((ks - 1) * NW + nw) * P + p) * MT + t) * 64 + lane] = acc[p][t];
        __syncthreads();
        if (ks) return;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int k = 1; k < KS; k++) acc[p][t] += meet[((((k - 1) * NW + nw) * P + p) * MT + t) * 64 + lane];
    }
    T *y = static_cast<T *>(a.y) + (size_t)r0 * a.w.rows;
#pragma unroll
    for (int p = 0; p < (UP ? 1 : P); p++) {
        const int n = n0 + 16 * p;
        if (n >= a.w.rows) continue;
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = t * 16 + 4 * q + i;
                if (row >= rows) continue;
                float v = acc[p][t][i];
                if constexpr (UP) v = silu_mul<T>(v, acc[1][t][i]);
                y[(size_t)row * a.w.rows + n] = (T)v;
            }
    }
}

// The same product for 16-bit activations and many rows of x: x goes straight from
// memory to LDS in its own order, the codes take that order (in_order), and in bf16 the
// sums of x, which the zero points multiply, come from a third product with a matrix of
// ones, whose accumulator holds them where the scaled sums need them.  A step is 128 columns; x lies in two buffers, so
// one barrier a step hands over what arrived and frees what was read.
//
// A row of x is 256 bytes of a buffer, its 16-byte pieces exchanged by the row's
// number (piece ^ row % 16), so that 16 rows' pieces fall on all the banks.
template <typename T, int G, bool UP, int MT, int NW, int KS, int MW>
__global__ __launch_bounds__(64 * NW * KS, MW) void q4_flow_kernel(Q4Args a) {
    constexpr int TM = 16 * MT, THREADS = 64 * NW * KS, P = 2, NG = 128 / G, SP = 4 / NG;
    constexpr int CH = TM / 4 / NW;                        // copies of 1 KB a wave and step
    constexpr int RW = 16 * NW * P, XS = KS * NG, SC = XS > 16 ? XS : 16, SPC = SC / XS, SI = RW * SC / THREADS;
    constexpr int WIDE = UP ? 16 : 32;
    static_assert(CH * NW * 4 == TM && SI * THREADS == RW * SC && SC % SI == 0, "whole shares");
    static_assert((KS - 1) * NW * P * MT * 1024 <= KS * 2 * TM * 256, "the partial sums take the place of x");
    __shared__ __align__(16) uint8_t lds[KS][2][TM * 256];
    __shared__ float scale[RW][SC + 1], zero[RW][SC + 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const int nw = KS > 1 ? wave % NW : wave, ks = KS > 1 ? wave / NW : 0;
    const int col = lane & 15, q = lane >> 4;
    int e, r0, rows, tn;
    {
        const int nt = (a.w.rows + NW * WIDE - 1) / (NW * WIDE), id = blockIdx.x, run = a.spread ? id >> 3 : id;
        tn = run % nt;
        if (!tile_of(a, a.tile0 + (a.spread ? (run / nt) * 8 + (id & 7) : run / nt), TM, e, r0, rows)) return;
    }
    const int cols = a.w.cols, groups = cols / G, blocks = (cols + 127) / 128, steps = (blocks + KS - 1) / KS;
    const int first = (tn * NW + nw) * WIDE, n0 = first + col, top = min(first, a.w.rows - 1);
    const int last_block = (cols - 32 - q * 32) >= 0 ? (cols - 32 - q * 32) / 128 : 0;
    const size_t row0 = (size_t)e * a.w.rows + top;
    uint32_t code[P];
#pragma unroll
    for (int p = 0; p < P; p++)
        code[p] = (min(n0 + (UP ? 0 : 16 * p), a.w.rows - 1) - top) * (cols / 2) + (q * 32 < cols ? q * 16 : 0);

    v4u codes[2][P];
    auto fetch_w = [&](auto at, int step) {
#pragma unroll
        for (int p = 0; p < P; p++) {
            const hoard_q4_matrix &m = UP && p == 1 ? a.up : a.w;
            const uint8_t *const from = static_cast<const uint8_t *>(m.codes) + row0 * (cols / 2);
            codes[decltype(at)::value][p] = *reinterpret_cast<const v4u *>(from + (code[p] + min(step * KS + ks, last_block) * 64));
        }
    };
    // the wave's copies: lane l of a copy brings piece (l % 16) ^ row of row l / 16
    const uint8_t *const x0 = static_cast<const uint8_t *>(a.x) + (size_t)r0 * cols * 2;
    uint32_t src[CH];
#pragma unroll
    for (int j = 0; j < CH; j++) src[j] = (uint32_t)min((nw * CH + j) * 4 + q, rows - 1) * (uint32_t)cols * 2;
    const int piece = col ^ q;  // of rows 0..3 of 16; rows 4 j on differ in bits 2 and 3
    auto fetch_x = [&](int buffer, int step) {
#pragma unroll
        for (int j = 0; j < CH; j++)
            if ((nw * CH + j) * 4 < rows)
                dma_lanes_at(lds[ks][buffer] + (nw * CH + j) * 1024, x0,
                             src[j] + 2 * min((step * KS + ks) * 128 + (piece ^ (((nw * CH + j) & 3) * 4)) * 8, cols - 8));
    };
    auto stage_scales = [&](int chunk) {
        const int row = tid / (SC / SI), g0 = (tid % (SC / SI)) * SI, p = row / (16 * NW), in = row % (16 * NW);
        const int n = tn * NW * WIDE + (UP ? in : (in / 16) * WIDE + p * 16 + in % 16);
        const hoard_q4_matrix &m = UP && p == 1 ? a.up : a.w;
        const size_t from = ((size_t)e * a.w.rows + min(n, a.w.rows - 1)) * groups;
        const int g1 = chunk * SC + g0;
        if (SI > 1 && g1 + SI <= groups) {
            load_scales<SI>(m, from + g1, scale[row] + g0, zero[row] + g0, kInOrderBias<T>);
        } else {
#pragma unroll
            for (int g = 0; g < SI; g++)
                load_scales<1>(m, from + min(g1 + g, groups - 1), scale[row] + g0 + g, zero[row] + g0 + g, kInOrderBias<T>);
        }
    };

    v4f acc[P][MT];
#pragma unroll
    for (int p = 0; p < P; p++)
#pragma unroll
        for (int t = 0; t < MT; t++) acc[p][t] = (v4f)(0.0f);
    const v4u ones = (v4u)(kOnes<T>);
    auto body = [&](auto at, int step) {
        constexpr int B = decltype(at)::value;
        if (step % SPC == 0) {
            if (step) __syncthreads();
            stage_scales(step / SPC);
        }
        // this step's codes, and with them the copies of x issued before the next step's
        // codes: what the compiler waits for here, and the wait by itself
#pragma unroll
        for (int p = 0; p < P; p++) asm volatile("" : "+v"(codes[B][p]));
        if (step + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(P) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        v4u now[P];
#pragma unroll
        for (int p = 0; p < P; p++) now[p] = exchange<G>(codes[B][p]);
        if (step + 1 < steps) fetch_x(B ^ 1, step + 1);
        if (step + 2 < steps) fetch_w(at, step + 2);
#pragma unroll
        for (int g = 0; g < NG; g++) {
            if ((step * KS + ks) * 128 + g * G >= cols) break;  // a group lies inside or behind the last column as a whole
            v4u w[P][SP];
            float sc[P], zc[P];
#pragma unroll
            for (int p = 0; p < P; p++) {
                sc[p] = scale[(p * NW + nw) * 16 + col][(step % SPC) * XS + ks * NG + g];
                zc[p] = zero[(p * NW + nw) * 16 + col][(step % SPC) * XS + ks * NG + g];
#pragma unroll
                for (int i = 0; i < SP; i++) {
                    w[p][i] = in_order<T>(now[p][g * SP + i]);
                    if (kExact<T>) w[p][i] = less(w[p][i], zc[p]);
                }
            }
#pragma unroll
            for (int t = 0; t < MT; t++) {
                if (t * 16 >= rows) break;
                v4f d[P] = {}, xs = (v4f)(0.0f);
                const uint8_t *from = lds[ks][B] + (t * 16 + col) * 256;
#pragma unroll
                for (int i = 0; i < SP; i++) {
                    const v4u x = *reinterpret_cast<const v4u *>(from + (((column_of<G>(g * SP + i, q) / 8) ^ col) * 16));
                    if (!kExact<T>) xs = mfma_16x16x32<T>(x, ones, xs);
#pragma unroll
                    for (int p = 0; p < P; p++) d[p] = mfma_16x16x32<T>(x, w[p][i], d[p]);
                }
                if constexpr (kExact<T>) settle(d);
                else settle(d, xs);
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        acc[p][t][i] = fmaf(sc[p], kExact<T> ? d[p][i] : fmaf(-zc[p], xs[i], d[p][i]), acc[p][t][i]);
            }
        }
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    fetch_w(even, 0);
    fetch_x(0, 0);
    if (steps > 1) fetch_w(odd, 1);
    for (int step = 0; step < steps; step += 2) {
        body(even, step);
        if (step + 1 < steps) body(odd, step + 1);
    }
    if constexpr (KS > 1) {
        __syncthreads();
        v4f *meet = reinterpret_cast<v4f *>(&lds[0][0][0]);
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int t = 0; t < MT; t++)
                if (ks) meet[((((ks - 1) * NW + nw) * P + p) * MT + t) * 64 + lane] = acc[p][t];
        __syncthreads();
        if (ks) return;
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int c = 1; c < KS; c++) acc[p][t] += meet[((((c - 1) * NW + nw) * P + p) * MT + t) * 64 + lane];
    }
    T *y = static_cast<T *>(a.y) + (size_t)r0 * a.w.rows;
#pragma unroll
    for (int p = 0; p < (UP ? 1 : P); p++) {
        const int n = n0 + 16 * p;
        if (n >= a.w.rows) continue;
#pragma unroll
        for (int t = 0; t < MT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = t * 16 + 4 * q + i;
                if (row >= rows) continue;
                float v = acc[p][t][i];
                if constexpr (UP) v = silu_mul<T>(v, acc[1][t][i]);
                y[(size_t)row * a.w.rows + n] = (T)v;
            }
    }
}

// Tiles of tm rows of x; with offsets, which the host does not see, at most so many.
inline int64_t tiles_of(const Q4Args &a, int tm) {
    if (a.mode == kQ4Sorted) return a.n_rows / tm + (a.n_rows < a.w.n_mat ? a.n_rows : a.w.n_mat);
    return ((int64_t)a.n_rows + tm - 1) / tm;
}

// launch(part, grid) over the launches that cover the call's tiles.
template <int TM, int TN, typename F>
hipError_t over_tiles(const Q4Args &a, F launch) {
    const int64_t tiles = tiles_of(a, TM);
    const int64_t nt = (a.w.rows + TN - 1) / TN, most = std::max<int64_t>(8, ((1 << 22) / nt) & ~7);  // tiles of a launch
    Q4Args part = a;
    part.spread = tiles >= 32;
    for (part.tile0 = 0; part.tile0 < tiles; part.tile0 += most) {
        const int64_t now = std::min(most, tiles - part.tile0);
        launch(part, (unsigned)(nt * (part.spread ? (now + 7) / 8 * 8 : now)));
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

template <typename T, int G, bool UP, int P, int MT, int NW, int KS, int MW>
hipError_t launch_tiles_of(const Q4Args &a, hipStream_t s) {
    return over_tiles<16 * MT, NW *(UP ? 16 : 16 * P)>(a, [&](const Q4Args &part, unsigned grid) {
        q4_tiles_kernel<T, G, UP, P, MT, NW, KS, MW><<<grid, 64 * NW * KS, 0, s>>>(part);
    });
}
template <typename T, int G, bool UP, int MT, int NW, int KS, int MW>
hipError_t launch_flow_of(const Q4Args &a, hipStream_t s) {
    return over_tiles<16 * MT, NW *(UP ? 16 : 32)>(a, [&](const Q4Args &part, unsigned grid) {
        q4_flow_kernel<T, G, UP, MT, NW, KS, MW><<<grid, 64 * NW * KS, 0, s>>>(part);
    });
}

// The form of a call, by the workgroups it makes.  A workgroup's steps follow one
// another at a latency of 0.7 us or so, whatever the tile's size, so while there are
// fewer workgroups than the 256 CUs hold, smaller tiles and columns split over more
// waves are faster; above that, larger tiles read x and unpack the codes less often.
// Measured on bf16 (us):
//   4096 x 4096, rows of x          16    20    32    64   128   256   512
//     tiles 16, columns / 8        7.8
//     tiles 16, columns / 8, two wide     9.8  10.0  12.8  22.7
//     flow 16, columns / 4        13.8  14.1  14.0  14.9  15.8  28.8  59.6
//     flow 32, columns / 4        14.7  17.7  18.0  18.4  18.8  20.1  37.6
//     flow 64, columns / 2                    20.5  28.6  29.0  29.7  31.6
//     flow 64                     22.0  27.0  27.2  42.0  42.3  42.4  43.8 (8192 rows of W:
//                                               59.5 at 512, where flow 64 / 2 takes 60.8)
//   8192 x 4096, 20 / 64 rows: 12.8 / 25.4 by tiles 16 / 8 two wide, 17.2 / 17.7 by flow 16 / 4.
//   16384 x 8192, 16 rows: 24.5 by tiles 16 / 4 two wide, 34.3 by tiles 16 / 8.
//   Sorted, 10 of 512 experts of 512 x 2048 twice, tokens   1     4    16    64   384
//     tiles 16, columns / 4, two wide                     10.9  18.0  47.7   119   219
//     flow 16, columns / 2                                14.4  17.0  36.1  79.5   156
//     flow 32                                             20.0  21.5  32.3  61.5   118
//   8 of 128 experts of 768 x 2048 twice, 512 tokens: 79 by flow 64, 92 by flow 32.
// On fp32, tiles two streams deep (rows of x x rows of W / columns):
//   4096 x 4096, rows of x           20    64   128   256   512   (8192 x 4096)  20    64   128   512
//     16 x 32 / 8                  14.4  26.1  48.6  93.7   190                23.8  52.6   100   394
//     16 x 64 / 4                  18.9  19.7  36.4  68.2   137                20.2  29.3  53.4   202
//     32 x 64 / 4                  25.1  29.9  30.8  58.4   114                26.5  31.1  57.6   215
//     32 x 128 / 2                 38.5  39.7  40.1  41.9  78.9                40.2  41.5  43.5   157
//     32 x 128                     50.1  50.5  51.2  52.6  68.1                53.4  54.4  56.0   122
//     64 x 128                     50.6  82.7  83.6  84.4  86.2                55.0  92.9  93.3   125
//   Sorted, 4 of 32 experts of 2048 x 2048, tokens   1     4    16    64   512
//     16 x 32 / 4                                  9.1  12.0  22.0  39.2   176
//     16 x 64 / 2                                 10.9  14.4  19.0  33.9   124
//     16 x 128                                    17.2  19.9  24.3  29.5  86.9
//     32 x 128                                    17.5  20.0  24.6  34.0  80.6
constexpr int64_t kCUs = 256;

template <typename T, int G, bool UP>
hipError_t launch_tiles_sized(const Q4Args &a, hipStream_t s) {
    constexpr int P = UP ? 2 : 1;
    const bool sorted = a.mode == kQ4Sorted;
    const int64_t per = sorted ? ((int64_t)a.n_rows + a.w.n_mat - 1) / a.w.n_mat : a.n_rows;  // rows of x of a matrix
    // workgroups with tiles of tm rows of x and tn of W
    auto groups = [&](int tm, int tn) { return (int64_t)((a.w.rows + tn - 1) / tn) * tiles_of(a, tm); };
    constexpr int TN = UP ? 64 : 128;  // rows of W of a workgroup four wide
    if constexpr (sizeof(T) == 4) {
        if (sorted) {
            if (groups(16, TN) <= 5 * kCUs / 4) return launch_tiles_of<T, G, UP, 2, 1, 1, 4, 2>(a, s);
            if (groups(16, TN) <= 5 * kCUs / 2) return launch_tiles_of<T, G, UP, 2, 1, 2, 2, 2>(a, s);
            if (per <= 16) return launch_tiles_of<T, G, UP, 2, 1, 4, 1, 2>(a, s);
            return launch_tiles_of<T, G, UP, 2, 2, 4, 1, 2>(a, s);
        }
        if (groups(16, TN / 4) <= kCUs) return launch_tiles_of<T, G, UP, 2, 1, 1, 8, 2>(a, s);
        if (groups(16, TN / 2) <= kCUs) return launch_tiles_of<T, G, UP, 2, 1, 2, 4, 2>(a, s);
        if (groups(32, TN / 2) <= kCUs) return launch_tiles_of<T, G, UP, 2, 2, 2, 4, 2>(a, s);
        if (groups(32, TN) <= kCUs) return launch_tiles_of<T, G, UP, 2, 2, 4, 2, 2>(a, s);
        return launch_tiles_of<T, G, UP, 2, 2, 4, 1, 2>(a, s);
    } else {
        if (sorted) {
            if (groups(16, TN) <= kCUs / 2) return launch_tiles_of<T, G, UP, P, 1, 2, 4, 2>(a, s);
            if (groups(16, TN) <= 2 * kCUs) return launch_flow_of<T, G, UP, 1, 4, 2, 4>(a, s);
            return per <= 24 ? launch_flow_of<T, G, UP, 2, 4, 1, 4>(a, s) : launch_flow_of<T, G, UP, 4, 4, 1, 3>(a, s);
        }
        if (per <= 16)
            return groups(16, 16) <= 3 * kCUs ? launch_tiles_of<T, G, UP, P, 1, 1, 8, 2>(a, s)
                                              : launch_tiles_of<T, G, UP, P, 1, 2, 4, 2>(a, s);
        if (groups(16, TN / 4) <= 2 * kCUs) return launch_tiles_of<T, G, UP, 2, 1, 1, 8, 2>(a, s);
        if (groups(16, TN) <= kCUs) return launch_flow_of<T, G, UP, 1, 4, 4, 4>(a, s);
        if (groups(32, TN) <= kCUs) return launch_flow_of<T, G, UP, 2, 4, 4, 4>(a, s);
        if (groups(64, TN) <= kCUs) return launch_flow_of<T, G, UP, 4, 4, 2, 2>(a, s);
        return launch_flow_of<T, G, UP, 4, 4, 1, 3>(a, s);
    }
}

template <typename T>
hipError_t launch_tiles_typed(const Q4Args &a, hipStream_t s) {
    const bool up = a.up.codes != nullptr;
    switch (a.w.group) {
        case 32: return up ? launch_tiles_sized<T, 32, true>(a, s) : launch_tiles_sized<T, 32, false>(a, s);
        case 64: return up ? launch_tiles_sized<T, 64, true>(a, s) : launch_tiles_sized<T, 64, false>(a, s);
        default: return up ? launch_tiles_sized<T, 128, true>(a, s) : launch_tiles_sized<T, 128, false>(a, s);
    }
}

}  // namespace hoard

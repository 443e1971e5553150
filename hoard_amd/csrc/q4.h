// Pieces shared by the kernels of the 4-bit products.
#pragma once

#include "ops.h"
#include "opsdev.h"

namespace hoard {

typedef bf16 v2bf __attribute__((ext_vector_type(2)));
typedef f16 v2h __attribute__((ext_vector_type(2)));
typedef bf16 v8bf __attribute__((ext_vector_type(8)));
typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// Codes as 16 + code in 16-bit floats: a code placed in the high fraction bits of
// 16.0 adds exactly itself, so eight codes cost four shifts and four masked ors.
// The sum over a group is then (sum of (16 + code) x) - (16 + zero) (sum of x),
// whose terms are at most some five times the plain ones'.  Word j of the result
// holds elements j (low) and j + 4 (high): x is laid out the same way (paired).
template <typename T>
struct Biased;
template <>
struct Biased<bf16> {
    static constexpr uint32_t base = 0x41804180u, mask = 0x00780078u;
    static constexpr int shift = 3;  // 16.0 has steps of 1/8
};
template <>
struct Biased<f16> {
    static constexpr uint32_t base = 0x4c004c00u, mask = 0x03c003c0u;
    static constexpr int shift = 6;  // steps of 1/64
};
template <typename T>
__device__ __forceinline__ v4u biased(uint32_t codes) {
    typedef Biased<T> B;
    // in a register the compiler cannot see through: the masked or is then one
    // instruction (v_and_or_b32 takes no two constants), not two
    uint32_t base = B::base;
    asm("" : "+v"(base));
    v4u o;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int s = B::shift - 4 * j;
        o[j] = ((s >= 0 ? codes << (s > 0 ? s : 0) : codes >> (s < 0 ? -s : 0)) & B::mask) | base;
    }
    return o;
}

// Codes plus kInOrderBias in their own order, words {0, 1}, {2, 3}, {4, 5}, {6, 7}, for x
// that is not rearranged.  f16: the code in the lowest fraction bits of 1024, so that a
// byte permute and a masked or make a word; the sum is taken off exactly (less).  bf16:
// half a byte is the 8-bit float of code * 2^-9 (4 exponent bits, the lowest of which is
// the code's fourth bit), which one conversion to bf16 takes two at a time.  There is no
// offset to correct: sums of 128 + code, at the same cost, lost four bits to it, and
// 0.36 % of a prompt's results fell to the other side of their bf16 rounding (now 0.015).
template <typename T>
constexpr float kInOrderBias = __is_same(T, bf16) ? 0.0f : 1024.0f;
template <typename T>
__device__ __forceinline__ v4u in_order(uint32_t codes) {
    const uint32_t high = codes >> 4;
    v4u o;
    if constexpr (__is_same(T, bf16)) {
        const uint32_t front = __builtin_amdgcn_perm(high, codes, 0x05010400u) & 0x0f0f0f0fu;
        const uint32_t back = __builtin_amdgcn_perm(high, codes, 0x07030602u) & 0x0f0f0f0fu;
        o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(front, 512.0f, false));
        o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(front, 512.0f, true));
        o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(back, 512.0f, false));
        o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(back, 512.0f, true));
    } else {
        uint32_t base = 0x64006400u;
        asm("" : "+v"(base));
#pragma unroll
        for (int j = 0; j < 4; j++)  // byte j of both into the two halves; the upper nibbles are masked off
            o[j] = (__builtin_amdgcn_perm(high, codes, 0x0c040c00u + 0x00010001u * j) & 0x000f000fu) | base;
    }
    return o;
}

// Eight consecutive 16-bit values as words {0, 4}, {1, 5}, {2, 6}, {3, 7}.
__device__ __forceinline__ v4u paired(v4u x) {
    v4u o;
    o[0] = __builtin_amdgcn_perm(x[2], x[0], 0x05040100u);
    o[1] = __builtin_amdgcn_perm(x[2], x[0], 0x07060302u);
    o[2] = __builtin_amdgcn_perm(x[3], x[1], 0x05040100u);
    o[3] = __builtin_amdgcn_perm(x[3], x[1], 0x07060302u);
    return o;
}

// s + the products of two pairs of values; a pair of ones.
template <typename T>
__device__ __forceinline__ float dot2(uint32_t w, uint32_t x, float s) {
    if constexpr (__is_same(T, bf16))
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w), __builtin_bit_cast(v2bf, x), s, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, x), s, false);
}
template <typename T>
constexpr uint32_t kOnes = __is_same(T, bf16) ? 0x3f803f80u : 0x3c003c00u;

// A scale as it is stored, and its value.
__device__ __forceinline__ uint32_t raw_scale(const hoard_q4_matrix &m, size_t i) {
    if (m.scale_type == HOARD_TYPE_F32) return static_cast<const uint32_t *>(m.scales)[i];
    return static_cast<const uint16_t *>(m.scales)[i];
}
__device__ __forceinline__ float scale_of(int type, uint32_t raw) {
    if (type == HOARD_TYPE_F32) return __uint_as_float(raw);
    if (type == HOARD_TYPE_BF16) return __uint_as_float(raw << 16);
    return (float)__builtin_bit_cast(f16, (uint16_t)raw);
}

// The matrix of row r of a call without offsets, or -1.
__device__ __forceinline__ int matrix_of(const Q4Args &a, int r) {
    if (a.mode == kQ4One) return 0;
    const int e = a.sel[r];
    return e < 0 || e >= a.w.n_mat ? -1 : e;
}

// g / (1 + e^-g) * u.  Where the result is rounded to 16 bits, with the exponential of
// 2 and the reciprocal of one instruction each (1 step of 32 bits; the product with
// log2 e adds at most 2^-24 |g| of it, g being at most some 100 where e^-g counts).  The
// reciprocal has no subnormal results, and 1 + e^-g goes up to 2^128: it is taken of a
// sixteenth.
template <typename T>
__device__ __forceinline__ float silu_mul(float g, float u) {
    if constexpr (sizeof(T) == 2) {
        const float e = __builtin_amdgcn_exp2f(g * -1.44269504f);
        return g * (__builtin_amdgcn_rcpf((1.0f + e) * 0.0625f) * 0.0625f) * u;
    }
    return g / (1.0f + expf(-g)) * u;
}

// Matrix tiles (q4_tiles.h), by the activations' type.
hipError_t launch_q4_tiles_f32(const Q4Args &a, hipStream_t s);
hipError_t launch_q4_tiles_f16(const Q4Args &a, hipStream_t s);
hipError_t launch_q4_tiles_bf16(const Q4Args &a, hipStream_t s);

}  // namespace hoard

// Device pieces shared by the operators of include/hoard_ops.h: activation
// types, eight values at a time at any element alignment, workgroup sums.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.h"

namespace hoard {

typedef _Float16 f16;
typedef __bf16 bf16;

// Sixteen bytes at any 2-byte aligned address: gfx950 loads and stores them from
// there, so rows of an odd length take the same path.
typedef uint32_t u128 __attribute__((ext_vector_type(4), aligned(2)));

// Eight values of T at p as floats.  NT: with the non-temporal policy, for what is
// read or written once and would only push other data out of the caches.
template <bool NT = false, typename T>
__device__ __forceinline__ void load8(const T *p, float o[8]) {
    T v[8];
#pragma unroll
    for (int i = 0; i < (int)sizeof v / 16; i++) {
        const u128 *from = reinterpret_cast<const u128 *>(p) + i;
        const u128 w = NT ? __builtin_nontemporal_load(from) : *from;
        __builtin_memcpy(reinterpret_cast<char *>(v) + 16 * i, &w, 16);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (float)v[i];
}
// Stored values are rounded to nearest, ties to even, once.
template <bool NT = false, typename T>
__device__ __forceinline__ void store8(T *p, const float o[8]) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (T)o[i];
#pragma unroll
    for (int i = 0; i < (int)sizeof v / 16; i++) {
        u128 w, *to = reinterpret_cast<u128 *>(p) + i;
        __builtin_memcpy(&w, reinterpret_cast<const char *>(v) + 16 * i, 16);
        if (NT) __builtin_nontemporal_store(w, to);
        else *to = w;
    }
}
// The first `some` of them; the rest of o is zero.
template <bool NT = false, typename T>
__device__ __forceinline__ void load_some(const T *p, int some, float o[8]) {
    if (some >= 8) return load8<NT>(p, o);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = i < some ? (float)p[i] : 0.0f;
}
template <bool NT = false, typename T>
__device__ __forceinline__ void store_some(T *p, int some, const float o[8]) {
    if (some >= 8) return store8<NT>(p, o);
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < some) p[i] = (T)o[i];
}

// Sum over the wave's 64 lanes, in every lane, in a fixed order.
__device__ __forceinline__ float wave_sum_f(float v) {
    v += dpp_f<kDppQuadXor1>(v);
    v += dpp_f<kDppQuadXor2>(v);
    v += dpp_f<kDppRowHalfMirror>(v);
    v += dpp_f<kDppRowMirror>(v);
    return (readlane_f(v, 0) + readlane_f(v, 16)) + (readlane_f(v, 32) + readlane_f(v, 48));
}

// Sum over a workgroup of WAVES waves, in every thread.  `part` is LDS of WAVES
// words that no other sum between two barriers uses.
template <int WAVES>
__device__ __forceinline__ float group_sum(float v, float *part) {
    v = wave_sum_f(v);
    if (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) part[wave_index()] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; i++) s += part[i];
    return s;
}

}  // namespace hoard

// Device pieces shared by the operators of include/hoard_ops.h: activation
// types, eight values at a time at any element alignment, workgroup sums.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wave.h"

namespace hoard {

typedef _Float16 f16;
typedef __bf16 bf16;

// Eight values of T at p as floats.  p is aligned to T only: gfx950 loads 16
// bytes from any address, so rows of an odd length take the same path.
template <typename T>
struct Pack8 {
    T v[8];
};
template <typename T>
__device__ __forceinline__ void load8(const T *p, float o[8]) {
    Pack8<T> t;
    __builtin_memcpy(&t, p, sizeof t);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (float)t.v[i];
}
// Stored values are rounded to nearest, ties to even, once.
template <typename T>
__device__ __forceinline__ void store8(T *p, const float o[8]) {
    Pack8<T> t;
#pragma unroll
    for (int i = 0; i < 8; i++) t.v[i] = (T)o[i];
    __builtin_memcpy(p, &t, sizeof t);
}
// The first `some` of them; the rest of o is zero.
template <typename T>
__device__ __forceinline__ void load_some(const T *p, int some, float o[8]) {
    if (some >= 8) return load8(p, o);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = i < some ? (float)p[i] : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_some(T *p, int some, const float o[8]) {
    if (some >= 8) return store8(p, o);
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

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

// Eight columns of a row of n, at .. at + 7, of which those from at + lo on are the
// thread's.  A row whose length is no multiple of 8 ends in columns that overlap the
// ones before (lo > 0); a thread behind the end has none (lo 8).  So no load stands
// under a condition: loads of many rows and arrays are in flight together.
struct Cols {
    int at, lo;
};
__device__ __forceinline__ Cols cols_of(int first, int n) {
    const int last = max(n - 8, 0);
    return first < n ? Cols{min(first, last), first - min(first, last)} : Cols{last, 8};
}

// Eight values as they lie in memory.
template <typename T>
struct Raw {
    u128 w[sizeof(T) / 2];
};
// NT: with the non-temporal policy, for what is read or written once and would only
// push other data out of the caches.
template <bool NT = false, typename T>
__device__ __forceinline__ Raw<T> fetch(const T *row, Cols c, int n) {
    Raw<T> r;
    if (n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const u128 *from = reinterpret_cast<const u128 *>(row + c.at) + i;
            r.w[i] = NT ? __builtin_nontemporal_load(from) : *from;
        }
    } else {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? row[i] : (T)0.0f;
        __builtin_memcpy(&r, v, sizeof r);
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void widen(const Raw<T> &r, float o[8]) {
    T v[8];
    __builtin_memcpy(v, &r, sizeof v);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (float)v[i];
}
// Zero in the columns that are not the thread's, for sums.
__device__ __forceinline__ void mask_cols(Cols c, float o[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = i >= c.lo ? o[i] : 0.0f;
}
// The thread's columns, rounded to nearest, ties to even, once.
template <bool NT = false, typename T>
__device__ __forceinline__ void put(T *row, Cols c, int n, const float o[8]) {
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (T)o[i];
    if (c.lo == 0 && n >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof v / 16; i++) {
            u128 w, *to = reinterpret_cast<u128 *>(row + c.at) + i;
            __builtin_memcpy(&w, reinterpret_cast<const char *>(v) + 16 * i, 16);
            if (NT) __builtin_nontemporal_store(w, to);
            else *to = w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i >= c.lo && i < n) row[c.at + i] = v[i];
    }
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

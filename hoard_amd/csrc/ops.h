// Internal launch interface between the operators' C ABI (ops.cpp) and their
// kernels.  Arguments are checked by ops.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "hoard_ops.h"

namespace hoard {

// How the rows of a 4-bit product find their matrix.
constexpr int kQ4One = 0;     // matrix 0
constexpr int kQ4Ids = 1;     // matrix sel[r]
constexpr int kQ4Sorted = 2;  // the matrix e with sel[e] <= r < sel[e + 1]

struct Q4Args {
    hoard_q4_matrix w, up;  // up.codes NULL: no second matrix
    int mode, type, n_rows, x_share;
    const void *x;
    const int32_t *sel;
    void *y;
    // matrix tiles, set by their launch: its first tile of rows of x, and whether the
    // workgroups of a tile go to one XCD
    int64_t tile0;
    bool spread;
};
hipError_t launch_q4(const Q4Args &a, hipStream_t s);

struct PairsArgs {
    int n_tokens, k, n_expert;
    const int32_t *ids;
    int32_t *place, *order, *offsets;
    int32_t *work;
};
size_t sort_work_bytes(int64_t pairs, int n_expert);
hipError_t launch_sort_pairs(const PairsArgs &a, hipStream_t s);

struct RowsArgs {
    int type, n_tokens, k, n;
    const void *x;         // gather: x; combine: y; combine_grad: y
    const int32_t *place;
    const float *w;        // or NULL: ones
    const void *res;       // combine: res or NULL; combine_grad: dout
    void *out;             // gather: xs; combine: out; combine_grad: dy or NULL
    float *dw;
};
hipError_t launch_gather(const RowsArgs &a, hipStream_t s);
hipError_t launch_combine(const RowsArgs &a, hipStream_t s);
hipError_t launch_combine_grad(const RowsArgs &a, hipStream_t s);

constexpr int kNormMaxN = 16384;
hipError_t launch_norm(const hoard_norm_args &a, hipStream_t s);
// Groups of rows whose partial sums the workspace holds.
int norm_groups(int n_rows, int n);
hipError_t launch_norm_grad(const hoard_norm_args &a, const hoard_norm_grads &g, float *work, hipStream_t s);

}  // namespace hoard

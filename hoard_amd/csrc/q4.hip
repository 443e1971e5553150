// Products with 4-bit weights and group scales (hoard_q4_matmul*).
//
// y[r][n] = sum over groups of scale[n][g] * sum over k in g of
// (code[n][k] - zero[n][g]) x[r][k]; with a second matrix silu(y) * y_up.
#include "ops.h"
#include "opsdev.h"

namespace hoard {

namespace {

__device__ __forceinline__ float scale_at(const hoard_q4_matrix &m, size_t i) {
    if (m.scale_type == HOARD_TYPE_F32) return static_cast<const float *>(m.scales)[i];
    if (m.scale_type == HOARD_TYPE_F16) return (float)static_cast<const f16 *>(m.scales)[i];
    return (float)static_cast<const bf16 *>(m.scales)[i];
}

// The matrix of row r, or -1.
__device__ __forceinline__ int matrix_of(const Q4Args &a, int r) {
    if (a.mode == kQ4One) return 0;
    if (a.mode == kQ4Ids) {
        const int e = a.sel[r];
        return e < 0 || e >= a.w.n_mat ? -1 : e;
    }
    // the last e with sel[e] <= r
    int lo = 0, hi = a.w.n_mat;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.sel[mid] <= r) lo = mid;
        else hi = mid;
    }
    return a.sel[lo] <= r && r < a.sel[lo + 1] ? lo : -1;
}

// One row of m times one row of x, by a wave; every lane gets it.
template <typename T>
__device__ __forceinline__ float dot_row(const hoard_q4_matrix &m, size_t row, const T *x) {
    const int lane = threadIdx.x & 63, groups = m.cols / m.group;
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(m.codes) + row * (m.cols / 2));
    float s = 0.0f;
    for (int at = lane * 8; at < m.cols; at += 512) {
        float v[8], g = 0.0f;
        load8(x + at, v);
        const uint32_t c = codes[at / 8];
        const size_t gi = row * groups + at / m.group;
        const float z = m.zeros ? (float)m.zeros[gi] : 8.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) g = fmaf((float)((c >> (4 * i)) & 15u) - z, v[i], g);
        s = fmaf(scale_at(m, gi), g, s);
    }
    return wave_sum_f(s);
}

// A wave takes one output.
template <typename T>
__global__ __launch_bounds__(256) void q4_kernel(Q4Args a) {
    const int n = blockIdx.x * 4 + wave_index();
    if (n >= a.w.rows) return;
    for (int r = blockIdx.y; r < a.n_rows; r += gridDim.y) {
        const int e = matrix_of(a, r);
        float y = __builtin_nanf("");
        if (e >= 0) {
            const T *x = static_cast<const T *>(a.x) + (size_t)(r / a.x_share) * a.w.cols;
            const size_t row = (size_t)e * a.w.rows + n;
            y = dot_row(a.w, row, x);
            if (a.up.codes) y = y / (1.0f + expf(-y)) * dot_row(a.up, row, x);
        } else if (a.mode == kQ4Sorted) {
            continue;
        }
        if ((threadIdx.x & 63) == 0) static_cast<T *>(a.y)[(size_t)r * a.w.rows + n] = (T)y;
    }
}

}  // namespace

hipError_t launch_q4(const Q4Args &a, hipStream_t s) {
    if (!a.n_rows) return hipSuccess;
    const dim3 grid((a.w.rows + 3) / 4, a.n_rows < 65535 ? a.n_rows : 65535);
    if (a.type == HOARD_TYPE_F32) q4_kernel<float><<<grid, 256, 0, s>>>(a);
    else if (a.type == HOARD_TYPE_F16) q4_kernel<f16><<<grid, 256, 0, s>>>(a);
    else q4_kernel<bf16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace hoard

// Products with 4-bit weights and group scales (hoard_q4_matmul*).
//
// y[r][n] = sum over groups of scale[n][g] * sum over k in g of
// (code[n][k] - zero[n][g]) x[r][k]; with a second matrix silu(y) * y_up.
//
// One row of x, or a few: dots (below).  More: matrix tiles (q4_tiles.h).
#include "q4.h"

namespace hoard {

namespace {

// 32 values of a row of x against 32 codes: laid out once for all rows of W.
template <typename T>
struct Slice {  // 16-bit types: words of two values in the order of biased()
    v4u x[4];
    float sum;
    __device__ __forceinline__ void load(const T *p) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const v4u w = reinterpret_cast<const v4u *>(p)[i];
#pragma unroll
            for (int c = 0; c < 4; c++) sum = dot2<T>(w[c], kOnes<T>, sum);
            x[i] = paired(w);
        }
    }
};
template <>
struct Slice<float> {
    float x[32];
    float sum;
    __device__ __forceinline__ void load(const float *p) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const v4f w = reinterpret_cast<const v4f *>(p)[i];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                x[4 * i + c] = w[c];
                sum += w[c];
            }
        }
    }
};

// Sum over k of (code - zero) x for the lane's 32 columns of R rows of x.
template <typename T, int R>
__device__ __forceinline__ void dots(v4u codes, float zero, const Slice<T> (&x)[R], float (&d)[R]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int r = 0; r < R; r++) d[r] = -(16.0f + zero) * x[r].sum;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const v4u w = biased<T>(codes[i]);
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int j = 0; j < 4; j++) d[r] = dot2<T>(w[j], x[r].x[i][j], d[r]);
        }
    } else {
        // a byte of a masked word converts in one instruction
#pragma unroll
        for (int r = 0; r < R; r++) d[r] = -zero * x[r].sum;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t even = codes[i] & 0x0f0f0f0fu, odd = (codes[i] >> 4) & 0x0f0f0f0fu;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float w0 = (float)((even >> (8 * j)) & 0xffu), w1 = (float)((odd >> (8 * j)) & 0xffu);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    d[r] = fmaf(w0, x[r].x[8 * i + 2 * j], d[r]);
                    d[r] = fmaf(w1, x[r].x[8 * i + 2 * j + 1], d[r]);
                }
            }
        }
    }
}

// A wave takes NR rows of W per run of 2^lanes_log lanes; the run's lanes split the
// columns, 32 consecutive ones (16 bytes of codes) at a time.  R rows of x.
template <typename T, int R, bool UP, int NR>
__global__ __launch_bounds__(256) void q4_rows_kernel(Q4Args a, int lanes_log) {
    constexpr int P = UP ? 2 : 1;
    const int lane = threadIdx.x & 63, run = lane >> lanes_log, lk = lane & ((1 << lanes_log) - 1);
    const int n0 = (int)(((int64_t)blockIdx.x * 4 + wave_index()) << (6 - lanes_log)) * NR + run * NR;
    const int cols = a.w.cols, groups = cols / a.w.group, group_log = __ffs(a.w.group) - 1;
    for (int r0 = blockIdx.y * R; r0 < a.n_rows; r0 += gridDim.y * R) {
        const int e = matrix_of(a, r0);  // R is 1 where rows differ in their matrix
        float acc[P][NR][R] = {};
        if (e >= 0) {
            const T *x[R];
#pragma unroll
            for (int r = 0; r < R; r++)
                x[r] = static_cast<const T *>(a.x) + (size_t)(min(r0 + r, a.n_rows - 1) / a.x_share) * cols;
            size_t row[NR];
#pragma unroll
            for (int j = 0; j < NR; j++) row[j] = (size_t)e * a.w.rows + min(n0 + j, a.w.rows - 1);
            for (int k = lk * 32; k < cols; k += 32 << lanes_log) {
                v4u codes[P][NR];
                uint32_t scale[P][NR], zero[P][NR];
#pragma unroll
                for (int p = 0; p < P; p++) {
                    const hoard_q4_matrix &m = p ? a.up : a.w;
#pragma unroll
                    for (int j = 0; j < NR; j++) {
                        codes[p][j] = *reinterpret_cast<const v4u *>(static_cast<const uint8_t *>(m.codes) +
                                                                     row[j] * (cols / 2) + k / 2);
                        const size_t gi = row[j] * groups + (k >> group_log);
                        scale[p][j] = raw_scale(m, gi, 0);
                        zero[p][j] = m.zeros ? m.zeros[gi] : 8;
                    }
                }
                Slice<T> xs[R];
#pragma unroll
                for (int r = 0; r < R; r++) xs[r].load(x[r] + k);
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int j = 0; j < NR; j++) {
                        float d[R];
                        dots<T, R>(codes[p][j], (float)zero[p][j], xs, d);
                        const float s = scale_of(p ? a.up.scale_type : a.w.scale_type, scale[p][j]);
#pragma unroll
                        for (int r = 0; r < R; r++) acc[p][j][r] = fmaf(s, d[r], acc[p][j][r]);
                    }
            }
        }
        // the run's lanes added up; lane j of the run then stores row j
#pragma unroll
        for (int r = 0; r < R; r++) {
            float mine[P] = {};
#pragma unroll
            for (int p = 0; p < P; p++)
#pragma unroll
                for (int j = 0; j < NR; j++) {
                    float v = acc[p][j][r];
                    v += dpp_f<kDppQuadXor1>(v);
                    v += dpp_f<kDppQuadXor2>(v);
                    v += dpp_f<kDppRowHalfMirror>(v);
                    if (lanes_log >= 4) v += dpp_f<kDppRowMirror>(v);
                    if (lanes_log >= 5) v += __shfl_xor(v, 16);
                    if (lanes_log >= 6) v += __shfl_xor(v, 32);
                    if (lk == j) mine[p] = v;
                }
            if (lk < NR && n0 + lk < a.w.rows && r0 + r < a.n_rows) {
                float v = UP ? silu_mul<T>(mine[0], mine[P - 1]) : mine[0];
                if (e < 0) v = __builtin_nanf("");
                static_cast<T *>(a.y)[(size_t)(r0 + r) * a.w.rows + n0 + lk] = (T)v;
            }
        }
    }
}

template <typename T, int R, bool UP, int NR>
hipError_t launch_rows_of(const Q4Args &a, hipStream_t s) {
    int lanes_log = 3;
    while (lanes_log < 6 && (32 << lanes_log) < a.w.cols) lanes_log++;
    const int64_t per = (int64_t)4 * NR << (6 - lanes_log), y = ((int64_t)a.n_rows + R - 1) / R;
    const dim3 grid((unsigned)((a.w.rows + per - 1) / per), (unsigned)(y < 65535 ? y : 65535));
    q4_rows_kernel<T, R, UP, NR><<<grid, 256, 0, s>>>(a, lanes_log);
    return hipGetLastError();
}

template <typename T, int R>
hipError_t launch_rows_sized(const Q4Args &a, hipStream_t s) {
    const bool many = (int64_t)a.w.rows * ((a.n_rows + R - 1) / R) >= 8192;
    if (a.up.codes) return many ? launch_rows_of<T, R, true, 4>(a, s) : launch_rows_of<T, R, true, 1>(a, s);
    return many ? launch_rows_of<T, R, false, 8>(a, s) : launch_rows_of<T, R, false, 2>(a, s);
}

template <typename T>
hipError_t launch_rows(const Q4Args &a, hipStream_t s) {
    if (a.mode == kQ4Ids || a.n_rows == 1) return launch_rows_sized<T, 1>(a, s);
    if (a.n_rows == 2) return launch_rows_sized<T, 2>(a, s);
    return launch_rows_sized<T, 4>(a, s);
}

}  // namespace

hipError_t launch_q4(const Q4Args &a, hipStream_t s) {
    if (!a.n_rows) return hipSuccess;
    const bool few = a.mode == kQ4Ids || (a.mode == kQ4One && a.n_rows <= 4);
    if (a.type == HOARD_TYPE_F32) return few ? launch_rows<float>(a, s) : launch_q4_tiles_f32(a, s);
    if (a.type == HOARD_TYPE_F16) return few ? launch_rows<f16>(a, s) : launch_q4_tiles_f16(a, s);
    return few ? launch_rows<bf16>(a, s) : launch_q4_tiles_bf16(a, s);
}

}  // namespace hoard

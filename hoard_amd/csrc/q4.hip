// Products with 4-bit weights and group scales (hoard_q4_matmul*).
//
// y[r][n] = sum over groups of scale[n][g] * sum over k in g of
// (code[n][k] - zero[n][g]) x[r][k]; with a second matrix silu(y) * y_up.
//
// One row of x, or rows with a matrix each: dots (below).  More: tiles (q4_tiles.h).
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
    __device__ __forceinline__ void load(const float *p) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const v4f w = reinterpret_cast<const v4f *>(p)[i];
#pragma unroll
            for (int c = 0; c < 4; c++) x[4 * i + c] = w[c];
        }
    }
};

// Sum over k of (code - zero) x for the lane's 32 columns.
template <typename T>
__device__ __forceinline__ float dots(v4u codes, float zero, const Slice<T> &x) {
    float d;
    if constexpr (sizeof(T) == 2) {
        d = -(16.0f + zero) * x.sum;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const v4u w = biased<T>(codes[i]);
#pragma unroll
            for (int j = 0; j < 4; j++) d = dot2<T>(w[j], x.x[i][j], d);
        }
    } else {
        // a byte of a masked word converts in one instruction; less its zero point it is
        // exact, and the terms' sum needs no correction (which cost digits, not time)
        d = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t even = codes[i] & 0x0f0f0f0fu, odd = (codes[i] >> 4) & 0x0f0f0f0fu;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                d = fmaf((float)((even >> (8 * j)) & 0xffu) - zero, x.x[8 * i + 2 * j], d);
                d = fmaf((float)((odd >> (8 * j)) & 0xffu) - zero, x.x[8 * i + 2 * j + 1], d);
            }
        }
    }
    return d;
}

// A row of x at a time.  A wave takes NR rows of W per run of 2^lanes_log lanes; the
// run's lanes split the columns, 32 consecutive ones (16 bytes of codes) at a time.
//
// Bound by memory, and below a few MB of codes by its latency: two rows of W a wave
// keep enough waves in flight (16384 x 8192 in bf16: 15.9 us with 2 rows, 18.1 with 4,
// 19.3 with 8, 21.5 with 1; 8 experts' 768 x 2048 twice in fp32: 8.4 with 2, 9.2 with 4,
// 9.9 with 1).  In fp32 a row of x is four times its codes, and from 4096 rows of W on
// four rows a wave that share it are faster (8192 x 8192: 13.8 against 18.6; 512 x 2048:
// 5.2 against 4.4).  x goes from the caches to registers: through LDS, shared by the
// four waves, 16384 x 8192 took 18.1 and the 8 experts 10.3.
template <typename T, bool UP, int NR>
__global__ __launch_bounds__(256) void q4_rows_kernel(Q4Args a, int lanes_log) {
    constexpr int P = UP ? 2 : 1;
    const int lane = threadIdx.x & 63, run = lane >> lanes_log, lk = lane & ((1 << lanes_log) - 1);
    const int64_t at = (((int64_t)blockIdx.x * 4 + wave_index()) << (6 - lanes_log)) * NR + run * NR;
    const int n0 = (int)min(at, (int64_t)a.w.rows);
    const int cols = a.w.cols, groups = cols / a.w.group, group_log = __ffs(a.w.group) - 1;
    for (int64_t r = blockIdx.y; r < a.n_rows; r += gridDim.y) {
        const int e = matrix_of(a, (int)r);
        float acc[P][NR] = {};
        if (e >= 0) {
            const T *x = static_cast<const T *>(a.x) + (size_t)((int)r / a.x_share) * cols;
            size_t row[NR];  // clamped: what lies behind the last row is not stored
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
                        scale[p][j] = raw_scale(m, gi);
                        zero[p][j] = m.zeros ? m.zeros[gi] : 8;
                    }
                }
                Slice<T> xs;
                xs.load(x + k);
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int j = 0; j < NR; j++)
                        acc[p][j] = fmaf(scale_of(p ? a.up.scale_type : a.w.scale_type, scale[p][j]),
                                         dots(codes[p][j], (float)zero[p][j], xs), acc[p][j]);
            }
        }
        // the run's lanes added up; lane j of the run then stores row j
        float mine[P] = {};
#pragma unroll
        for (int p = 0; p < P; p++)
#pragma unroll
            for (int j = 0; j < NR; j++) {
                float v = acc[p][j];
                v += dpp_f<kDppQuadXor1>(v);
                v += dpp_f<kDppQuadXor2>(v);
                v += dpp_f<kDppRowHalfMirror>(v);
                if (lanes_log >= 4) v += dpp_f<kDppRowMirror>(v);
                if (lanes_log >= 5) v += __shfl_xor(v, 16);
                if (lanes_log >= 6) v += __shfl_xor(v, 32);
                if (lk == j) mine[p] = v;
            }
        if (lk < NR && n0 + lk < a.w.rows) {
            float v = UP ? silu_mul<T>(mine[0], mine[P - 1]) : mine[0];
            if (e < 0) v = __builtin_nanf("");
            static_cast<T *>(a.y)[(size_t)r * a.w.rows + n0 + lk] = (T)v;
        }
    }
}

template <typename T, bool UP, int NR>
hipError_t launch_rows_of(const Q4Args &a, hipStream_t s) {
    int lanes_log = 3;
    while (lanes_log < 6 && (32 << lanes_log) < a.w.cols) lanes_log++;
    const int64_t per = (int64_t)4 * NR << (6 - lanes_log);
    const dim3 grid((unsigned)((a.w.rows + per - 1) / per), (unsigned)(a.n_rows < 65535 ? a.n_rows : 65535));
    q4_rows_kernel<T, UP, NR><<<grid, 256, 0, s>>>(a, lanes_log);
    return hipGetLastError();
}
template <typename T>
hipError_t launch_rows(const Q4Args &a, hipStream_t s) {
    if (a.up.codes) return launch_rows_of<T, true, 2>(a, s);
    if (sizeof(T) == 4 && (int64_t)a.w.rows * a.n_rows >= 4096) return launch_rows_of<T, false, 4>(a, s);
    return launch_rows_of<T, false, 2>(a, s);
}

}  // namespace

hipError_t launch_q4(const Q4Args &a, hipStream_t s) {
    if (!a.n_rows) return hipSuccess;
    // A matrix instruction takes 16 rows of x for what two cost by dots (16384 x 8192,
    // bf16: 24.4 us by tiles for 2 to 4 rows; by dots 15.9 for 1, 23.5 for 2, 37.8 for 4;
    // 4096 x 4096 in fp32: 9.1 against 10.6 for 2, 19.7 for 4).
    const bool few = a.mode == kQ4Ids || (a.mode == kQ4One && a.n_rows == 1);
    if (a.type == HOARD_TYPE_F32) return few ? launch_rows<float>(a, s) : launch_q4_tiles_f32(a, s);
    if (a.type == HOARD_TYPE_F16) return few ? launch_rows<f16>(a, s) : launch_q4_tiles_f16(a, s);
    return few ? launch_rows<bf16>(a, s) : launch_q4_tiles_bf16(a, s);
}

}  // namespace hoard

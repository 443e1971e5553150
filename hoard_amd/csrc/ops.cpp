// The C ABI of include/hoard_ops.h: argument checks, then one launch interface
// call (ops.h).  Nothing here allocates, keeps state or throws.
#include <hip/hip_runtime.h>

#include "hoard_ops.h"
#include "host_error.h"
#include "ops.h"

using hoard::fail_fmt;

namespace {

bool activation_type(int t) { return t == HOARD_TYPE_F32 || t == HOARD_TYPE_F16 || t == HOARD_TYPE_BF16; }
size_t type_size(int t) { return t == HOARD_TYPE_F32 ? 4 : 2; }
bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int kMaxRows = 1 << 22;  // a launch's workgroups of 16 rows by 8 tiles of x within its 2^32 threads
constexpr int kMaxCols = 1 << 20;  // 64 rows of x lie within the kernels' 32-bit offsets
constexpr int kMaxMats = 1 << 30;  // a lane's run of matrices, rounded up, ends within 32 bits
constexpr int kMaxN = 1 << 30;     // columns of the pairs' rows: a wave's step of 2048 past the last stays within 32 bits

int launched(const char *what, hipError_t rc) {
    if (rc == hipSuccess) {
        hoard_set_error(HOARD_OK, "");
        return HOARD_OK;
    }
    return fail_fmt(HOARD_ERR_HIP, "%s: %s", what, hipGetErrorString(rc));
}

int check_matrix(const char *what, const hoard_q4_matrix &m) {
    if (!m.codes || !m.scales) return fail_fmt(HOARD_ERR_INVALID, "%s: null codes or scales", what);
    if (!aligned(m.codes, 16)) return fail_fmt(HOARD_ERR_INVALID, "%s: codes are not 16-byte aligned", what);
    if (m.rows <= 0 || m.n_mat <= 0) return fail_fmt(HOARD_ERR_INVALID, "%s: rows %d, n_mat %d", what, m.rows, m.n_mat);
    if (m.n_mat > kMaxMats) return fail_fmt(HOARD_ERR_UNSUPPORTED, "%s: n_mat %d above %d", what, m.n_mat, kMaxMats);
    if (m.rows > kMaxRows) return fail_fmt(HOARD_ERR_UNSUPPORTED, "%s: rows %d above %d", what, m.rows, kMaxRows);
    if (m.group != 32 && m.group != 64 && m.group != 128)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "%s: group %d is not 32, 64 or 128", what, m.group);
    if (m.cols <= 0 || m.cols % m.group)
        return fail_fmt(HOARD_ERR_INVALID, "%s: cols %d not a positive multiple of group %d", what, m.cols, m.group);
    if (m.cols > kMaxCols) return fail_fmt(HOARD_ERR_UNSUPPORTED, "%s: cols %d above %d", what, m.cols, kMaxCols);
    if (!activation_type(m.scale_type))
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "%s: scale type %d", what, m.scale_type);
    if (!aligned(m.scales, type_size(m.scale_type)))
        return fail_fmt(HOARD_ERR_INVALID, "%s: scales are not aligned to their type", what);
    return 0;
}

int q4(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int mode, int type, int n_rows, const void *x,
       int x_share, const int32_t *sel, void *y, void *stream) {
    if (!w) return fail_fmt(HOARD_ERR_INVALID, "null matrix");
    if (int rc = check_matrix("w", *w)) return rc;
    if (up) {
        if (int rc = check_matrix("up", *up)) return rc;
        if (up->rows != w->rows || up->cols != w->cols || up->n_mat != w->n_mat || up->group != w->group)
            return fail_fmt(HOARD_ERR_INVALID, "up is %d x %d x %d in groups of %d beside %d x %d x %d of %d", up->n_mat,
                            up->rows, up->cols, up->group, w->n_mat, w->rows, w->cols, w->group);
    }
    if (mode == hoard::kQ4One && w->n_mat != 1) return fail_fmt(HOARD_ERR_INVALID, "n_mat %d without ids or offsets", w->n_mat);
    if (!activation_type(type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", type);
    if (n_rows < 0) return fail_fmt(HOARD_ERR_INVALID, "n_rows %d", n_rows);
    if (x_share <= 0 || n_rows % x_share)
        return fail_fmt(HOARD_ERR_INVALID, "x_share %d does not divide n_rows %d", x_share, n_rows);
    if (n_rows == 0) return launched("", hipSuccess);
    if (!x || !y || (mode != hoard::kQ4One && !sel)) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (!aligned(x, 16)) return fail_fmt(HOARD_ERR_INVALID, "x is not 16-byte aligned");
    if (!aligned(y, type_size(type)) || !aligned(sel, 4)) return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    hoard::Q4Args a{*w, up ? *up : hoard_q4_matrix{}, mode, type, n_rows, x_share, x, sel, y, 0, false};
    return launched("4-bit product", hoard::launch_q4(a, static_cast<hipStream_t>(stream)));
}

int check_pairs(int n_tokens, int k) {
    if (n_tokens < 0) return fail_fmt(HOARD_ERR_INVALID, "n_tokens %d", n_tokens);
    if (k < 1 || k > 64) return fail_fmt(HOARD_ERR_INVALID, "k %d outside 1..64", k);
    if ((int64_t)n_tokens * k > INT32_MAX) return fail_fmt(HOARD_ERR_INVALID, "%d * %d pairs", n_tokens, k);
    return 0;
}

int check_sort(int n_tokens, int k, int n_expert) {
    if (int rc = check_pairs(n_tokens, k)) return rc;
    if (n_expert < 1 || n_expert > 1024) return fail_fmt(HOARD_ERR_INVALID, "n_expert %d outside 1..1024", n_expert);
    return 0;
}

int check_rows(int type, int n_tokens, int k, int n) {
    if (!activation_type(type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", type);
    if (n < 1 || n > kMaxN) return fail_fmt(HOARD_ERR_INVALID, "n %d outside 1..%d", n, kMaxN);
    return check_pairs(n_tokens, k);
}

int check_norm(const hoard_norm_args &a) {
    if (!activation_type(a.type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", a.type);
    if (a.res_type != HOARD_TYPE_F32 && a.res_type != a.type)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "residual type %d beside type %d", a.res_type, a.type);
    if (a.gate_kind < HOARD_GATE_NONE || a.gate_kind > HOARD_GATE_FULL)
        return fail_fmt(HOARD_ERR_INVALID, "gate_kind %d", a.gate_kind);
    if (a.n_rows < 0) return fail_fmt(HOARD_ERR_INVALID, "n_rows %d", a.n_rows);
    if (a.n < 1 || a.n > hoard::kNormMaxN) return fail_fmt(HOARD_ERR_INVALID, "n %d outside 1..%d", a.n, hoard::kNormMaxN);
    if (!(a.eps > 0.0f)) return fail_fmt(HOARD_ERR_INVALID, "eps %g is not above 0", (double)a.eps);
    return 0;
}

int check_norm_pointers(const hoard_norm_args &a) {
    if (!a.b && (a.gate_kind != HOARD_GATE_NONE || a.w_post))
        return fail_fmt(HOARD_ERR_INVALID, "a gate or w_post without b");
    if ((a.gate_kind != HOARD_GATE_NONE) != (a.gate != nullptr))
        return fail_fmt(HOARD_ERR_INVALID, "gate pointer and gate_kind %d disagree", a.gate_kind);
    const size_t t = type_size(a.type), r = type_size(a.res_type);
    if (!aligned(a.b, t) || !aligned(a.h, t) || !aligned(a.r, r) || !aligned(a.r_out, r) || !aligned(a.w_post, 4) ||
        !aligned(a.w_pre, 4) || !aligned(a.stats, 4) || !aligned(a.gate, a.gate_kind == HOARD_GATE_FULL ? t : 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    return 0;
}

size_t norm_work_bytes(const hoard_norm_args &a) {
    return sizeof(float) * 3 * (size_t)a.n * hoard::norm_groups(a.n_rows, a.n);
}

}  // namespace

extern "C" {

int hoard_q4_matmul(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                    void *y, void *stream) {
    return q4(w, up, hoard::kQ4One, type, n_rows, x, 1, nullptr, y, stream);
}

int hoard_q4_matmul_ids(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                        int x_share, const int32_t *ids, void *y, void *stream) {
    return q4(w, up, hoard::kQ4Ids, type, n_rows, x, x_share, ids, y, stream);
}

int hoard_q4_matmul_sorted(const hoard_q4_matrix *w, const hoard_q4_matrix *up, int type, int n_rows, const void *x,
                           const int32_t *offsets, void *y, void *stream) {
    return q4(w, up, hoard::kQ4Sorted, type, n_rows, x, 1, offsets, y, stream);
}

int hoard_sort_workspace(int n_tokens, int k, int n_expert, size_t *bytes) {
    if (!bytes) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_sort(n_tokens, k, n_expert)) return rc;
    *bytes = hoard::sort_work_bytes((int64_t)n_tokens * k, n_expert);
    return launched("", hipSuccess);
}

int hoard_sort_pairs(int n_tokens, int k, int n_expert, const int32_t *ids, int32_t *place, int32_t *order,
                     int32_t *offsets, void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_sort(n_tokens, k, n_expert)) return rc;
    if (!offsets || (n_tokens && (!ids || !place || !order))) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (!aligned(ids, 4) || !aligned(place, 4) || !aligned(order, 4) || !aligned(offsets, 4) || !aligned(workspace, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    const size_t need = hoard::sort_work_bytes((int64_t)n_tokens * k, n_expert);
    if (need && (!workspace || workspace_bytes < need))
        return fail_fmt(HOARD_ERR_INVALID, "workspace of %zu bytes, %zu wanted", workspace ? workspace_bytes : 0, need);
    hoard::PairsArgs a{n_tokens, k, n_expert, ids, place, order, offsets, static_cast<int32_t *>(workspace)};
    return launched("sort", hoard::launch_sort_pairs(a, static_cast<hipStream_t>(stream)));
}

int hoard_sort_gather(int type, int n_tokens, int k, int n, const void *x, const int32_t *place, const float *w,
                      void *xs, void *stream) {
    if (int rc = check_rows(type, n_tokens, k, n)) return rc;
    if (n_tokens == 0) return launched("", hipSuccess);
    if (!x || !place || !xs) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    const size_t t = type_size(type);
    if (!aligned(x, t) || !aligned(xs, t) || !aligned(place, 4) || !aligned(w, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    hoard::RowsArgs a{type, n_tokens, k, n, x, place, w, nullptr, xs, nullptr};
    return launched("gather", hoard::launch_gather(a, static_cast<hipStream_t>(stream)));
}

int hoard_sort_combine(int type, int n_tokens, int k, int n, const void *y, const int32_t *place, const float *w,
                       const void *res, void *out, void *stream) {
    if (int rc = check_rows(type, n_tokens, k, n)) return rc;
    if (n_tokens == 0) return launched("", hipSuccess);
    if (!y || !place || !out) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    const size_t t = type_size(type);
    if (!aligned(y, t) || !aligned(res, t) || !aligned(out, t) || !aligned(place, 4) || !aligned(w, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    hoard::RowsArgs a{type, n_tokens, k, n, y, place, w, res, out, nullptr};
    return launched("combine", hoard::launch_combine(a, static_cast<hipStream_t>(stream)));
}

int hoard_sort_combine_grad(int type, int n_tokens, int k, int n, const void *dout, const void *y,
                            const int32_t *place, const float *w, void *dy, float *dw, void *stream) {
    if (int rc = check_rows(type, n_tokens, k, n)) return rc;
    if (n_tokens == 0) return launched("", hipSuccess);
    if (!dout || !y || !place || !w || !dw) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    const size_t t = type_size(type);
    if (!aligned(y, t) || !aligned(dout, t) || !aligned(dy, t) || !aligned(place, 4) || !aligned(w, 4) || !aligned(dw, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    hoard::RowsArgs a{type, n_tokens, k, n, y, place, w, dout, dy, dw};
    return launched("combine gradient", hoard::launch_combine_grad(a, static_cast<hipStream_t>(stream)));
}

int hoard_norm_forward(const hoard_norm_args *a, void *stream) {
    if (!a) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_norm(*a)) return rc;
    if (int rc = check_norm_pointers(*a)) return rc;
    if (!a->b && !a->h) return fail_fmt(HOARD_ERR_INVALID, "neither b nor h: nothing to do");
    if ((a->h != nullptr) != (a->w_pre != nullptr)) return fail_fmt(HOARD_ERR_INVALID, "h and w_pre go together");
    if ((a->b != nullptr) != (a->r_out != nullptr)) return fail_fmt(HOARD_ERR_INVALID, "b and r_out go together");
    if (!a->r && a->n_rows) return fail_fmt(HOARD_ERR_INVALID, "null residual");
    return launched("norm", hoard::launch_norm(*a, static_cast<hipStream_t>(stream)));
}

int hoard_norm_workspace(const hoard_norm_args *a, size_t *bytes) {
    if (!a || !bytes) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_norm(*a)) return rc;
    *bytes = norm_work_bytes(*a);
    return launched("", hipSuccess);
}

int hoard_norm_backward(const hoard_norm_args *a, const hoard_norm_grads *g, void *workspace, size_t workspace_bytes,
                        void *stream) {
    if (!a || !g) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_norm(*a)) return rc;
    if (int rc = check_norm_pointers(*a)) return rc;
    if (!g->dr_out && !g->dh) return fail_fmt(HOARD_ERR_INVALID, "neither dr_out nor dh");
    if (g->dh && (!a->w_pre || !a->r_out)) return fail_fmt(HOARD_ERR_INVALID, "dh without w_pre and r_out");
    if (g->dw_pre && !g->dh) return fail_fmt(HOARD_ERR_INVALID, "dw_pre without dh");
    if ((g->db || g->dw_post || g->dgate) && !a->b) return fail_fmt(HOARD_ERR_INVALID, "db, dw_post or dgate without b");
    if (g->dw_post && !a->w_post) return fail_fmt(HOARD_ERR_INVALID, "dw_post without w_post");
    if (g->dgate && a->gate_kind == HOARD_GATE_NONE) return fail_fmt(HOARD_ERR_INVALID, "dgate without a gate");
    if (!g->dr && !g->db && !g->dgate && !g->dw_post && !g->dw_pre) return fail_fmt(HOARD_ERR_INVALID, "no gradient wanted");
    if (!a->stats && a->n_rows) return fail_fmt(HOARD_ERR_INVALID, "null stats");
    const size_t t = type_size(a->type), r = type_size(a->res_type);
    if (!aligned(g->dr_out, r) || !aligned(g->dr, r) || !aligned(g->dh, t) || !aligned(g->db, t) || !aligned(g->dw_post, 4) ||
        !aligned(g->dw_pre, 4) || !aligned(g->dgate, a->gate_kind == HOARD_GATE_FULL ? t : 4) || !aligned(workspace, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    const size_t need = norm_work_bytes(*a);
    if (need && (!workspace || workspace_bytes < need))
        return fail_fmt(HOARD_ERR_INVALID, "workspace of %zu bytes, %zu wanted", workspace ? workspace_bytes : 0, need);
    return launched("norm gradient",
                    hoard::launch_norm_grad(*a, *g, static_cast<float *>(workspace), static_cast<hipStream_t>(stream)));
}

}  // extern "C"

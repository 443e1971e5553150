// The C ABI of include/hoard_attn.h: argument checks, then one launch interface call
// (attn.h).  Nothing here allocates, keeps state or throws.
#include <hip/hip_runtime.h>

#include "attn.h"
#include "hoard_attn.h"
#include "host_error.h"

using hoard::fail_fmt;

namespace {

bool activation_type(int t) { return t == HOARD_TYPE_F32 || t == HOARD_TYPE_F16 || t == HOARD_TYPE_BF16; }
size_t type_size(int t) { return t == HOARD_TYPE_F32 ? 4 : t == HOARD_TYPE_I8 ? 1 : 2; }
bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int kMaxHeads = 1024;
constexpr int kMaxDim = 256;
constexpr int kMaxNew = 64;

int launched(const char *what, hipError_t rc) {
    if (rc == hipSuccess) {
        hoard_set_error(HOARD_OK, "");
        return HOARD_OK;
    }
    return fail_fmt(HOARD_ERR_HIP, "%s: %s", what, hipGetErrorString(rc));
}

int check_cache(const hoard_kv_cache &c) {
    if (c.type != HOARD_TYPE_F16 && c.type != HOARD_TYPE_BF16 && c.type != HOARD_TYPE_I8)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "cache type %d", c.type);
    if (c.page < 16 || c.page > 256 || (c.page & (c.page - 1)))
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "page %d is not 16, 32, 64, 128 or 256", c.page);
    if (c.head_dim < 16 || c.head_dim > kMaxDim || c.head_dim % 16)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "cache head_dim %d is not a multiple of 16 up to %d", c.head_dim, kMaxDim);
    if (c.n_kv_heads < 1 || c.n_kv_heads > kMaxHeads)
        return fail_fmt(HOARD_ERR_INVALID, "n_kv_heads %d outside 1..%d", c.n_kv_heads, kMaxHeads);
    if (c.n_pages < 1 || (int64_t)c.n_pages * c.page > INT32_MAX)
        return fail_fmt(HOARD_ERR_INVALID, "n_pages %d of %d tokens", c.n_pages, c.page);
    if (!c.k || !c.v) return fail_fmt(HOARD_ERR_INVALID, "null cache");
    if ((c.type == HOARD_TYPE_I8) != (c.k_scale != nullptr) || (c.type == HOARD_TYPE_I8) != (c.v_scale != nullptr))
        return fail_fmt(HOARD_ERR_INVALID, "scales and cache type %d disagree", c.type);
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 16) || !aligned(c.v_scale, 16))
        return fail_fmt(HOARD_ERR_INVALID, "cache is not 16-byte aligned");
    return 0;
}

int check_stride(const char *what, int64_t stride, int64_t row) {
    if (stride < row || stride > INT32_MAX)
        return fail_fmt(HOARD_ERR_INVALID, "%s stride %lld for rows of %lld", what, (long long)stride, (long long)row);
    return 0;
}

int check_heads(const hoard_heads_args &a) {
    if (!activation_type(a.type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", a.type);
    if (a.n_tokens < 0) return fail_fmt(HOARD_ERR_INVALID, "n_tokens %d", a.n_tokens);
    if (a.n_q_heads < 0 || a.n_q_heads > kMaxHeads || a.n_kv_heads < 0 || a.n_kv_heads > kMaxHeads)
        return fail_fmt(HOARD_ERR_INVALID, "n_q_heads %d, n_kv_heads %d outside 0..%d", a.n_q_heads, a.n_kv_heads, kMaxHeads);
    if (a.head_dim < 8 || a.head_dim > kMaxDim || a.head_dim % 8)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "head_dim %d is not a multiple of 8 up to %d", a.head_dim, kMaxDim);
    if (a.rot_dim < 0 || a.rot_dim > a.head_dim || a.rot_dim % 8)
        return fail_fmt(HOARD_ERR_UNSUPPORTED, "rot_dim %d is not a multiple of 8 up to head_dim %d", a.rot_dim, a.head_dim);
    if (a.rope != HOARD_ROPE_HALVES && a.rope != HOARD_ROPE_PAIRS) return fail_fmt(HOARD_ERR_INVALID, "rope %d", a.rope);
    if (a.n_axes < 1 || a.n_axes > 255) return fail_fmt(HOARD_ERR_INVALID, "n_axes %d outside 1..255", a.n_axes);
    if (!(a.eps > 0.0f)) return fail_fmt(HOARD_ERR_INVALID, "eps %g is not above 0", (double)a.eps);
    return 0;
}

// What forward and backward read beside the heads.
int check_heads_pointers(const hoard_heads_args &a) {
    if (a.n_tokens && a.rot_dim && (!a.pos || !a.freq)) return fail_fmt(HOARD_ERR_INVALID, "rot_dim %d without pos and freq", a.rot_dim);
    const size_t t = type_size(a.type);
    if (!aligned(a.q, t) || !aligned(a.k, t) || !aligned(a.v, t) || !aligned(a.q_out, t) || !aligned(a.k_out, t) ||
        !aligned(a.w_q, 4) || !aligned(a.w_k, 4) || !aligned(a.pos, 4) || !aligned(a.freq, 8) || !aligned(a.stats, 4) ||
        !aligned(a.slots, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    return 0;
}

size_t heads_work_bytes(const hoard_heads_args &a) { return sizeof(float) * 2 * (size_t)a.head_dim * hoard::heads_groups(a); }

int check_rows(const hoard_kv_cache *cache, int type, int n_tokens, const int32_t *slots, const void *k, int64_t k_stride,
               const void *v, int64_t v_stride) {
    if (!cache) return fail_fmt(HOARD_ERR_INVALID, "null cache");
    if (int rc = check_cache(*cache)) return rc;
    if (!activation_type(type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", type);
    if (n_tokens < 0) return fail_fmt(HOARD_ERR_INVALID, "n_tokens %d", n_tokens);
    if (n_tokens && (!slots || (!k && !v))) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    const int64_t row = (int64_t)cache->n_kv_heads * cache->head_dim;
    if (k)
        if (int rc = check_stride("k", k_stride, row)) return rc;
    if (v)
        if (int rc = check_stride("v", v_stride, row)) return rc;
    const size_t t = type_size(type);
    if (!aligned(k, t) || !aligned(v, t) || !aligned(slots, 4)) return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    return 0;
}

int check_attn(const hoard_kv_cache *cache, const hoard_attn_args *a) {
    if (!cache || !a) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_cache(*cache)) return rc;
    if (!activation_type(a->type)) return fail_fmt(HOARD_ERR_UNSUPPORTED, "activation type %d", a->type);
    if (a->n_new < 1 || a->n_new > kMaxNew) return fail_fmt(HOARD_ERR_INVALID, "n_new %d outside 1..%d", a->n_new, kMaxNew);
    if (a->n_seq < 0 || (int64_t)a->n_seq * a->n_new >= 1 << 24)
        return fail_fmt(HOARD_ERR_INVALID, "%d sequences of %d tokens", a->n_seq, a->n_new);
    if (a->n_q_heads < 1 || a->n_q_heads > kMaxHeads || a->n_q_heads % cache->n_kv_heads)
        return fail_fmt(HOARD_ERR_INVALID, "n_q_heads %d beside %d key heads", a->n_q_heads, cache->n_kv_heads);
    if (a->max_pages < 0 || (int64_t)a->max_pages * cache->page > 1 << 30)  // the end of a tile behind the last is a number
        return fail_fmt(HOARD_ERR_INVALID, "max_pages %d of %d tokens", a->max_pages, cache->page);
    if (a->scale != a->scale) return fail_fmt(HOARD_ERR_INVALID, "scale is NaN");
    return 0;
}

}  // namespace

extern "C" {

int hoard_kv_write(const hoard_kv_cache *cache, int type, int n_tokens, const int32_t *slots, const void *k,
                   int64_t k_stride, const void *v, int64_t v_stride, void *stream) {
    if (int rc = check_rows(cache, type, n_tokens, slots, k, k_stride, v, v_stride)) return rc;
    if (!n_tokens) return launched("", hipSuccess);
    hoard_heads_args a{};
    a.type = type;
    a.n_tokens = n_tokens;
    a.n_kv_heads = cache->n_kv_heads;
    a.head_dim = cache->head_dim;
    a.n_axes = 1;
    a.k = k;
    a.v = v;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cache = cache;
    a.slots = slots;
    return launched("cache write", hoard::launch_heads(a, static_cast<hipStream_t>(stream)));
}

int hoard_kv_read(const hoard_kv_cache *cache, int type, int n_tokens, const int32_t *slots, void *k, int64_t k_stride,
                  void *v, int64_t v_stride, void *stream) {
    if (int rc = check_rows(cache, type, n_tokens, slots, k, k_stride, v, v_stride)) return rc;
    if (!n_tokens) return launched("", hipSuccess);
    hoard::KvReadArgs a{*cache, type, n_tokens, slots, k, v, k_stride, v_stride};
    return launched("cache read", hoard::launch_kv_read(a, static_cast<hipStream_t>(stream)));
}

int hoard_heads_forward(const hoard_heads_args *a, void *stream) {
    if (!a) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_heads(*a)) return rc;
    if (int rc = check_heads_pointers(*a)) return rc;
    if (a->cache) {
        if (int rc = check_cache(*a->cache)) return rc;
        if (a->cache->head_dim != a->head_dim || a->cache->n_kv_heads != a->n_kv_heads)
            return fail_fmt(HOARD_ERR_INVALID, "cache of %d heads of %d beside %d of %d", a->cache->n_kv_heads,
                            a->cache->head_dim, a->n_kv_heads, a->head_dim);
        if (a->n_tokens && !a->slots) return fail_fmt(HOARD_ERR_INVALID, "a cache without slots");
    }
    if (a->v && !a->cache) return fail_fmt(HOARD_ERR_INVALID, "v without a cache");
    if ((!a->q && !a->k && !a->v) && a->n_tokens) return fail_fmt(HOARD_ERR_INVALID, "neither q, k nor v");
    if ((a->q != nullptr) != (a->q_out != nullptr)) return fail_fmt(HOARD_ERR_INVALID, "q and q_out go together");
    if (a->k_out && !a->k) return fail_fmt(HOARD_ERR_INVALID, "k_out without k");
    if (a->k && !a->k_out && !a->cache) return fail_fmt(HOARD_ERR_INVALID, "k without k_out or a cache");
    if ((a->w_q && !a->q && a->n_tokens) || (a->w_k && !a->k && a->n_tokens))
        return fail_fmt(HOARD_ERR_INVALID, "weights without their heads");
    const int64_t q_row = (int64_t)a->n_q_heads * a->head_dim, k_row = (int64_t)a->n_kv_heads * a->head_dim;
    if (a->q) {
        if (int rc = check_stride("q", a->q_stride, q_row)) return rc;
        if (int rc = check_stride("q_out", a->q_out_stride, q_row)) return rc;
        if (a->q == a->q_out && a->q_stride != a->q_out_stride)
            return fail_fmt(HOARD_ERR_INVALID, "q_out over q at another stride");
    }
    if (a->k) {
        if (int rc = check_stride("k", a->k_stride, k_row)) return rc;
        if (a->k_out)
            if (int rc = check_stride("k_out", a->k_out_stride, k_row)) return rc;
        if (a->k == a->k_out && a->k_stride != a->k_out_stride)
            return fail_fmt(HOARD_ERR_INVALID, "k_out over k at another stride");
    }
    if (a->v)
        if (int rc = check_stride("v", a->v_stride, k_row)) return rc;
    if (!a->n_tokens) return launched("", hipSuccess);
    return launched("heads", hoard::launch_heads(*a, static_cast<hipStream_t>(stream)));
}

int hoard_heads_workspace(const hoard_heads_args *a, size_t *bytes) {
    if (!a || !bytes) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_heads(*a)) return rc;
    *bytes = heads_work_bytes(*a);
    return launched("", hipSuccess);
}

int hoard_heads_backward(const hoard_heads_args *a, const hoard_heads_grads *g, void *workspace, size_t workspace_bytes,
                         void *stream) {
    if (!a || !g) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_heads(*a)) return rc;
    if (int rc = check_heads_pointers(*a)) return rc;
    if (!g->dq && !g->dk && !g->dw_q && !g->dw_k) return fail_fmt(HOARD_ERR_INVALID, "no gradient wanted");
    if ((g->dw_q && !a->w_q) || (g->dw_k && !a->w_k)) return fail_fmt(HOARD_ERR_INVALID, "a weight's gradient without the weight");
    const int64_t q_row = (int64_t)a->n_q_heads * a->head_dim, k_row = (int64_t)a->n_kv_heads * a->head_dim;
    hoard_heads_grads full = *g;
    if (!full.dq_stride) full.dq_stride = a->q_stride;
    if (!full.dk_stride) full.dk_stride = a->k_stride;
    if (g->dq || g->dw_q) {
        if (a->n_tokens && (!g->dq_out || (a->w_q && (!a->q || !a->stats))))
            return fail_fmt(HOARD_ERR_INVALID, "dq or dw_q without dq_out, or w_q without q and stats");
        if (int rc = check_stride("q_out", a->q_out_stride, q_row)) return rc;
        if (a->w_q)
            if (int rc = check_stride("q", a->q_stride, q_row)) return rc;
        if (g->dq)
            if (int rc = check_stride("dq", full.dq_stride, q_row)) return rc;
        if (g->dq && g->dq == g->dq_out && full.dq_stride != a->q_out_stride)
            return fail_fmt(HOARD_ERR_INVALID, "dq over dq_out at another stride");
    }
    if (g->dk || g->dw_k) {
        if (a->n_tokens && (!g->dk_out || (a->w_k && (!a->k || !a->stats))))
            return fail_fmt(HOARD_ERR_INVALID, "dk or dw_k without dk_out, or w_k without k and stats");
        if (int rc = check_stride("k_out", a->k_out_stride, k_row)) return rc;
        if (a->w_k)
            if (int rc = check_stride("k", a->k_stride, k_row)) return rc;
        if (g->dk)
            if (int rc = check_stride("dk", full.dk_stride, k_row)) return rc;
        if (g->dk && g->dk == g->dk_out && full.dk_stride != a->k_out_stride)
            return fail_fmt(HOARD_ERR_INVALID, "dk over dk_out at another stride");
    }
    const size_t t = type_size(a->type);
    if (!aligned(g->dq_out, t) || !aligned(g->dk_out, t) || !aligned(g->dq, t) || !aligned(g->dk, t) || !aligned(g->dw_q, 4) ||
        !aligned(g->dw_k, 4) || !aligned(workspace, 4))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    const size_t need = heads_work_bytes(*a);
    if (need && (!workspace || workspace_bytes < need))
        return fail_fmt(HOARD_ERR_INVALID, "workspace of %zu bytes, %zu wanted", workspace ? workspace_bytes : 0, need);
    return launched("heads gradient", hoard::launch_heads_grad(*a, full, static_cast<float *>(workspace), static_cast<hipStream_t>(stream)));
}

int hoard_attn_workspace(const hoard_kv_cache *cache, const hoard_attn_args *a, size_t *bytes) {
    if (!bytes) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_attn(cache, a)) return rc;
    *bytes = hoard::attn_work_bytes(*cache, *a);
    return launched("", hipSuccess);
}

int hoard_attn_decode(const hoard_kv_cache *cache, const hoard_attn_args *a, void *workspace, size_t workspace_bytes,
                      void *stream) {
    if (int rc = check_attn(cache, a)) return rc;
    if (!a->n_seq) return launched("", hipSuccess);
    if (!a->q || !a->lens || !a->out || (!a->pages && a->max_pages)) return fail_fmt(HOARD_ERR_INVALID, "null argument");
    if (int rc = check_stride("q", a->q_stride, (int64_t)a->n_q_heads * cache->head_dim)) return rc;
    const size_t t = type_size(a->type);
    if (!aligned(a->q, t) || !aligned(a->out, t) || !aligned(a->pages, 4) || !aligned(a->lens, 4) || !aligned(a->lse, 4) ||
        !aligned(workspace, 16))
        return fail_fmt(HOARD_ERR_INVALID, "misaligned argument");
    const size_t need = hoard::attn_work_bytes(*cache, *a);
    if (need && (!workspace || workspace_bytes < need))
        return fail_fmt(HOARD_ERR_INVALID, "workspace of %zu bytes, %zu wanted", workspace ? workspace_bytes : 0, need);
    return launched("attention", hoard::launch_attn(*cache, *a, static_cast<float *>(workspace), static_cast<hipStream_t>(stream)));
}

}  // extern "C"

"""What the operators of include/hoard_ops.h refuse, before anything is launched: no device is needed."""
import ctypes

import pytest

import hoard_amd as H

A = 0x10000  # an address that is aligned and never read: every call here returns before a launch


def q4(**kw):
    d = dict(codes=A, scales=A, zeros=None, rows=64, cols=256, group=128, n_mat=1, scale_type=H.TYPE_F16)
    d.update(kw)
    return H.Q4Matrix(*d.values())


def refused(rc, code, *words):
    text = H.load_library().hoard_last_error().decode()
    assert rc == code, (rc, text)
    assert all(w in text for w in words), text


@pytest.mark.parametrize("field,value,code,word", [
    ("codes", None, H.ERR_INVALID, "null"), ("codes", A + 8, H.ERR_INVALID, "16-byte"),
    ("scales", None, H.ERR_INVALID, "null"), ("scales", A + 1, H.ERR_INVALID, "aligned"),
    ("rows", (1 << 22) + 1, H.ERR_UNSUPPORTED, "rows"), ("rows", 0, H.ERR_INVALID, "rows"), ("rows", -4, H.ERR_INVALID, "rows"),
    ("cols", 0, H.ERR_INVALID, "cols"), ("cols", 192, H.ERR_INVALID, "cols"), ("cols", 100, H.ERR_INVALID, "cols"),
    ("cols", (1 << 20) + 128, H.ERR_UNSUPPORTED, "cols"), ("group", 16, H.ERR_UNSUPPORTED, "group"), ("group", 0, H.ERR_UNSUPPORTED, "group"),
    ("group", 256, H.ERR_UNSUPPORTED, "group"), ("n_mat", 0, H.ERR_INVALID, "n_mat"),
    ("scale_type", H.TYPE_Q4_K, H.ERR_UNSUPPORTED, "scale type")])
@pytest.mark.parametrize("second", [False, True])
def test_q4_matrix(hlib, field, value, code, word, second):
    w, bad = q4(), q4(**{field: value})
    a, b = (w, bad) if second else (bad, None)
    up = ctypes.byref(b) if b is not None else None
    refused(hlib.hoard_q4_matmul(ctypes.byref(a), up, H.TYPE_F32, 1, A, A, None), code, word)
    refused(hlib.hoard_q4_matmul_ids(ctypes.byref(a), up, H.TYPE_F32, 1, A, 1, A, A, None), code, word)
    refused(hlib.hoard_q4_matmul_sorted(ctypes.byref(a), up, H.TYPE_F32, 1, A, A, A, None), code, word)


def test_q4_call(hlib):
    w = ctypes.byref(q4())
    many = ctypes.byref(q4(n_mat=4))
    inv = H.ERR_INVALID
    refused(hlib.hoard_q4_matmul(None, None, H.TYPE_F32, 1, A, A, None), inv, "null")
    refused(hlib.hoard_q4_matmul(many, None, H.TYPE_F32, 1, A, A, None), inv, "n_mat")
    refused(hlib.hoard_q4_matmul(w, ctypes.byref(q4(rows=65)), H.TYPE_F32, 1, A, A, None), inv, "up")
    refused(hlib.hoard_q4_matmul(w, ctypes.byref(q4(cols=384)), H.TYPE_F32, 1, A, A, None), inv, "up")
    refused(hlib.hoard_q4_matmul(w, ctypes.byref(q4(group=64)), H.TYPE_F32, 1, A, A, None), inv, "groups of 64")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_Q4_K, 1, A, A, None), H.ERR_UNSUPPORTED, "type")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_F32, -1, A, A, None), inv, "n_rows")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_F32, 1, None, A, None), inv, "null")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_F32, 1, A, None, None), inv, "null")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_F32, 1, A + 4, A, None), inv, "x is not")
    refused(hlib.hoard_q4_matmul(w, None, H.TYPE_F32, 1, A, A + 2, None), inv, "misaligned")
    refused(hlib.hoard_q4_matmul_ids(many, None, H.TYPE_F32, 8, A, 3, A, A, None), inv, "x_share")
    refused(hlib.hoard_q4_matmul_ids(many, None, H.TYPE_F32, 8, A, 0, A, A, None), inv, "x_share")
    refused(hlib.hoard_q4_matmul_ids(many, None, H.TYPE_F32, 8, A, 8, None, A, None), inv, "null")
    refused(hlib.hoard_q4_matmul_sorted(many, None, H.TYPE_F32, 8, A, None, A, None), inv, "null")
    refused(hlib.hoard_q4_matmul_sorted(many, None, H.TYPE_F32, 8, A, A + 2, A, None), inv, "misaligned")
    # no rows: valid, nothing to do
    assert hlib.hoard_q4_matmul(w, None, H.TYPE_F32, 0, None, None, None) == H.OK
    assert hlib.hoard_q4_matmul_ids(many, None, H.TYPE_F32, 0, None, 1, None, None, None) == H.OK
    assert hlib.hoard_last_error() == b""


def test_sort(hlib):
    inv, n = H.ERR_INVALID, ctypes.c_size_t(7)
    for m, k, e, word in ((-1, 8, 64, "n_tokens"), (4, 0, 64, "k"), (4, 65, 64, "k"), (4, 8, 0, "n_expert"),
                          (4, 8, 1025, "n_expert"), (1 << 28, 8, 64, "pairs")):
        refused(hlib.hoard_sort_workspace(m, k, e, ctypes.byref(n)), inv, word)
        refused(hlib.hoard_sort_pairs(m, k, e, A, A, A, A, A, 1 << 40, None), inv, word)
    refused(hlib.hoard_sort_workspace(4, 8, 64, None), inv, "null")
    for hole in range(4):
        p = [A] * 4
        p[hole] = None
        refused(hlib.hoard_sort_pairs(4, 8, 64, *p, A, 1 << 20, None), inv, "null")
        p[hole] = A + 2
        refused(hlib.hoard_sort_pairs(4, 8, 64, *p, A, 1 << 20, None), inv, "misaligned")
    assert hlib.hoard_sort_workspace(4096, 8, 128, ctypes.byref(n)) == H.OK and n.value > 0
    refused(hlib.hoard_sort_pairs(4096, 8, 128, A, A, A, A, A, n.value - 1, None), inv, "workspace", str(n.value))
    refused(hlib.hoard_sort_pairs(4096, 8, 128, A, A, A, A, None, n.value, None), inv, "workspace")
    # the size that a caller may count on: a count an expert for every 1024 pairs
    for m, k, e in ((1, 1, 1), (128, 8, 64), (129, 8, 64), (5000, 10, 1024), (1 << 20, 64, 7)):
        assert hlib.hoard_sort_workspace(m, k, e, ctypes.byref(n)) == H.OK
        assert n.value <= 4 * e * ((m * k + 1023) // 1024)


def test_rows(hlib):
    inv = H.ERR_INVALID
    for call, args in ((hlib.hoard_sort_gather, 4), (hlib.hoard_sort_combine, 5), (hlib.hoard_sort_combine_grad, 6)):
        p = [A] * args
        refused(call(H.TYPE_Q4_K, 4, 8, 64, *p, None), H.ERR_UNSUPPORTED, "type")
        refused(call(H.TYPE_F32, -1, 8, 64, *p, None), inv, "n_tokens")
        refused(call(H.TYPE_F32, 4, 0, 64, *p, None), inv, "k")
        refused(call(H.TYPE_F32, 4, 65, 64, *p, None), inv, "k")
        refused(call(H.TYPE_F32, 4, 8, 0, *p, None), inv, "n")
        refused(call(H.TYPE_F32, 1 << 28, 8, 64, *p, None), inv, "pairs")
        for i in range(args):
            q = list(p)
            q[i] = A + 1
            refused(call(H.TYPE_F32, 4, 8, 64, *q, None), inv, "misaligned")
        assert call(H.TYPE_F32, 0, 8, 64, *([None] * args), None) == H.OK
    for hole in (0, 1, 3):
        p = [A] * 4
        p[hole] = None
        refused(hlib.hoard_sort_gather(H.TYPE_F32, 4, 8, 64, *p, None), inv, "null")
    for hole in (0, 1, 4):
        p = [A] * 5
        p[hole] = None
        refused(hlib.hoard_sort_combine(H.TYPE_F32, 4, 8, 64, *p, None), inv, "null")
    for hole in (0, 1, 2, 3, 5):
        p = [A] * 6
        p[hole] = None
        refused(hlib.hoard_sort_combine_grad(H.TYPE_F32, 4, 8, 64, *p, None), inv, "null")


def norm(**kw):
    d = dict(type=H.TYPE_BF16, res_type=H.TYPE_F32, gate_kind=H.GATE_CHANNEL, gate_sigmoid=0, n_rows=4, n=64, eps=1e-6,
             scale=1.0, w_offset=0.0, r=A, b=A, gate=A, w_post=A, w_pre=A, r_out=A, h=A, stats=A)
    d.update(kw)
    return H.NormArgs(*d.values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(type=H.TYPE_Q4_K), H.ERR_UNSUPPORTED, "type"), (dict(res_type=H.TYPE_F16), H.ERR_UNSUPPORTED, "residual type"),
    (dict(gate_kind=4), H.ERR_INVALID, "gate_kind"), (dict(gate_kind=-1), H.ERR_INVALID, "gate_kind"),
    (dict(n_rows=-1), H.ERR_INVALID, "n_rows"), (dict(n=0), H.ERR_INVALID, "n 0"),
    (dict(n=16385), H.ERR_INVALID, "16385"), (dict(eps=0.0), H.ERR_INVALID, "eps"),
    (dict(eps=-1.0), H.ERR_INVALID, "eps"), (dict(eps=float("nan")), H.ERR_INVALID, "eps"),
    (dict(b=None), H.ERR_INVALID, "without b"), (dict(gate=None), H.ERR_INVALID, "gate"),
    (dict(gate_kind=H.GATE_NONE), H.ERR_INVALID, "gate"), (dict(b=A + 1), H.ERR_INVALID, "misaligned"),
    (dict(r=A + 2), H.ERR_INVALID, "misaligned"), (dict(w_post=A + 2), H.ERR_INVALID, "misaligned"),
    (dict(w_pre=A + 2), H.ERR_INVALID, "misaligned"), (dict(r_out=A + 2), H.ERR_INVALID, "misaligned"),
    (dict(stats=A + 2), H.ERR_INVALID, "misaligned"), (dict(gate=A + 2), H.ERR_INVALID, "misaligned")])
def test_norm_both(hlib, kw, code, word):
    a, g = norm(**kw), H.NormGrads(A, A, A, A, A, A, A)
    refused(hlib.hoard_norm_forward(ctypes.byref(a), None), code, word)
    refused(hlib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(g), A, 1 << 40, None), code, word)


def test_norm_forward(hlib):
    inv = H.ERR_INVALID
    bare = dict(b=None, gate=None, gate_kind=H.GATE_NONE, w_post=None, r_out=None)
    refused(hlib.hoard_norm_forward(None, None), inv, "null")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(h=None)), None), inv, "w_pre")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(w_pre=None)), None), inv, "w_pre")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(r_out=None)), None), inv, "r_out")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(**dict(bare, r_out=A))), None), inv, "r_out")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(**bare, h=None, w_pre=None)), None), inv, "nothing")
    refused(hlib.hoard_norm_forward(ctypes.byref(norm(r=None)), None), inv, "null")
    assert hlib.hoard_norm_forward(ctypes.byref(norm(n_rows=0)), None) == H.OK


def test_norm_backward(hlib):
    inv, n = H.ERR_INVALID, ctypes.c_size_t()
    a = norm()

    def call(a, *g, work=A, size=1 << 40):
        return hlib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(H.NormGrads(*g)), work, size, None)

    refused(hlib.hoard_norm_backward(None, ctypes.byref(H.NormGrads()), A, 1, None), inv, "null")
    refused(hlib.hoard_norm_backward(ctypes.byref(a), None, A, 1, None), inv, "null")
    refused(hlib.hoard_norm_workspace(ctypes.byref(a), None), inv, "null")
    refused(hlib.hoard_norm_workspace(None, ctypes.byref(n)), inv, "null")
    refused(call(a, None, None, A, A, A, A, A), inv, "neither")
    refused(call(norm(w_pre=None), A, A, A, A, A, A, None), inv, "w_pre")
    refused(call(norm(r_out=None), A, A, A, A, A, A, A), inv, "r_out")
    refused(call(a, A, None, A, A, A, A, A), inv, "dw_pre without dh")
    bare = norm(b=None, gate=None, gate_kind=H.GATE_NONE, w_post=None)
    for i in (3, 4, 5):
        g = [A, A, A, None, None, None, None]
        g[i] = A
        refused(call(bare, *g), inv, "without b")
    refused(call(norm(w_post=None), A, A, A, A, A, A, A), inv, "w_post")
    refused(call(norm(gate=None, gate_kind=H.GATE_NONE), A, A, A, A, A, A, A), inv, "dgate")
    refused(call(a, A, A, None, None, None, None, None), inv, "no gradient")
    refused(call(norm(stats=None), A, A, A, A, A, A, A), inv, "stats")
    for i in range(7):
        g = [A] * 7
        g[i] = A + 1
        refused(call(a, *g), inv, "misaligned")
    assert hlib.hoard_norm_workspace(ctypes.byref(a), ctypes.byref(n)) == H.OK and n.value > 0
    refused(call(a, A, A, A, A, A, A, A, size=n.value - 1), inv, "workspace", str(n.value))
    refused(call(a, A, A, A, A, A, A, A, work=None), inv, "workspace")
    # the size that a caller may count on: three sums a column for at most 1024 groups of rows
    for rows in (0, 1, 7, 1000, 100000):
        for cols in (1, 64, 2048, 16384):
            assert hlib.hoard_norm_workspace(ctypes.byref(norm(n_rows=rows, n=cols)), ctypes.byref(n)) == H.OK
            assert n.value <= 12 * cols * min(rows, 1024)

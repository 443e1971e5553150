"""What the operators of include/hoard_attn.h refuse, before anything is launched: no device is needed."""
import ctypes

import pytest

import hoard_amd as H

A = 0x10000  # an address that is aligned and never read: every call here returns before a launch


def cache(**kw):
    d = dict(k=A, v=A, k_scale=None, v_scale=None, type=H.TYPE_F16, n_pages=4, page=16, n_kv_heads=2, head_dim=64)
    d.update(kw)
    return H.KvCache(**d)


def heads(**kw):
    d = dict(type=H.TYPE_F32, n_tokens=3, n_q_heads=4, n_kv_heads=2, head_dim=64, rot_dim=64, rope=H.ROPE_HALVES, n_axes=1,
             eps=1e-6, w_offset=0.0, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, k_out_stride=128, q=A, k=A,
             v=None, w_q=A, w_k=A, pos=A, freq=A, axis=None, q_out=A, k_out=A, stats=A)
    d.update(kw)
    return H.HeadsArgs(**d)


def attn(**kw):
    d = dict(type=H.TYPE_F32, n_seq=2, n_new=1, n_q_heads=4, max_pages=3, scale=0.125, q_stride=256, q=A, pages=A, lens=A,
             out=A, lse=None)
    d.update(kw)
    return H.AttnArgs(**d)


def refused(rc, code, *words):
    text = H.load_library().hoard_last_error().decode()
    assert rc == code, (rc, text)
    assert all(w in text for w in words), text


CACHES = [("type", H.TYPE_F32, H.ERR_UNSUPPORTED, "type"), ("type", H.TYPE_Q4_K, H.ERR_UNSUPPORTED, "type"),
          ("type", H.TYPE_I8, H.ERR_INVALID, "scales"), ("k_scale", A, H.ERR_INVALID, "scales"), ("v_scale", A, H.ERR_INVALID, "scales"),
          ("page", 8, H.ERR_UNSUPPORTED, "page"), ("page", 48, H.ERR_UNSUPPORTED, "page"), ("page", 512, H.ERR_UNSUPPORTED, "page"),
          ("page", 0, H.ERR_UNSUPPORTED, "page"), ("page", -16, H.ERR_UNSUPPORTED, "page"), ("n_pages", 0, H.ERR_INVALID, "n_pages"),
          ("n_pages", -1, H.ERR_INVALID, "n_pages"), ("n_pages", 1 << 27, H.ERR_INVALID, "n_pages"),
          ("n_kv_heads", 0, H.ERR_INVALID, "n_kv_heads"), ("n_kv_heads", 1025, H.ERR_INVALID, "n_kv_heads"),
          ("head_dim", 24, H.ERR_UNSUPPORTED, "head_dim"), ("head_dim", 272, H.ERR_UNSUPPORTED, "head_dim"),
          ("head_dim", 0, H.ERR_UNSUPPORTED, "head_dim"), ("k", None, H.ERR_INVALID, "null"), ("v", None, H.ERR_INVALID, "null"),
          ("k", A + 8, H.ERR_INVALID, "16-byte"), ("v", A + 2, H.ERR_INVALID, "16-byte")]


@pytest.mark.parametrize("field,value,code,word", CACHES)
def test_cache(hlib, field, value, code, word):
    c = ctypes.byref(cache(**{field: value}))
    refused(hlib.hoard_kv_write(c, H.TYPE_F32, 1, A, A, 4096, A, 4096, None), code, word)
    refused(hlib.hoard_kv_read(c, H.TYPE_F32, 1, A, A, 4096, A, 4096, None), code, word)
    refused(hlib.hoard_attn_decode(c, ctypes.byref(attn()), None, 0, None), code, word)
    need = ctypes.c_size_t()
    refused(hlib.hoard_attn_workspace(c, ctypes.byref(attn()), ctypes.byref(need)), code, word)
    kept = cache(**{field: value})
    a = heads(cache=ctypes.addressof(kept), slots=A)
    refused(hlib.hoard_heads_forward(ctypes.byref(a), None), code)


def test_rows(hlib):
    c = ctypes.byref(cache())
    for call in (hlib.hoard_kv_write, hlib.hoard_kv_read):
        refused(call(None, H.TYPE_F32, 1, A, A, 128, A, 128, None), H.ERR_INVALID, "null")
        refused(call(c, H.TYPE_I8, 1, A, A, 128, A, 128, None), H.ERR_UNSUPPORTED, "type")
        refused(call(c, H.TYPE_F32, -1, A, A, 128, A, 128, None), H.ERR_INVALID, "n_tokens")
        refused(call(c, H.TYPE_F32, 1, None, A, 128, A, 128, None), H.ERR_INVALID, "null")
        refused(call(c, H.TYPE_F32, 1, A, None, 128, None, 128, None), H.ERR_INVALID, "null")
        refused(call(c, H.TYPE_F32, 1, A, A, 127, A, 128, None), H.ERR_INVALID, "k stride")
        refused(call(c, H.TYPE_F32, 1, A, A, 128, A, 1 << 31, None), H.ERR_INVALID, "v stride")
        refused(call(c, H.TYPE_F32, 1, A, A + 2, 128, A, 128, None), H.ERR_INVALID, "misaligned")
        refused(call(c, H.TYPE_F32, 1, A + 1, A, 128, A, 128, None), H.ERR_INVALID, "misaligned")
        assert call(c, H.TYPE_F32, 0, None, None, 128, None, 128, None) == H.OK


HEADS = [(dict(type=H.TYPE_I8), H.ERR_UNSUPPORTED, "type"), (dict(n_tokens=-1), H.ERR_INVALID, "n_tokens"),
         (dict(n_q_heads=-1), H.ERR_INVALID, "n_q_heads"), (dict(n_kv_heads=1025), H.ERR_INVALID, "n_kv_heads"),
         (dict(head_dim=12), H.ERR_UNSUPPORTED, "head_dim"), (dict(head_dim=264), H.ERR_UNSUPPORTED, "head_dim"),
         (dict(head_dim=0), H.ERR_UNSUPPORTED, "head_dim"), (dict(rot_dim=72), H.ERR_UNSUPPORTED, "rot_dim"),
         (dict(rot_dim=20), H.ERR_UNSUPPORTED, "rot_dim"), (dict(rot_dim=-8), H.ERR_UNSUPPORTED, "rot_dim"),
         (dict(rope=2), H.ERR_INVALID, "rope"), (dict(n_axes=0), H.ERR_INVALID, "n_axes"), (dict(n_axes=256), H.ERR_INVALID, "n_axes"),
         (dict(eps=0.0), H.ERR_INVALID, "eps"), (dict(eps=float("nan")), H.ERR_INVALID, "eps"), (dict(pos=None), H.ERR_INVALID, "pos"),
         (dict(freq=None), H.ERR_INVALID, "freq"), (dict(freq=A + 4), H.ERR_INVALID, "misaligned"), (dict(q=A + 2), H.ERR_INVALID, "misaligned"),
         (dict(w_k=A + 2), H.ERR_INVALID, "misaligned"), (dict(stats=A + 1), H.ERR_INVALID, "misaligned")]


@pytest.mark.parametrize("kw,code,word", HEADS)
def test_heads(hlib, kw, code, word):
    a = heads(**kw)
    refused(hlib.hoard_heads_forward(ctypes.byref(a), None), code, word)
    g = H.HeadsGrads(A, A, A, A, A, A)
    refused(hlib.hoard_heads_backward(ctypes.byref(a), ctypes.byref(g), A, 1 << 30, None), code, word)


@pytest.mark.parametrize("kw,word", [
    (dict(v=A), "v without"), (dict(q=None), "q and q_out"), (dict(q_out=None), "q and q_out"), (dict(k=None), "k_out without k"),
    (dict(k_out=None), "k without"), (dict(q=None, q_out=None), "weights"), (dict(q=None, q_out=None, k=None, k_out=None), "neither"),
    (dict(q_stride=255), "q stride"), (dict(q_out_stride=255), "q_out stride"), (dict(k_stride=1 << 31), "k stride"),
    (dict(k_out_stride=-1), "k_out stride"), (dict(q_stride=512), "another stride"), (dict(k_stride=512, k_out_stride=256), "another stride")])
def test_heads_forward(hlib, kw, word):
    refused(hlib.hoard_heads_forward(ctypes.byref(heads(**kw)), None), H.ERR_INVALID, word)


def test_heads_with_a_cache(hlib):
    refused(hlib.hoard_heads_forward(None, None), H.ERR_INVALID, "null")
    for c, kw, word in ((cache(head_dim=128), {}, "beside"), (cache(n_kv_heads=4), {}, "beside"), (cache(), dict(slots=None), "slots"),
                        (cache(), dict(v=A, v_stride=100), "v stride"), (cache(), dict(slots=A + 2), "misaligned")):
        a = heads(cache=ctypes.addressof(c), **{"slots": A, **kw})
        refused(hlib.hoard_heads_forward(ctypes.byref(a), None), H.ERR_INVALID, word)
    c = cache()
    assert hlib.hoard_heads_forward(ctypes.byref(heads(n_tokens=0, cache=ctypes.addressof(c))), None) == H.OK


@pytest.mark.parametrize("kw,grads,word", [
    ({}, {}, "no gradient"), (dict(w_q=None), dict(dw_q=A), "without the weight"), ({}, dict(dq=A), "dq_out"),
    (dict(stats=None), dict(dq=A, dq_out=A), "stats"), (dict(q=None), dict(dq=A, dq_out=A), "without q"),
    (dict(k=None), dict(dw_k=A, dk_out=A), "without k"), ({}, dict(dk=A, dk_out=A, dk_stride=100), "dk stride"),
    ({}, dict(dq=A, dq_out=A, dq_stride=512), "another stride"), ({}, dict(dk=A, dk_out=A, dk_stride=512), "another stride"),
    (dict(k_out_stride=5), dict(dk=A, dk_out=A), "k_out stride"), (dict(q_stride=5), dict(dq=A + 4, dq_out=A), "q stride"),
    ({}, dict(dq=A + 2, dq_out=A), "misaligned"), ({}, dict(dq=A + 4, dq_out=A, dw_q=A + 2), "misaligned")])
def test_heads_backward(hlib, kw, grads, word):
    a, g = heads(**kw), H.HeadsGrads(**grads)
    refused(hlib.hoard_heads_backward(ctypes.byref(a), ctypes.byref(g), A, 1 << 30, None), H.ERR_INVALID, word)


def test_heads_workspace(hlib):
    need, a, g = ctypes.c_size_t(), heads(n_tokens=100000), H.HeadsGrads(dq=A, dq_out=A)
    assert hlib.hoard_heads_workspace(ctypes.byref(a), ctypes.byref(need)) == H.OK
    assert 0 < need.value <= 2 * 4 * 64 * 1024
    refused(hlib.hoard_heads_workspace(ctypes.byref(a), None), H.ERR_INVALID, "null")
    refused(hlib.hoard_heads_workspace(None, ctypes.byref(need)), H.ERR_INVALID, "null")
    back = lambda *w: hlib.hoard_heads_backward(ctypes.byref(a), ctypes.byref(g), *w, None)  # noqa: E731
    refused(back(A, need.value - 1), H.ERR_INVALID, "workspace")
    refused(back(None, need.value), H.ERR_INVALID, "workspace")
    refused(back(A + 2, need.value), H.ERR_INVALID, "misaligned")
    refused(hlib.hoard_heads_backward(ctypes.byref(a), None, A, need.value, None), H.ERR_INVALID, "null")


@pytest.mark.parametrize("kw,code,word", [
    (dict(type=H.TYPE_I8), H.ERR_UNSUPPORTED, "type"), (dict(n_seq=-1), H.ERR_INVALID, "sequences"), (dict(n_new=0), H.ERR_INVALID, "n_new"),
    (dict(n_new=65), H.ERR_INVALID, "n_new"), (dict(n_seq=1 << 24), H.ERR_INVALID, "sequences"), (dict(n_q_heads=0), H.ERR_INVALID, "n_q_heads"),
    (dict(n_q_heads=3), H.ERR_INVALID, "n_q_heads"), (dict(n_q_heads=1026), H.ERR_INVALID, "n_q_heads"),
    (dict(max_pages=-1), H.ERR_INVALID, "max_pages"), (dict(max_pages=1 << 27), H.ERR_INVALID, "max_pages"), (dict(max_pages=(1 << 26) + 1), H.ERR_INVALID, "max_pages"),
    (dict(scale=float("nan")), H.ERR_INVALID, "scale")])
def test_attention(hlib, kw, code, word):
    c, a, need = cache(), attn(**kw), ctypes.c_size_t()
    refused(hlib.hoard_attn_decode(ctypes.byref(c), ctypes.byref(a), A, 1 << 40, None), code, word)
    refused(hlib.hoard_attn_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(need)), code, word)


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null"), (dict(lens=None), "null"), (dict(out=None), "null"), (dict(pages=None), "null"), (dict(q_stride=255), "q stride"),
    (dict(q=A + 2), "misaligned"), (dict(out=A + 1), "misaligned"), (dict(pages=A + 2), "misaligned"), (dict(lens=A + 1), "misaligned"),
    (dict(lse=A + 2), "misaligned")])
def test_attention_call(hlib, kw, word):
    c, a = cache(), attn(**kw)
    refused(hlib.hoard_attn_decode(ctypes.byref(c), ctypes.byref(a), A, 1 << 40, None), H.ERR_INVALID, word)


def test_attention_workspace(hlib):
    c, need = cache(n_pages=1 << 12), ctypes.c_size_t()
    a = attn(max_pages=1 << 12)
    refused(hlib.hoard_attn_workspace(ctypes.byref(c), ctypes.byref(a), None), H.ERR_INVALID, "null")
    refused(hlib.hoard_attn_workspace(None, ctypes.byref(a), ctypes.byref(need)), H.ERR_INVALID, "null")
    assert hlib.hoard_attn_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(need)) == H.OK
    call = lambda *w: hlib.hoard_attn_decode(ctypes.byref(c), ctypes.byref(a), *w, None)  # noqa: E731
    refused(call(A + 8, need.value), H.ERR_INVALID, "misaligned")
    if need.value:
        refused(call(A, need.value - 1), H.ERR_INVALID, "workspace")
        refused(call(None, need.value), H.ERR_INVALID, "workspace")
    assert hlib.hoard_attn_decode(ctypes.byref(c), ctypes.byref(attn(n_seq=0, q=None, lens=None, out=None)), None, 0, None) == H.OK

"""Calls of the attention half on torch tensors that its documentation allows or refuses: one tensor for two arguments,
a cache whose tensors overlap."""
import pytest

import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def rand(*shape):
    return torch.randn(shape, device="cuda")


def test_one_tensor_for_two_arguments():
    """Read twice it may be; written over it may not, as the other heads are read from it by other waves."""
    from hoard_amd import attn
    x, w = rand(5, 2, 32), rand(32)
    cache = attn.KVCache.new(1, 16, 2, 32, torch.float16)
    slots = torch.arange(5, dtype=torch.int32, device="cuda")
    kept = x.clone()
    st = attn.heads_forward(x, x, w_q=w, w_k=w, want_stats=True)
    assert torch.equal(st.q_out, st.k_out) and torch.equal(x, kept)
    back = attn.heads_backward(x, x, q=x, k=x, w_q=w, w_k=w, stats=st.stats)
    assert torch.equal(back.dq, back.dk)
    bad = [
        lambda: attn.heads_forward(x, x, w_q=w, q_out=x),
        lambda: attn.heads_forward(x, x, w_q=w, k_out=x),
        lambda: attn.heads_forward(x, None, x, cache=cache, slots=slots, q_out=x),
        lambda: attn.heads_forward(k=x, v=x, cache=cache, slots=slots, k_out=x),
        lambda: attn.heads_backward(x, x, dq=x),
        lambda: attn.heads_backward(x, x, dk=x),
        lambda: attn.heads_backward(x, q=x, w_q=w, stats=st.stats[:, :2].contiguous(), dq=x),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(H.HoardError, match="overlaps"):
            call()
            pytest.fail(str(i))
    assert torch.equal(x, kept)
    # heads that are not normed are not read by the gradient
    attn.heads_backward(x, q=x, dq=x)
    assert torch.equal(x, kept)


def test_a_cache_over_itself():
    """Keys and values, or scales, in the same memory may be read; they are not written."""
    from hoard_amd import attn
    x, slots = rand(5, 2, 32), torch.arange(5, dtype=torch.int32, device="cuda")
    buf = torch.zeros(2 * 2 * 16 * 32, dtype=torch.float16, device="cuda")
    half = buf[:1024].view(1, 2, 16, 32)
    shared = attn.KVCache(half, half)
    attn.attn_decode(rand(1, 4, 32), shared, slots[:1].view(1, 1), slots[3:4])
    codes, scales = torch.zeros((2, 1, 2, 16, 32), dtype=torch.int8, device="cuda"), torch.zeros((1, 2, 16), device="cuda")
    for c in (shared, attn.KVCache(half, buf[512:1536].view(1, 2, 16, 32)), attn.KVCache(codes[0], codes[1], scales, scales)):
        with pytest.raises(H.HoardError, match="cache: overlaps"):
            attn.kv_write(c, slots, x, x)
        with pytest.raises(H.HoardError, match="cache: overlaps"):
            attn.heads_forward(k=x, v=x, cache=c, slots=slots)
    attn.kv_write(attn.KVCache(half, buf[1024:].view(1, 2, 16, 32)), slots, x, x)

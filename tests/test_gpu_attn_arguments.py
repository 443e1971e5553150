"""Calls of the attention half on torch tensors that its documentation allows or refuses: one tensor for two arguments,
a cache whose tensors overlap, one of the two gradients alone, what is no tensor."""
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


@pytest.mark.parametrize("rope", [False, True])
def test_one_gradient_alone(rope):
    """One of the two, with the statistics of both heads: the other's heads need not be given."""
    from hoard_amd import attn
    q, k, w_q, w_k, dq_out, dk_out = rand(7, 4, 32), rand(7, 2, 32), rand(32), rand(32), rand(7, 4, 32), rand(7, 2, 32)
    r = attn.Rope(torch.arange(7, dtype=torch.int32, device="cuda"), attn.rope_freq(16, 100.0)) if rope else None
    st = attn.heads_forward(q, k, w_q=w_q, w_k=w_k, rope=r, want_stats=True)
    both = attn.heads_backward(dq_out, dk_out, q=q, k=k, w_q=w_q, w_k=w_k, rope=r, stats=st.stats)
    one = attn.heads_backward(dq_out, q=q, w_q=w_q, rope=r, stats=st.stats)
    assert torch.equal(one.dq, both.dq) and one.dk is None and one.dw_k is None
    # few tokens: a workgroup's sums, in the same order
    assert torch.allclose(one.dw_q, both.dw_q, rtol=1e-5, atol=1e-5)
    one = attn.heads_backward(None, dk_out, k=k, w_k=w_k, rope=r, stats=st.stats)
    assert torch.equal(one.dk, both.dk) and one.dq is None and one.dw_q is None
    assert torch.allclose(one.dw_k, both.dw_k, rtol=1e-5, atol=1e-5)
    # q normed beside heads that go into a cache, whose columns the statistics have too
    cache = attn.KVCache.new(1, 16, 2, 32, torch.float16)
    slots = torch.arange(7, dtype=torch.int32, device="cuda")
    st = attn.heads_forward(q, None, k, w_q=w_q, rope=r, want_stats=True, cache=cache, slots=slots)
    assert torch.equal(attn.heads_backward(dq_out, q=q, w_q=w_q, rope=r, stats=st.stats).dq, both.dq)
    for stats in (st.stats[:, :3].contiguous(), st.stats[:6], rand(7, 4, 2), rand(7), 5):
        with pytest.raises(H.HoardError, match="stats"):
            attn.heads_backward(dq_out, q=q, w_q=w_q, stats=stats)


def test_what_is_no_tensor():
    from hoard_amd import attn
    x, w = rand(3, 2, 32), rand(32)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    cache = attn.KVCache.new(1, 16, 2, 32, torch.float16)
    freq = attn.rope_freq(16, 100.0)
    bad = [
        lambda: attn.heads_forward([1.0], x),
        lambda: attn.heads_forward(x, [1.0]),
        lambda: attn.heads_forward(x, 5),
        lambda: attn.heads_forward(x, rand(3, 64)),
        lambda: attn.heads_forward(x, v=[1.0], cache=cache, slots=slots),
        lambda: attn.heads_forward(x, w_q=1.0),
        lambda: attn.heads_forward(x, rope=(slots, freq)),
        lambda: attn.heads_forward(x, rope=attn.Rope(slots, [1.0])),
        lambda: attn.heads_forward(x, rope=attn.Rope([1, 2, 3], freq)),
        lambda: attn.heads_forward(x, rope=attn.Rope(slots, freq, [0])),
        lambda: attn.heads_forward(k=x, cache=(x, x), slots=slots),
        lambda: attn.heads_forward(k=x, cache=cache, slots=[0, 1, 2]),
        lambda: attn.heads_forward(x, q_out=[1.0]),
        lambda: attn.heads_backward([1.0]),
        lambda: attn.heads_backward(x, 5),
        lambda: attn.heads_backward(x, q=5, w_q=w, stats=rand(3, 2)),
        lambda: attn.heads_backward(x, dq=[1.0]),
        lambda: attn.kv_write(None, slots, x),
        lambda: attn.kv_write(cache, slots, x, [1.0]),
        lambda: attn.kv_write(cache, slots, [1.0], x),
        lambda: attn.kv_read(None, slots),
        lambda: attn.kv_read(cache, slots, k=[1.0]),
        lambda: attn.kv_read(cache, slots, v=3),
        lambda: attn.kv_read(cache, [0, 1]),
        lambda: attn.attn_decode(rand(1, 4, 32), None, slots.view(3, 1), slots),
        lambda: attn.attn_decode([1.0], cache, slots.view(3, 1), slots),
        lambda: attn.attn_decode(rand(3, 4, 32), cache, [[0]], slots),
        lambda: attn.attn_decode(rand(3, 4, 32), cache, slots.view(3, 1), [1]),
        lambda: attn.attn_decode(rand(3, 4, 32), cache, slots.view(3, 1), slots, out=[1.0]),
        lambda: attn.KVCache(None, None),
        lambda: attn.KVCache(cache.k, [1.0]),
        lambda: attn.split_heads([1.0], 1, 1, 1),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(H.HoardError):
            call()
            pytest.fail(str(i))

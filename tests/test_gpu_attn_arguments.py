"""Calls of the attention half on torch tensors that its documentation allows or refuses: one tensor for two arguments."""
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

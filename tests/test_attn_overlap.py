"""The check of tensors to write to against the inputs that a call goes on reading: no device is needed."""
import pytest

import hoard_amd as H

torch = pytest.importorskip("torch")


def test_one_tensor_twice():
    """What may be written over is one input, once: a second that is the same tensor is still read."""
    from hoard_amd import attn
    x, y = torch.zeros((3, 2, 16)), torch.zeros((3, 2, 16))
    attn._written("q_out", x, (x, y), x)
    attn._written("q_out", x, (None, x, y), x)
    attn._written("q_out", torch.zeros((3, 2, 16)), (x, x, y), x)
    for inputs in ((x, x), (x, y, x), (x, x.view(3, 2, 16)), (x, x[:, :1])):
        with pytest.raises(H.HoardError, match="q_out: overlaps"):
            attn._written("q_out", x, inputs, x)
    with pytest.raises(H.HoardError, match="overlaps"):
        attn._written("q_out", x, (y, x))

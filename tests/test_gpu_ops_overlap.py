"""A tensor to write to that overlaps an input is refused, except where the whole of one may be written over."""
import pytest

import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_overlaps():
    from hoard_amd import ops
    buf = torch.randn(8192, device="cuda")
    at = lambda first, *shape: buf[first:first + torch.Size(shape).numel()].view(*shape)  # noqa: E731
    w = ops.Q4Weight(torch.zeros((64, 32), dtype=torch.uint8, device="cuda"), torch.ones((64, 1), device="cuda"))
    ids = torch.tensor([[0, 1], [1, 2], [3, 0]], dtype=torch.int32, device="cuda")
    place = ops.sort_pairs(ids, 4).place
    wt, par = torch.rand((3, 2), device="cuda"), torch.ones(40, device="cuda")
    x, y = at(0, 3, 40), at(400, 6, 40)
    q = at(0, 4, 64)
    bad = {
        "q4 over x": lambda: ops.q4_matmul(q, w, out=q),
        "q4 beside x": lambda: ops.q4_matmul(q, w, out=at(192, 4, 64)),
        "gather": lambda: ops.sort_gather(x, place, out=at(100, 6, 40)),
        "combine over y": lambda: ops.sort_combine(y, place, wt, out=at(400, 3, 40)),
        "combine beside res": lambda: ops.sort_combine(y, place, wt, x, out=at(40, 3, 40)),
        "gradient over dout": lambda: ops.sort_combine_grad(x, y, place, wt, dy=at(0, 6, 40)),
        "gradient beside y": lambda: ops.sort_combine_grad(x, y, place, wt, dy=at(440, 6, 40)),
        "norm over b": lambda: ops.norm_forward(x, at(400, 3, 40), w_pre=par, eps=1e-6, r_out=at(400, 3, 40)),
        "norm beside r": lambda: ops.norm_forward(x, at(400, 3, 40), w_pre=par, eps=1e-6, r_out=at(39, 3, 40)),
    }
    kept = buf.clone()
    for name, call in bad.items():
        with pytest.raises(H.HoardError, match="overlaps"):
            call()
            pytest.fail(name)
    assert torch.equal(buf, kept)
    # side by side, and the whole of what may be written over
    ops.q4_matmul(q, w, out=at(256, 4, 64))
    ops.sort_combine(y, place, wt, x, out=x)
    ops.sort_combine_grad(x, y, place, wt, dy=y)
    ops.norm_forward(x, at(400, 3, 40), w_pre=par, eps=1e-6, r_out=x)


def test_what_is_no_tensor_is_refused_as_that():
    from hoard_amd import ops
    r, b, par = torch.randn((3, 40), device="cuda"), torch.randn((3, 40), device="cuda"), torch.ones(40, device="cuda")
    for kw in (dict(gate=[1.0] * 40), dict(gate=0.5), dict(w_post=[1.0] * 40)):
        with pytest.raises(H.HoardError):
            ops.norm_forward(r, b, w_pre=par, eps=1e-6, r_out=r, **kw)

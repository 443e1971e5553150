"""The operators on torch tensors beside autograd: no gradient is lost without a word."""
import pytest

import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def calls():
    """name -> (call over a dict of float tensors, those tensors)."""
    from hoard_amd import ops
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
    w = ops.Q4Weight(torch.randint(0, 256, (48, 32), generator=g, dtype=torch.uint8).cuda(), rand(48, 2))
    ids = torch.randint(0, 5, (6, 2), generator=g, dtype=torch.int32).cuda()
    place = ops.sort_pairs(ids, 5).place
    st = ops.norm_forward(rand(6, 40), rand(6, 40), rand(40), rand(40), rand(40), eps=1e-6, want_stats=True)
    n = dict(b=rand(6, 40), w_post=rand(40), gate=rand(40), w_pre=rand(40))
    return {
        "q4_matmul": (lambda t: ops.q4_matmul(t["x"], w, out=t["out"]), dict(x=rand(6, 64), out=rand(6, 48))),
        "sort_gather": (lambda t: ops.sort_gather(t["x"], place, t["w"], out=t["out"]), dict(x=rand(6, 40), w=rand(6, 2), out=rand(12, 40))),
        "sort_combine": (lambda t: ops.sort_combine(t["y"], place, t["w"], t["res"], out=t["out"]),
                         dict(y=rand(12, 40), w=rand(6, 2), res=rand(6, 40), out=rand(6, 40))),
        "sort_combine_grad": (lambda t: ops.sort_combine_grad(t["dout"], t["y"], place, t["w"], dy=t["dy"]),
                              dict(dout=rand(6, 40), y=rand(12, 40), w=rand(6, 2), dy=rand(12, 40))),
        "norm_forward": (lambda t: ops.norm_forward(t["r"], t["b"], t["w_post"], t["gate"], t["w_pre"], eps=1e-6, r_out=t["r_out"]),
                         dict(n, r=rand(6, 40), r_out=rand(6, 40))),
        "norm_backward": (lambda t: ops.norm_backward(st, t["dr_out"], t["dh"], t["b"], t["w_post"], t["gate"], t["w_pre"], eps=1e-6),
                          dict(n, dr_out=rand(6, 40), dh=rand(6, 40))),
    }


NAMES = ["q4_matmul", "sort_gather", "sort_combine", "sort_combine_grad", "norm_forward", "norm_backward"]


@pytest.mark.parametrize("name", NAMES)
def test_a_wanted_gradient_is_refused(calls, name):
    call, tensors = calls[name]
    call(tensors)
    for which in tensors:
        t = {k: v.clone().requires_grad_(k == which) for k, v in tensors.items()}
        with pytest.raises(H.HoardError, match=which + ": wants a gradient"):
            call(t)
        with torch.no_grad():
            call(t)
        call({k: v.detach() for k, v in t.items()})
    with torch.inference_mode():
        call({k: v.clone() for k, v in tensors.items()})


@pytest.mark.parametrize("name,out", [("q4_matmul", "out"), ("sort_gather", "out"), ("sort_combine", "out"), ("sort_combine_grad", "dy"),
                                      ("norm_forward", "r_out")])
def test_a_write_counts(calls, name, out):
    """A tensor that autograd keeps for a gradient and a call then writes over: backward refuses it."""
    call, tensors = calls[name]
    t = {k: v.clone() for k, v in tensors.items()}
    factor = torch.ones_like(t[out], requires_grad=True)
    product = (factor * t[out]).sum()
    call(t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


@pytest.mark.parametrize("name", NAMES)
def test_tensors_of_inference_mode(calls, name):
    """Buffers made in inference mode are written to outside it."""
    call, tensors = calls[name]
    with torch.inference_mode():
        t = {k: v.clone() for k, v in tensors.items()}
    call(t)

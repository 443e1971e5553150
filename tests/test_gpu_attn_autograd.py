"""The attention half's operators on torch tensors beside autograd, and tensors to write to that overlap inputs."""
import pytest

import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def calls():
    """name -> (call over a dict of float tensors, those tensors)."""
    from hoard_amd import attn
    g = torch.Generator().manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = attn.KVCache.new(4, 16, 2, 32, torch.float16)
    slots = dev([1, 17, 33])
    rope = attn.Rope(dev([5, 6, 7]), attn.rope_freq(16, 100.0))
    st = attn.heads_forward(rand(3, 4, 32), rand(3, 2, 32), w_q=rand(32), w_k=rand(32), want_stats=True)
    pages, lens = dev([[0, 1], [1, 2], [3, 0]]), dev([3, 20, 32])
    return {
        "heads_forward": (lambda t: attn.heads_forward(t["q"], t["k"], w_q=t["w_q"], w_k=t["w_k"], rope=rope, q_out=t["q_out"], k_out=t["k_out"]),
                          dict(q=rand(3, 4, 32), k=rand(3, 2, 32), w_q=rand(32), w_k=rand(32), q_out=rand(3, 4, 32), k_out=rand(3, 2, 32))),
        "with a cache": (lambda t: attn.heads_forward(k=t["k"], v=t["v"], cache=cache, slots=slots), dict(k=rand(3, 2, 32), v=rand(3, 2, 32))),
        "heads_backward": (lambda t: attn.heads_backward(t["dq_out"], t["dk_out"], q=t["q"], k=t["k"], w_q=t["w_q"], w_k=t["w_k"],
                                                         stats=st.stats, dq=t["dq"], dk=t["dk"]),
                           dict(q=rand(3, 4, 32), k=rand(3, 2, 32), w_q=rand(32), w_k=rand(32), dq_out=rand(3, 4, 32),
                                dk_out=rand(3, 2, 32), dq=rand(3, 4, 32), dk=rand(3, 2, 32))),
        "kv_write": (lambda t: attn.kv_write(cache, slots, t["k"], t["v"]), dict(k=rand(3, 2, 32), v=rand(3, 2, 32))),
        "kv_read": (lambda t: attn.kv_read(cache, slots, k=t["k"], v=t["v"]), dict(k=rand(3, 2, 32), v=rand(3, 2, 32))),
        "attn_decode": (lambda t: attn.attn_decode(t["q"], cache, pages, lens, out=t["out"]), dict(q=rand(3, 4, 32), out=rand(3, 4, 32))),
    }


NAMES = ["heads_forward", "with a cache", "heads_backward", "kv_write", "kv_read", "attn_decode"]


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


@pytest.mark.parametrize("name,out", [("heads_forward", "q_out"), ("heads_forward", "k_out"), ("heads_backward", "dq"), ("kv_read", "v"),
                                      ("attn_decode", "out")])
def test_a_write_counts(calls, name, out):
    """A tensor that autograd keeps for a gradient and a call then writes over: backward refuses it."""
    call, tensors = calls[name]
    t = {k: v.clone() for k, v in tensors.items()}
    factor = torch.ones_like(t[out], requires_grad=True)
    product = (factor * t[out]).sum()
    call(t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_a_write_to_the_cache_counts():
    from hoard_amd import attn
    cache = attn.KVCache.new(1, 16, 1, 16, torch.bfloat16)
    factor = torch.ones_like(cache.v, requires_grad=True)
    product = (factor * cache.v).sum()
    x = torch.randn((1, 1, 16), device="cuda")
    attn.kv_write(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), x, x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_overlaps():
    from hoard_amd import attn
    buf = torch.randn(8192, device="cuda")
    at = lambda first, *shape: buf[first:first + torch.Size(shape).numel()].view(*shape)  # noqa: E731
    q, k, v = attn.split_heads(at(0, 3, 8 * 32), 4, 2, 32)
    w = torch.ones(32, device="cuda")
    cache = attn.KVCache.new(2, 16, 2, 32, torch.float16)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    inside = cache.k.view(-1)[:192].view(3, 2, 32)
    bad = {
        "q_out over k": lambda: attn.heads_forward(q, k, q_out=at(0, 3, 4, 32)),
        "k_out over q": lambda: attn.heads_forward(q, k, k_out=q[:, 1:3]),
        "k_out over q_out": lambda: attn.heads_forward(q, k, q_out=at(2000, 3, 4, 32), k_out=at(2100, 3, 2, 32)),
        "k_out beside v": lambda: attn.heads_forward(q, k, v, cache=cache, slots=slots, k_out=at(130, 3, 2, 32)),
        "dq over q": lambda: attn.heads_backward(at(4000, 3, 4, 32), q=q, w_q=w, stats=torch.ones((3, 4), device="cuda"), dq=q),
        "dk over dq": lambda: attn.heads_backward(at(4000, 3, 4, 32), at(4500, 3, 2, 32), dq=at(5000, 3, 4, 32), dk=at(5100, 3, 2, 32)),
        "write from the cache": lambda: attn.kv_write(cache, slots, inside),
        "read into the cache": lambda: attn.kv_read(cache, slots, k=inside),
        "v over k": lambda: attn.kv_read(cache, slots, k=at(0, 3, 2, 32), v=at(100, 3, 2, 32)),
        "out over q": lambda: attn.attn_decode(at(0, 3, 4, 32), cache, slots.view(3, 1), slots, out=at(64, 3, 4, 32)),
    }
    kept = buf.clone()
    for name, call in bad.items():
        with pytest.raises(H.HoardError, match="overlaps"):
            call()
            pytest.fail(name)
    torch.cuda.synchronize()
    assert torch.equal(buf, kept)
    # other columns of the same rows, and the whole of what may be written over
    attn.heads_forward(q, k, w_q=w, q_out=q, k_out=k)
    attn.heads_forward(q, k, k_out=v)
    d = at(4000, 3, 4, 32)
    attn.heads_backward(d, dq=d)


def test_what_does_not_fit_is_refused():
    from hoard_amd import attn
    r = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    cache = attn.KVCache.new(2, 16, 2, 32, torch.float16)
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    rope = attn.Rope(slots, attn.rope_freq(16, 100.0))
    bad = [
        lambda: attn.heads_forward(r(3, 4, 32), r(2, 2, 32)),
        lambda: attn.heads_forward(r(3, 4, 32), r(3, 2, 64)),
        lambda: attn.heads_forward(r(3, 4, 32), r(3, 2, 32).half()),
        lambda: attn.heads_forward(r(3, 128)),
        lambda: attn.heads_forward(),
        lambda: attn.heads_forward([1.0]),
        lambda: attn.heads_forward(r(3, 4, 32), w_q=r(31)),
        lambda: attn.heads_forward(r(3, 4, 32), w_k=r(32)),
        lambda: attn.heads_forward(r(3, 4, 32), v=r(3, 2, 32)),
        lambda: attn.heads_forward(r(3, 4, 32), slots=slots),
        lambda: attn.heads_forward(k=r(3, 2, 32), cache=cache),
        lambda: attn.heads_forward(k=r(3, 4, 32), cache=cache, slots=slots),
        lambda: attn.heads_forward(r(3, 4, 32), rope=rope._replace(pos=slots.long())),
        lambda: attn.heads_forward(r(3, 4, 32), rope=rope._replace(freq=rope.freq.float())),
        lambda: attn.heads_forward(r(3, 4, 32), rope=rope._replace(pos=slots[:2])),
        lambda: attn.heads_forward(r(3, 4, 32), rope=rope._replace(axis=slots)),
        lambda: attn.heads_forward(r(3, 4, 8), rope=rope),
        lambda: attn.heads_forward(r(3, 4, 12)),
        lambda: attn.heads_forward(r(3, 4, 32).cpu()),
        lambda: attn.heads_forward(r(3, 4, 32), q_out=r(3, 4, 31)),
        lambda: attn.heads_forward(r(3, 32, 4).transpose(1, 2)),
        lambda: attn.heads_forward(r(1, 4, 32).expand(3, 4, 32)),
        lambda: attn.heads_backward(),
        lambda: attn.heads_backward(r(3, 4, 32), w_q=r(32)),
        lambda: attn.heads_backward(r(3, 4, 32), q=r(3, 4, 32), w_q=r(32)),
        lambda: attn.heads_backward(r(3, 4, 32), dk=r(3, 2, 32)),
        lambda: attn.kv_write(cache, slots),
        lambda: attn.kv_write(cache, slots[:2], r(3, 2, 32)),
        lambda: attn.kv_read(cache, slots.long()),
        lambda: attn.kv_read(cache, slots, torch.float64),
        lambda: attn.split_heads(r(3, 100), 4, 2, 32),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(H.HoardError):
            call()
            pytest.fail(str(i))


def test_another_device_or_stream_than_the_current():
    """Tensors made on one stream and used on another that waits for it."""
    from hoard_amd import attn
    side = torch.cuda.Stream()
    q = torch.randn((64, 8, 128), device="cuda")
    w = torch.ones(128, device="cuda")
    want = attn.heads_forward(q, w_q=w).q_out
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attn.heads_forward(q, w_q=w).q_out
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)

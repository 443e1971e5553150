"""Heads normed, rotated and written to the cache, and their gradients, against 64 bits."""
import pytest

import attnref as A
import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8
EPS = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rope_of(m, rot, seed, axes=1, pairs=False, far=0):
    from hoard_amd import attn
    if not rot:
        return None
    pos = torch.randint(0, 5000, (axes, m), generator=gen(seed)) + far
    axis = (torch.arange(rot // 2) % 3).to(torch.uint8).cuda() if axes > 1 else None
    return attn.Rope(pos.to(torch.int32).cuda() if axes > 1 else pos[0].to(torch.int32).cuda(), attn.rope_freq(rot, 1e6), axis, pairs)


def make(m, hq, hkv, d, dtype, seed, fused=True):
    from hoard_amd import attn
    qkv = torch.randn((m, (hq + 2 * hkv) * d), generator=gen(seed)).to(dtype).cuda()
    q, k, v = attn.split_heads(qkv, hq, hkv, d)
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


def weight(d, seed, offset):
    return (1.0 - offset + 0.3 * torch.randn(d, generator=gen(seed))).cuda()


# tokens, query heads, key heads, dim, rotated, type, pairs, axes, offset, first position
SHAPES = [
    (1, 32, 4, 128, 128, F32, False, 1, 0.0, 8191),
    (3, 16, 2, 256, 64, F16, False, 3, 1.0, 0),
    (5, 5, 1, 64, 64, BF16, True, 1, 0.0, 900000),
    (7, 3, 3, 96, 24, F32, False, 1, 0.0, 0),
    (2, 4, 2, 96, 96, BF16, True, 2, 0.0, 0),
    (4, 6, 2, 192, 96, F16, False, 1, 0.5, 77),
    (9, 1, 1, 8, 8, F32, False, 1, 0.0, 0),
    (9, 2, 1, 16, 8, F16, True, 1, 0.0, 0),
    (9, 7, 1, 40, 0, F32, False, 1, 0.0, 0),
    (33, 2, 2, 248, 240, BF16, False, 1, 0.0, 0),
    (700, 16, 16, 128, 128, BF16, False, 1, 0.0, 0),
    (1500, 8, 1, 64, 32, F32, False, 1, 0.0, 0),
]


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,pairs,axes,offset,far", SHAPES)
def test_forward(m, hq, hkv, d, rot, dtype, pairs, axes, offset, far, normed):
    from hoard_amd import attn
    q, k, _ = make(m, hq, hkv, d, dtype, 1)
    rope = rope_of(m, rot, 2, axes, pairs, far)
    w_q, w_k = (weight(d, 3, offset), weight(d, 4, offset)) if normed else (None, None)
    st = attn.heads_forward(q, k, w_q=w_q, w_k=w_k, rope=rope, eps=EPS, w_offset=offset, want_stats=True)
    for x, w, out, at in ((q, w_q, st.q_out, slice(0, hq)), (k, w_k, st.k_out, slice(hq, hq + hkv))):
        want, bound, rho = A.heads(x, w, rope, EPS, offset)
        A.close(out, want, A.stored(want, bound, dtype), "heads")
        A.close(st.stats[:, at], rho, rho * (d / 2 + 8) * A.U32, "stats")
    # in place, in the projection's rows, whose values stay
    qkv = torch.randn((m, (hq + 2 * hkv) * d), generator=gen(1)).to(dtype).cuda()
    kept = qkv.clone()
    q, k, v = attn.split_heads(qkv, hq, hkv, d)
    got = attn.heads_forward(q, k, w_q=w_q, w_k=w_k, rope=rope, eps=EPS, w_offset=offset, q_out=q, k_out=k)
    assert got.q_out is q and torch.equal(q, st.q_out) and torch.equal(k, st.k_out)
    assert torch.equal(qkv[:, (hq + hkv) * d:], kept[:, (hq + hkv) * d:])
    # one of the two alone, one of the two normed
    alone = attn.heads_forward(k=attn.split_heads(kept, hq, hkv, d)[1], w_k=w_k, rope=rope, eps=EPS, w_offset=offset)
    assert alone.q_out is None and torch.equal(alone.k_out, st.k_out)


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,pairs,axes,offset,far", SHAPES)
def test_backward(m, hq, hkv, d, rot, dtype, pairs, axes, offset, far, normed):
    from hoard_amd import attn
    q, k, _ = make(m, hq, hkv, d, dtype, 5)
    rope = rope_of(m, rot, 6, axes, pairs, far)
    w_q, w_k = (weight(d, 7, offset), weight(d, 8, offset)) if normed else (None, None)
    args = dict(w_q=w_q, w_k=w_k, rope=rope, eps=EPS, w_offset=offset)
    st = attn.heads_forward(q, k, want_stats=True, **args)
    dq_out, dk_out = (torch.randn(t.shape, generator=gen(9)).to(dtype).cuda() for t in (q, k))
    got = attn.heads_backward(dq_out, dk_out, q=q, k=k, stats=st.stats, **args)
    for name, x, dz, w, dx, dw, at in (("q", q, dq_out, w_q, got.dq, got.dw_q, slice(0, hq)),
                                       ("k", k, dk_out, w_k, got.dk, got.dw_k, slice(hq, hq + hkv))):
        want, bound, want_w, bound_w = A.heads_grad(dz, x, w, rope, st.stats[:, at], offset)
        A.close(dx, want, A.stored(want, bound, dtype), "d" + name)
        if w is not None:
            A.close(dw, want_w, bound_w, "dw_" + name)
    again = attn.heads_backward(dq_out.clone(), dk_out.clone(), q=q, k=k, stats=st.stats, **args)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a, b)
    # into the projection's gradient, and over what it is the gradient of
    dqkv = torch.zeros((m, (hq + 2 * hkv) * d), dtype=dtype, device="cuda")
    dq, dk, dv = attn.split_heads(dqkv, hq, hkv, d)
    attn.heads_backward(dq_out, dk_out, q=q, k=k, stats=st.stats, dq=dq, dk=dk, **args)
    assert torch.equal(dq, got.dq) and torch.equal(dk, got.dk) and not dv.any()
    over = dq_out.clone()
    assert attn.heads_backward(over, dk_out, q=q, k=k, stats=st.stats, dq=over, **args).dq is over
    assert torch.equal(over, got.dq)
    if normed:  # one of the two alone
        alone = attn.heads_backward(None, dk_out, q=q, k=k, w_k=w_k, rope=rope, eps=EPS, w_offset=offset, stats=st.stats)
        assert alone.dq is None and torch.equal(alone.dk, got.dk)
        A.close(alone.dw_k, want_w, bound_w, "dw_k alone")  # its terms are added in another order


def test_gradient_by_differences():
    """The chain q -> out against a 64-bit difference along a direction."""
    from hoard_amd import attn
    m, h, d = 6, 3, 64
    g = gen(11)
    q, w, dz = torch.randn((m, h, d), generator=g), 1 + 0.2 * torch.randn(d, generator=g), torch.randn((m, h, d), generator=g)
    rope = rope_of(m, 32, 12, pairs=True)
    st = attn.heads_forward(q.cuda(), w_q=w.cuda(), rope=rope, eps=EPS, want_stats=True)
    got = attn.heads_backward(dz.cuda(), q=q.cuda(), w_q=w.cuda(), rope=rope, eps=EPS, stats=st.stats)
    dir_q, dir_w = torch.randn((m, h, d), generator=g, dtype=A.D), torch.randn(d, generator=g, dtype=A.D)

    def loss(t):
        return (A.heads(q.to(A.D) + t * dir_q, w.to(A.D) + t * dir_w, rope, EPS, 0.0)[0] * dz.to(A.D)).sum()

    diff = float(loss(1e-5) - loss(-1e-5)) / 2e-5
    tq, tw = A.t64(got.dq) * dir_q, A.t64(got.dw_q) * dir_w
    # some 100 roundings of sums whose magnitudes are up to 10 times the gradients', and the step's square
    assert abs(diff - float(tq.sum() + tw.sum())) <= (1000 * A.U32 + 1e-8) * float(tq.abs().sum() + tw.abs().sum())


def test_far_positions():
    """Positions of 2^31 - 1 and negative ones: their angle modulo a turn."""
    from hoard_amd import attn
    pos = torch.tensor([2 ** 31 - 1, -(2 ** 31), 123456789, -7], dtype=torch.int32, device="cuda")
    rope = attn.Rope(pos, attn.rope_freq(64, 10000.0))
    q = torch.randn((4, 2, 64), generator=gen(13)).cuda()
    want, bound, _ = A.heads(q, None, rope, EPS, 0.0)
    A.close(attn.heads_forward(q, rope=rope).q_out, want, A.stored(want, bound, F32), "far")


def test_an_axis_past_the_last():
    from hoard_amd import attn
    pos = torch.randint(0, 100, (2, 5), generator=gen(14), dtype=torch.int32).cuda()
    axis = torch.tensor([0, 1, 2, 255], dtype=torch.uint8, device="cuda")
    q = torch.randn((5, 1, 8), generator=gen(15)).cuda()
    rope = attn.Rope(pos, attn.rope_freq(8, 100.0), axis)
    a = attn.heads_forward(q, rope=rope).q_out
    b = attn.heads_forward(q, rope=rope._replace(axis=axis.clamp(max=1))).q_out
    assert torch.equal(a, b)


def test_infinities_stay_in_their_head():
    from hoard_amd import attn
    q = torch.randn((4, 3, 64), generator=gen(16))
    q[1, 2, 5] = float("inf")
    q[2, 0, 63] = float("nan")
    rope = rope_of(4, 64, 17)
    w = weight(64, 18, 0.0)
    for kw in (dict(), dict(w_q=w)):
        got = attn.heads_forward(q.cuda(), rope=rope, **kw).q_out.cpu()
        clean = attn.heads_forward(torch.where(torch.isfinite(q), q, 0.5).cuda(), rope=rope, **kw).q_out.cpu()
        keep = torch.ones((4, 3), dtype=torch.bool)
        keep[1, 2] = keep[2, 0] = False
        assert torch.equal(got[keep], clean[keep])
        assert not torch.isfinite(got[1, 2]).all() and got[2, 0].isnan().any()


def test_no_tokens():
    from hoard_amd import attn
    q, k, v = make(0, 4, 2, 64, F32, 1)
    w = weight(64, 1, 0.0)
    cache = attn.KVCache.new(2, 16, 2, 64, F16)
    slots = torch.empty(0, dtype=torch.int32, device="cuda")
    assert attn.heads_forward(q, k, v, w_q=w, w_k=w, cache=cache, slots=slots).q_out.shape == (0, 4, 64)
    attn.kv_write(cache, slots, k, v)
    assert attn.kv_read(cache, slots)[0].shape == (0, 2, 64)
    got = attn.heads_backward(q, k, q=q, k=k, w_q=w, w_k=w, stats=torch.empty((0, 6), device="cuda"))
    assert got.dq.shape == (0, 4, 64) and not got.dw_q.any() and not got.dw_k.any()
    assert not cache.k.any()


# -- the cache ------------------------------------------------------------------------

def slots_of(m, cache, seed, drop=0.0):
    s = torch.randperm(cache.n_pages * cache.page, generator=gen(seed))[:m].to(torch.int32)
    lost = torch.rand(m, generator=gen(seed + 1)) < drop
    s = torch.where(lost, torch.where(torch.arange(m) % 2 == 0, -1 - s, cache.n_pages * cache.page + s), s)
    return s.cuda(), ~lost


def rows_of(cache, slots):
    """(k, v) rows [tokens, heads, ...] of a cache's tensors at slots on the CPU."""
    p, o = slots.cpu().long() // cache.page, slots.cpu().long() % cache.page
    return [t.cpu()[p, :, o] if t is not None else None for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("m,heads,d,page", [(1, 4, 128, 64), (13, 2, 256, 16), (40, 3, 96, 32), (37, 1, 16, 128), (300, 5, 80, 256)])
def test_write_and_read(m, heads, d, page, ct, dtype, fused):
    from hoard_amd import attn
    _, k, v = make(m, 2, heads, d, dtype, 21, fused)
    k = k * 3.0 if not fused else k
    cache = attn.KVCache.new(m // page + 3, page, heads, d, ct)
    for t in cache._tensors():
        t.fill_(77)
    before = [t.clone() for t in cache._tensors()]
    slots, kept = slots_of(m, cache, 22, 0.2)
    attn.kv_write(cache, slots, k, v)
    rows = rows_of(cache, slots[kept.cuda()])
    for x, codes, scale in ((k, rows[0], rows[2]), (v, rows[1], rows[3])):
        x = x.cpu()[kept]
        if ct == I8:
            q, step = A.quantised(x)
            assert torch.equal(codes, q) and torch.equal(scale, step)
            assert ((A.values(codes, scale) - A.t64(x)).abs() <= 0.5001 * A.t64(step).unsqueeze(-1)).all()
        else:
            assert torch.equal(codes, x.to(torch.float32).to(ct))
    # nothing else was written
    p, o = slots.cpu().long()[kept] // page, slots.cpu().long()[kept] % page
    for t, b in zip(cache._tensors(), before):
        t, b = t.cpu(), b.cpu()
        b[p, :, o] = t[p, :, o]
        assert torch.equal(t, b)
    # and back, in each type; rows of dropped tokens stay
    for to in (F32, F16, BF16):
        out = [torch.full((m, 2, heads, d), 5.0, dtype=to, device="cuda")[:, i] for i in range(2)]
        attn.kv_read(cache, slots, k=out[0], v=out[1])
        for got, codes, scale in ((out[0], rows[0], rows[2]), (out[1], rows[1], rows[3])):
            want = codes.to(torch.float32) if scale is None else scale.unsqueeze(-1) * codes.to(torch.float32)
            assert torch.equal(got.cpu()[kept], want.to(to)) and (got.cpu()[~kept] == 5.0).all()
    # one of the two alone
    lone = attn.KVCache.new(cache.n_pages, page, heads, d, ct)
    attn.kv_write(lone, slots, v=v)
    assert not lone.k.any() and torch.equal(rows_of(lone, slots[kept.cuda()])[1], rows[1])


@pytest.mark.parametrize("ct", [F16, I8])
def test_rows_of_zeros_infinities_and_tiny_values(ct):
    from hoard_amd import attn
    d = 64
    x = torch.randn((8, 2, d), generator=gen(31))
    x[0] = 0.0
    x[1, 0, 3] = float("inf")
    x[2, 1, 60] = float("nan")
    x[3] *= 1e-38
    x[4] = 0.0
    x[4, :, 7] = -1e-45
    x[5] *= 1e37
    x[6, 0] = 127.0
    x[6, 0, 1] = -127.0
    cache = attn.KVCache.new(1, 16, 2, d, ct)
    slots = torch.arange(8, dtype=torch.int32, device="cuda")
    attn.kv_write(cache, slots, x.cuda(), x.cuda())
    k, _ = attn.kv_read(cache, slots, F32)
    codes, step = A.quantised(x)
    want = step.unsqueeze(-1) * codes.to(F32) if ct == I8 else x.to(F16).to(F32)
    assert torch.equal(k.cpu().nan_to_num(nan=1e30), want.nan_to_num(nan=1e30))
    if ct == I8:
        assert k[1, 0].isnan().all() and k[2, 1].isnan().all() and torch.isfinite(k[1, 1]).all() and not k[0].any()
        assert torch.equal(rows_of(cache, slots)[0], codes)


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,pairs,axes,offset,far", [s for s in SHAPES if s[3] % 16 == 0])
def test_forward_into_the_cache(m, hq, hkv, d, rot, dtype, pairs, axes, offset, far, ct):
    """The same values that heads_forward gives in fp32, written as kv_write does."""
    from hoard_amd import attn
    q, k, v = make(m, hq, hkv, d, dtype, 41)
    rope = rope_of(m, rot, 42, axes, pairs, far)
    args = dict(w_q=weight(d, 43, offset), w_k=weight(d, 44, offset), rope=rope, eps=EPS, w_offset=offset)
    cache, other = (attn.KVCache.new(m // 16 + 2, 16, hkv, d, ct) for _ in range(2))
    slots, kept = slots_of(m, cache, 45, 0.1)
    st = attn.heads_forward(q, k, v, cache=cache, slots=slots, k_out=torch.empty(k.shape, dtype=dtype, device="cuda"), **args)
    plain = attn.heads_forward(q, k, **args)
    assert torch.equal(st.q_out, plain.q_out) and torch.equal(st.k_out, plain.k_out)
    wide = attn.heads_forward(k=k.to(F32), w_k=args["w_k"], rope=rope, eps=EPS, w_offset=offset).k_out
    attn.kv_write(other, slots, wide, v.to(F32))
    for a, b in zip(cache._tensors(), other._tensors()):
        assert torch.equal(a, b)
    assert attn.heads_forward(q, k, v, cache=cache, slots=slots, **args).k_out is None


def test_beyond_32_bits():
    """A cache and rows whose offsets pass 2^32 bytes."""
    from hoard_amd import attn
    heads, d, page = 16, 256, 256
    pages = (5 << 30) // (heads * d * page) + 1  # more than 5 GiB of codes each
    cache = attn.KVCache.new(pages, page, heads, d, I8)
    m, step = 9, (1 << 31) // 4
    slots = (torch.arange(m) * (pages * page // m - 1) + 3).to(torch.int32).cuda()
    slots[-1] = pages * page - 1
    big = torch.zeros((m - 1) * step + 2 * heads * d, dtype=F16, device="cuda")
    k = big.as_strided((m, heads, d), (step, d, 1))
    v = big[heads * d:].as_strided((m, heads, d), (step, d, 1))
    k.copy_(torch.randn((m, heads, d), generator=gen(51)))
    v.copy_(torch.randn((m, heads, d), generator=gen(52)))
    attn.heads_forward(k=k, v=v, cache=cache, slots=slots)
    assert (m - 1) * step * 2 > 1 << 32 and cache.k.numel() > 1 << 32
    p, o = slots.long() // page, slots.long() % page
    for x, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        q, st = A.quantised(x)
        assert torch.equal(codes[p, :, o].cpu(), q) and torch.equal(scale[p, :, o].cpu(), st)
    assert int((cache.k_scale != 0).sum()) == m * heads
    got, _ = attn.kv_read(cache, slots, F16)
    assert torch.equal(got, (cache.k_scale[p, :, o].unsqueeze(-1) * cache.k[p, :, o].float()).to(F16))
    out = attn.heads_forward(k=k, k_out=k, w_k=torch.ones(d, device="cuda")).k_out
    want, bound, _ = A.heads(got * 0 + torch.randn((m, heads, d), generator=gen(51)).to(F16).cuda(), torch.ones(d), None, EPS, 0.0)
    A.close(out, want, A.stored(want, bound, F16), "far rows")


# -- graphs and streams ------------------------------------------------------------------

def test_graph_and_streams():
    from hoard_amd import attn
    m, hq, hkv, d = 200, 8, 2, 128
    qkv = torch.randn((m, (hq + 2 * hkv) * d), generator=gen(61)).to(BF16).cuda()
    q, k, v = attn.split_heads(qkv, hq, hkv, d)
    w = weight(d, 62, 0.0)
    rope = rope_of(m, d, 63)
    cache = attn.KVCache.new(m // 16 + 2, 16, hkv, d, I8)
    slots, _ = slots_of(m, cache, 64)
    args = dict(w_q=w, w_k=w, rope=rope)

    def step():
        st = attn.heads_forward(q, k, v, cache=cache, slots=slots, want_stats=True, **args)
        g = attn.heads_backward(st.q_out, st.q_out[:, :hkv].contiguous(), q=q, k=k, stats=st.stats, **args)
        return (st.q_out, *g, *attn.kv_read(cache, slots), *cache._tensors())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for turn in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), turn
        eager = [t.clone() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(eager, want))
        torch.cuda.synchronize()

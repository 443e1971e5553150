"""Heads and cache rows of more tokens than there are waves, and past the caches: each row as in calls of few tokens."""
import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8
EPS = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(m, hq, hkv, d, rot, dtype, axes, offset):
    from hoard_amd import attn
    qkv = torch.randn((m, (hq + 2 * hkv) * d), generator=gen(1)).to(dtype).cuda()
    w = [(1.0 - offset + 0.3 * torch.randn(d, generator=gen(s))).cuda() for s in (2, 3)]
    pos = torch.randint(0, 5000, (axes, m), generator=gen(4), dtype=torch.int32).cuda()
    axis = (torch.arange(rot // 2) % axes).to(torch.uint8).cuda()
    return qkv, attn.split_heads(qkv, hq, hkv, d), w, attn.Rope(pos, attn.rope_freq(rot, 1e6), axis)


def parts(m, step=2500):
    return [slice(i, min(i + step, m)) for i in range(0, m, step)]


# tokens, query heads, key heads, dim, rotated, type, axes, offset: above 6144 tokens each wave takes several (the
# gradient's from fewer on), from 64 MB of heads on they go past the caches
SHAPES = [
    (12301, 3, 1, 64, 32, F32, 1, 0.0),
    (6149, 2, 2, 96, 96, BF16, 3, 1.0),
    (20003, 1, 1, 16, 8, F16, 1, 0.0),
    (6500, 4, 1, 256, 64, F16, 2, 0.0),
    (9001, 12, 4, 128, 128, F32, 1, 0.0),   # 74 MB
    (14701, 16, 2, 128, 64, BF16, 2, 1.0),  # 68 MB
    (9203, 7, 8, 248, 128, F16, 1, 0.0),    # 68 MB, lanes without values
]


@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,axes,offset", SHAPES)
def test_forward(m, hq, hkv, d, rot, dtype, axes, offset):
    from hoard_amd import attn
    qkv, (q, k, v), w, rope = make(m, hq, hkv, d, rot, dtype, axes, offset)
    args = dict(w_q=w[0], w_k=w[1], eps=EPS, w_offset=offset)
    st = attn.heads_forward(q, k, rope=rope, want_stats=True, **args)
    for at in parts(m):
        few = attn.heads_forward(q[at], k[at], rope=rope._replace(pos=rope.pos[:, at].contiguous()), want_stats=True, **args)
        assert torch.equal(st.q_out[at], few.q_out) and torch.equal(st.k_out[at], few.k_out) and torch.equal(st.stats[at], few.stats)
    some = torch.cat([torch.arange(0, m, 97), torch.tensor([m - 1])])
    for x, out, wx in ((q, st.q_out, w[0]), (k, st.k_out, w[1])):
        want, bound, _ = A.heads(x[some.cuda()], wx, (rope.pos[:, some.cuda()].cpu(), rope.freq, rope.axis, False), EPS, offset)
        A.close(out[some.cuda()], want, A.stored(want, bound, dtype), "heads")
    kept = v.clone()
    attn.heads_forward(q, k, rope=rope, q_out=q, k_out=k, **args)
    assert torch.equal(q, st.q_out) and torch.equal(k, st.k_out) and torch.equal(v, kept)


@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,axes,offset", SHAPES)
def test_backward(m, hq, hkv, d, rot, dtype, axes, offset):
    from hoard_amd import attn
    _, (q, k, _), w, rope = make(m, hq, hkv, d, rot, dtype, axes, offset)
    args = dict(w_q=w[0], w_k=w[1], eps=EPS, w_offset=offset)
    stats = attn.heads_forward(q, k, rope=rope, want_stats=True, **args).stats
    dq_out, dk_out = (torch.randn(t.shape, generator=gen(5)).to(dtype).cuda() for t in (q, k))
    got = attn.heads_backward(dq_out, dk_out, q=q, k=k, rope=rope, stats=stats, **args)
    for at in parts(m, 800):
        few = attn.heads_backward(dq_out[at], dk_out[at], q=q[at], k=k[at], rope=rope._replace(pos=rope.pos[:, at].contiguous()),
                                  stats=stats[at], **args)
        assert torch.equal(got.dq[at], few.dq) and torch.equal(got.dk[at], few.dk)
    cpu = rope.pos.cpu(), rope.freq, rope.axis, False
    for dz, x, wx, rho, dw in ((dq_out, q, w[0], stats[:, :hq], got.dw_q), (dk_out, k, w[1], stats[:, hq:], got.dw_k)):
        want, bound = 0.0, 0.0
        for h in range(x.shape[1]):
            _, _, one, e = A.heads_grad(dz[:, h:h + 1], x[:, h:h + 1], wx, cpu, rho[:, h:h + 1], offset)
            want, bound = want + one, bound + e
        A.close(dw, want, bound * x.shape[1], "dw")  # a sum over all heads rounds that many times more
        # and by its mean square, where roundings do not add up: a token left out is far more
        assert (A.t64(dw) - want).norm() <= 1e-5 * want.norm() + 1e-6 * (m * x.shape[1] * d) ** 0.5
    again = attn.heads_backward(dq_out, dk_out, q=q, k=k, rope=rope, stats=stats, **args)
    assert torch.equal(again.dw_q, got.dw_q) and torch.equal(again.dw_k, got.dw_k)
    attn.heads_backward(dq_out, dk_out, q=q, k=k, rope=rope, stats=stats, dq=dq_out, dk=dk_out, **args)
    assert torch.equal(dq_out, got.dq) and torch.equal(dk_out, got.dk)


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("m,hq,hkv,d,rot,dtype,axes,offset", [SHAPES[i] for i in (0, 1, 2, 5)])
def test_cache(m, hq, hkv, d, rot, dtype, axes, offset, ct):
    from hoard_amd import attn
    _, (q, k, v), w, rope = make(m, hq, hkv, d, rot, dtype, axes, offset)
    args = dict(w_q=w[0], w_k=w[1], eps=EPS, w_offset=offset)
    cache, few = (attn.KVCache.new(m // 16 + 9, 16, hkv, d, ct) for _ in range(2))
    slots = torch.randperm(cache.n_pages * 16, generator=gen(6))[:m].to(torch.int32)
    slots[::7] = -1
    slots = slots.cuda()
    st = attn.heads_forward(q, k, v, rope=rope, cache=cache, slots=slots, **args)
    for at in parts(m):
        one = attn.heads_forward(q[at], k[at], v[at], rope=rope._replace(pos=rope.pos[:, at].contiguous()), cache=few,
                                 slots=slots[at], **args)
        assert torch.equal(st.q_out[at], one.q_out)
    for a, b in zip(cache._tensors(), few._tensors()):
        assert torch.equal(a, b)
    out = [torch.full((m, hkv, d), 3.0, dtype=F32, device="cuda") for _ in range(2)]
    attn.kv_read(cache, slots, k=out[0], v=out[1])
    kept = slots >= 0
    p, o = slots[kept].long() // 16, slots[kept].long() % 16
    for got, x, s in ((out[0], cache.k, cache.k_scale), (out[1], cache.v, cache.v_scale)):
        want = x[p, :, o].to(F32) if s is None else s[p, :, o].unsqueeze(-1) * x[p, :, o].to(F32)
        assert torch.equal(got[kept], want) and (got[~kept] == 3.0).all()
    # values as they are, in 32 bits and rounded once
    if ct != I8:
        assert torch.equal(cache.v[p, :, o], v[kept].to(F32).to(ct))

"""Attention of new tokens over a paged cache, against 64 bits."""
import math

import pytest

import attnref as A
import hoard_amd as H

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cache_of(pages, page, heads, d, ct, seed, v_size=1.0):
    """A cache whose every place holds values."""
    from hoard_amd import attn
    c = attn.KVCache.new(pages, page, heads, d, ct)
    slots = torch.arange(pages * page, dtype=torch.int32, device="cuda")
    x = torch.randn((2, pages * page, heads, d), generator=gen(seed))
    attn.kv_write(c, slots, x[0].cuda(), (x[1] * v_size).cuda())
    return c


def table(n_seq, width, pages, seed):
    return torch.stack([torch.randperm(pages, generator=gen(seed + i))[:width] for i in range(n_seq)]).to(torch.int32).cuda()


def check(q, c, pages, lens, scale=None, **kw):
    from hoard_amd import attn
    got = attn.attn_decode(q, c, pages, lens, scale=scale, want_lse=True, **kw)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    # the scale is an argument of 32 bits
    want, bound, lse, lse_bound = A.attention(q, c.k, c.v, c.k_scale, c.v_scale, pages, lens,
                                              float(torch.tensor(scale, dtype=F32)), q.dtype)
    A.close(got.out, want, A.stored(want, bound, q.dtype), "out")
    seen = lse > -math.inf
    assert torch.equal(torch.isneginf(got.lse.cpu()), ~seen)
    A.close(got.lse.cpu()[seen], lse[seen], A.stored(lse, lse_bound, F32)[seen], "lse")
    return got


# sequences, new tokens, query heads, key heads, dim, page, longest
SHAPES = [
    (1, 1, 32, 4, 128, 64, 257),
    (2, 1, 16, 2, 256, 32, 70),
    (3, 1, 4, 4, 64, 16, 130),
    (1, 1, 16, 16, 128, 16, 33),
    (2, 5, 16, 2, 256, 16, 100),
    (1, 16, 8, 1, 128, 64, 300),
    (2, 3, 5, 1, 96, 32, 90),
    (1, 2, 6, 2, 80, 128, 200),
    (1, 1, 3, 1, 16, 16, 40),
    (1, 1, 2, 1, 192, 256, 600),
    (2, 7, 20, 4, 128, 16, 65),
    (1, 64, 2, 1, 64, 16, 100),
    (1, 1, 64, 2, 112, 16, 50),
    (5, 1, 8, 2, 48, 16, 31),
]


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,t,hq,hkv,d,page,longest", SHAPES)
def test_shapes(n, t, hq, hkv, d, page, longest, dtype, ct):
    width = -(-longest // page) + 1
    c = cache_of(n * width + 3, page, hkv, d, ct, 1)
    q = (2.0 * torch.randn((n * t, hq, d), generator=gen(2))).to(dtype).cuda()
    lens = torch.randint(1, longest + 1, (n, t), generator=gen(3), dtype=torch.int32)
    lens[0] = longest - t + 1 + torch.arange(t)
    lens = lens.clamp(min=0).cuda()
    check(q, c, table(n, width, c.n_pages, 4), lens if t > 1 else lens.view(n))


@pytest.mark.parametrize("ct", [BF16, I8])
@pytest.mark.parametrize("n", list(range(0, 36)) + [63, 64, 65, 127, 128, 129, 191, 193, 255, 256, 257, 511, 513])
def test_lengths(n, ct):
    """Every length around the runs of keys, the longer ones in one batch of both."""
    c = cache_of(40, 16, 2, 64, ct, 11)
    q = torch.randn((2, 4, 64), generator=gen(12)).to(BF16).cuda()
    lens = torch.tensor([n, max(n - 1, 0)], dtype=torch.int32, device="cuda")
    got = check(q, c, table(2, 33, 40, 13), lens)
    if n == 0:
        assert not got.out.any() and torch.isneginf(got.lse).all()


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("longest", [2000, 5003])
def test_long(longest, dtype, ct):
    """A length that is split over many workgroups, beside short ones of the same call."""
    page = 64
    width = -(-longest // page)
    c = cache_of(width + 10, page, 1, 128, ct, 21)
    q = (2.0 * torch.randn((4, 8, 128), generator=gen(22))).to(dtype).cuda()
    lens = torch.tensor([longest, 0, 1, longest // 3], dtype=torch.int32, device="cuda")
    check(q, c, table(4, width, c.n_pages, 23), lens)


@pytest.mark.parametrize("ct", [F16, BF16, I8])
def test_what_is_not_seen_may_hold_anything(ct):
    """NaN and infinities behind a row's last key, in other pages, and for rows that see fewer keys than others."""
    from hoard_amd import attn
    page, hkv, d, t = 16, 2, 64, 4
    c = cache_of(12, page, hkv, d, ct, 31)
    pages = table(2, 5, 12, 32)
    q = torch.randn((2 * t, 4, d), generator=gen(33)).to(BF16).cuda()
    lens = torch.tensor([[35, 36, 37, 38], [0, 5, 70, 0]], dtype=torch.int32, device="cuda")
    want = attn.attn_decode(q, c, pages, lens, want_lse=True)
    seen = torch.zeros((12, page), dtype=torch.bool)
    for s, n in ((0, 38), (1, 70)):
        for j in range(n):
            seen[int(pages[s, j // page]), j % page] = True
    hidden = ~seen.cuda()
    for bad in (math.nan, math.inf, -math.inf):
        for x, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
            if ct == I8:
                scale.masked_fill_(hidden.unsqueeze(1), bad)
            else:
                x.masked_fill_(hidden.view(12, 1, page, 1), bad)
        got = attn.attn_decode(q, c, pages, lens, want_lse=True)
        assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse), bad
    # a key that some rows see and others do not: only those that see it change
    for j, rows in ((37, [3]), (36, [2, 3]), (35, [1, 2, 3])):
        p, o = int(pages[0, j // page]), j % page
        for x, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
            kept = (scale if ct == I8 else x)[p, 0, o].clone()
            (scale if ct == I8 else x)[p, 0, o] = math.nan
            got = attn.attn_decode(q, c, pages, lens, want_lse=True)
            for r in range(2 * t):
                hit = r in rows
                assert torch.equal(got.out[r, 2:], want.out[r, 2:]), (j, r)
                assert bool(got.out[r, :2].isnan().any()) == hit and (hit or torch.equal(got.out[r], want.out[r])), (j, r)
            (scale if ct == I8 else x)[p, 0, o] = kept
    # a query of NaN is its own row's
    q2 = q.clone()
    q2[1, 0, 3] = math.nan
    got = attn.attn_decode(q2, c, pages, lens)
    assert got.out[1, 0].isnan().all()
    got.out[1, 0] = want.out[1, 0]
    assert torch.equal(got.out, want.out)


@pytest.mark.parametrize("ct", [BF16, I8])
def test_page_numbers_outside_the_cache(ct):
    c = cache_of(9, 16, 2, 64, ct, 41)
    pages = table(3, 6, 9, 42)
    pages[0, 1] = -1
    pages[0, 4] = 9
    pages[1] = torch.tensor([-5, 2 ** 31 - 1, 9, 10, -(2 ** 31), 12], dtype=torch.int32)
    pages[2, 5] = 12345  # behind the last key
    q = torch.randn((6, 4, 64), generator=gen(43)).to(F16).cuda()
    lens = torch.tensor([[90, 96], [50, 96], [64, 80]], dtype=torch.int32, device="cuda")
    got = check(q, c, pages, lens)
    assert not got.out[2:4].any() and torch.isneginf(got.lse[2:4]).all()


def test_lengths_outside_the_table():
    from hoard_amd import attn
    c = cache_of(8, 16, 1, 64, F16, 51)
    pages = table(3, 4, 8, 52)
    q = torch.randn((3, 2, 64), generator=gen(53)).to(F16).cuda()
    lens = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    a = attn.attn_decode(q, c, pages, lens(2 ** 31 - 1, -1, -(2 ** 31)), want_lse=True)
    b = attn.attn_decode(q, c, pages, lens(64, 0, 0), want_lse=True)
    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse) and not a.out[1:].any()
    none = attn.attn_decode(q, c, pages[:, :0].contiguous(), lens(5, 5, 5), want_lse=True)
    assert not none.out.any() and torch.isneginf(none.lse).all()
    assert attn.attn_decode(q[:0], c, pages[:0], lens()).out.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype,ct,size,v_size", [
    (F32, F16, 1e4, 1.0), (F32, F16, 1e-4, 1.0), (F32, I8, 300.0, 1e-6), (F32, I8, 1.0, 1e6), (BF16, I8, 1e5, 1e30),
    (BF16, I8, 1.0, 1e-30), (BF16, F16, 1e6, 1e4), (F16, BF16, 1.0, 1e-30), (F32, BF16, 1e-6, 1e30), (F16, I8, 1e-6, 1e4)])
def test_sizes_of_values(dtype, ct, size, v_size):
    """Queries and values of sizes far from one, some rows of either far from the others; scores stay of order 4."""
    c = cache_of(20, 16, 2, 128, ct, 61, v_size)
    q = size * torch.randn((3, 8, 128), generator=gen(62))
    q[1, 3] *= 1e-3
    if ct == I8:
        c.v_scale[5] *= 1e-3
        c.v_scale[7, :, 3] = 0.0
        c.k_scale[6] *= 1e-3
    lens = torch.tensor([300, 77, 31], dtype=torch.int32, device="cuda")
    check(q.to(dtype).cuda(), c, table(3, 19, 20, 63), lens, scale=4.0 / (size * 128 ** 0.5))


def test_scores_far_apart():
    """Scores of thousands: the largest alone counts; a later one that is larger takes over."""
    from hoard_amd import attn
    d, n = 64, 200
    c = attn.KVCache.new(16, 16, 1, d, BF16)
    k = torch.zeros((256, 1, d))
    k[:, 0, 0] = torch.arange(256) * 16.0
    v = torch.randn((256, 1, d), generator=gen(71))
    slots = torch.arange(256, dtype=torch.int32, device="cuda")
    attn.kv_write(c, slots, k.cuda(), v.cuda())
    pages = torch.arange(16, dtype=torch.int32, device="cuda").view(1, 16)
    q = torch.zeros((1, 2, d))
    q[0, 0, 0], q[0, 1, 0] = 8.0, -8.0
    got = attn.attn_decode(q.to(BF16).cuda(), c, pages, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0, want_lse=True)
    assert torch.equal(got.out[0, 0].cpu(), v[n - 1, 0].to(BF16)) and torch.equal(got.out[0, 1].cpu(), v[0, 0].to(BF16))
    assert got.lse.cpu().tolist() == [[8.0 * 16 * (n - 1), 0.0]]


def test_rows_of_a_wider_tensor_and_given_output():
    from hoard_amd import attn
    c = cache_of(10, 16, 2, 64, I8, 81)
    pages = table(2, 4, 10, 82)
    lens = torch.tensor([[20, 21], [60, 61]], dtype=torch.int32, device="cuda")
    wide = torch.randn((4, 8 * 64), generator=gen(83)).to(F16).cuda()
    q, _, _ = attn.split_heads(wide, 4, 2, 64)
    out = torch.empty((4, 4, 64), dtype=F16, device="cuda")
    got = attn.attn_decode(q, c, pages, lens, out=out)
    assert got.out is out and got.lse is None
    assert torch.equal(out, attn.attn_decode(q.contiguous(), c, pages, lens).out)


def test_parts_join_by_their_logarithms():
    """Attention over two caches joined by lse is that over both."""
    from hoard_amd import attn
    c = cache_of(12, 16, 1, 64, F16, 91)
    q = torch.randn((1, 4, 64), generator=gen(92)).cuda()
    pages = table(1, 12, 12, 93)
    lens = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    whole = attn.attn_decode(q, c, pages, lens(180), want_lse=True)
    a = attn.attn_decode(q, c, pages[:, :5].contiguous(), lens(80), want_lse=True)
    b = attn.attn_decode(q, c, pages[:, 5:].contiguous(), lens(100), want_lse=True)
    w = torch.softmax(torch.stack([a.lse, b.lse]).double(), 0).unsqueeze(-1)
    joined = w[0] * a.out.double() + w[1] * b.out.double()
    # both within 2^-21 of the weights and some 200 roundings of the values' sums, which are up to 20 times the result
    assert ((joined - whole.out.double()).abs().max() <= (4 * 2.0 ** -21 + 500 * A.U32) * 4).item()


def test_beyond_32_bits():
    """Pages whose offsets pass 2^32 bytes and 2^31 elements."""
    from hoard_amd import attn
    hkv, d, page = 8, 256, 256
    n_pages = (5 << 30) // (hkv * d * page) + 1
    c = attn.KVCache.new(n_pages, page, hkv, d, I8)
    use = torch.tensor([n_pages - 1, 3, n_pages - 2, n_pages // 2 + 1], dtype=torch.int32)
    m = 4 * page
    slots = (use.view(4, 1) * page + torch.arange(page)).view(-1).to(torch.int32).cuda()
    x = torch.randn((2, m, hkv, d), generator=gen(101))
    attn.kv_write(c, slots, x[0].cuda(), x[1].cuda())
    small = attn.KVCache.new(4, page, hkv, d, I8)
    attn.kv_write(small, torch.arange(m, dtype=torch.int32, device="cuda"), x[0].cuda(), x[1].cuda())
    q = torch.randn((1, 16, d), generator=gen(102)).to(BF16).cuda()
    lens = torch.tensor([m - 5], dtype=torch.int32, device="cuda")
    a = attn.attn_decode(q, c, use.view(1, 4).cuda(), lens)
    b = attn.attn_decode(q, small, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), lens)
    assert c.k.numel() > 1 << 32 and torch.equal(a.out, b.out)


@pytest.mark.parametrize("longest", [100, 4000])
def test_graphs_streams_and_workspaces(longest):
    """Captured and replayed with other lengths, two graphs in turn, two streams at once."""
    from hoard_amd import attn
    page = 16
    width = -(-longest // page)
    c = cache_of(width + 5, page, 2, 128, I8, 111)
    pages = table(2, width, c.n_pages, 112)
    q = torch.randn((2, 16, 128), generator=gen(113)).to(BF16).cuda()
    lens = torch.tensor([longest, longest // 2], dtype=torch.int32, device="cuda")
    other = torch.tensor([3, longest - 1], dtype=torch.int32, device="cuda")
    want = [attn.attn_decode(q, c, pages, n, want_lse=True) for n in (lens, other)]
    graphs, outs, now = [], [], lens.clone()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attn.attn_decode(q, c, pages, now, want_lse=True))
        graphs.append(g)
    for turn in range(4):
        now.copy_(other if turn & 1 else lens)
        for o in outs:
            o.out.zero_()
            o.lse.zero_()
        for g in graphs:
            g.replay()
        attn.attn_decode(q, c, pages, lens)
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o.out, want[turn & 1].out) and torch.equal(o.lse, want[turn & 1].lse)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(8):
        s = streams[i % 2]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(attn.attn_decode(q, c, pages, (lens, other)[i % 2]))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o.out, want[i % 2].out)


@pytest.mark.parametrize("n,hkv,t,longest", [
    (40, 2, 1, 900), (65, 1, 1, 700), (100, 2, 1, 600), (130, 1, 3, 560), (256, 1, 1, 640), (257, 1, 1, 700), (300, 2, 1, 200),
    (3, 2, 4, 3000), (5, 4, 1, 5000), (70, 4, 1, 600), (2, 1, 64, 700)])
@pytest.mark.parametrize("ct", [F16, I8])
def test_batches(n, hkv, t, longest, ct):
    """Batches on both sides of where lanes are cut, share runs or have their own, some sequences empty, all of one table."""
    page, d = 16, 64
    width = -(-longest // page)
    c = cache_of(200, page, hkv, d, ct, 131)
    pages = torch.randint(0, 200, (n, width), generator=gen(132), dtype=torch.int32).cuda()
    lens = torch.randint(0, longest + 1, (n, 1), generator=gen(133), dtype=torch.int32) - torch.arange(t - 1, -1, -1, dtype=torch.int32)
    lens[torch.rand(n, generator=gen(134)) < 0.1] = 0
    lens[n // 2, -1] = longest
    q = (2.0 * torch.randn((n * t, 2 * hkv, d), generator=gen(135))).to(BF16).cuda()
    check(q, c, pages, lens.cuda().contiguous())


@pytest.mark.parametrize("n,t,longest,d", [(16, 5, 3001, 256), (8, 20, 1500, 256), (60, 1, 900, 256), (130, 1, 700, 256), (9, 7, 2000, 160)])
@pytest.mark.parametrize("dtype,ct", [(BF16, BF16), (F32, F16), (F16, I8)])
def test_batches_of_wide_heads(n, t, longest, d, dtype, ct):
    """Heads of which a CU holds one workgroup, in one or several blocks of rows: runs of one lane, fewer and more than CUs."""
    page, hkv = 32, 2
    width = -(-longest // page)
    c = cache_of(150, page, hkv, d, ct, 151)
    pages = torch.randint(0, 150, (n, width), generator=gen(152), dtype=torch.int32).cuda()
    lens = torch.randint(0, longest + 1, (n, 1), generator=gen(153), dtype=torch.int32) - torch.arange(t - 1, -1, -1, dtype=torch.int32)
    lens[n // 2, -1] = longest
    q = (2.0 * torch.randn((n * t, 8 * hkv, d), generator=gen(154))).to(dtype).cuda()
    check(q, c, pages, lens.cuda().contiguous())


def test_a_sequence_whose_tokens_see_far_apart_numbers_of_keys():
    """Rows of one tile that see 1 key, all of them, or none, over several parts, with values that are not finite between."""
    c = cache_of(300, 16, 1, 128, BF16, 141)
    pages = table(1, 260, 300, 142)
    lens = torch.tensor([[1, 4000, 0, 70, 4160, 2000]], dtype=torch.int32, device="cuda")
    q = torch.randn((6, 2, 128), generator=gen(143)).to(BF16).cuda()
    got = check(q, c, pages, lens)
    clean = got.out.clone()
    for j, value in ((3000, math.inf), (3999, -math.inf), (2500, math.nan)):
        c.v[int(pages[0, j // 16]), 0, j % 16, 5] = value
    from hoard_amd import attn
    got = attn.attn_decode(q, c, pages, lens).out
    for r in (0, 2, 3, 5):
        assert torch.equal(got[r], clean[r]), r
    for r in (1, 4):
        assert got[r, :, 5].isnan().all() and torch.isfinite(got[r][:, [0, 1, 2, 3, 4, 6, 127]]).all()


def test_refusals():
    from hoard_amd import attn
    c = cache_of(4, 16, 2, 64, F16, 121)
    pages = table(2, 2, 4, 122)
    lens = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    q = torch.randn((2, 4, 64), device="cuda")
    bad = {
        "heads": lambda: attn.attn_decode(q[:, :3].contiguous(), c, pages, lens),
        "dim": lambda: attn.attn_decode(q[:, :, :32].contiguous(), c, pages, lens),
        "rows": lambda: attn.attn_decode(q[:1], c, pages, lens),
        "lens type": lambda: attn.attn_decode(q, c, pages, lens.long()),
        "pages rows": lambda: attn.attn_decode(q, c, pages[:1], lens),
        "type": lambda: attn.attn_decode(q.double(), c, pages, lens),
        "out over q": lambda: attn.attn_decode(q, c, pages, lens, out=q),
        "no dense heads": lambda: attn.attn_decode(q.transpose(1, 2).contiguous().transpose(1, 2), c, pages, lens),
        "new": lambda: attn.attn_decode(torch.zeros((65, 4, 64), device="cuda"), c, pages[:1], lens.new_zeros((1, 65))),
        "scales": lambda: attn.KVCache(c.k, c.v, torch.zeros(c.k.shape[:3], device="cuda"), torch.zeros(c.k.shape[:3], device="cuda")),
        "a scale": lambda: attn.KVCache(c.k.to(I8), c.v.to(I8), torch.zeros(c.k.shape[:3], device="cuda")),
        "k only": lambda: attn.KVCache(c.k, c.v[:2]),
    }
    for name, call in bad.items():
        with pytest.raises(H.HoardError):
            call()
            pytest.fail(name)
    odd = attn.KVCache(torch.zeros((2, 2, 24, 64), dtype=F16, device="cuda"), torch.zeros((2, 2, 24, 64), dtype=F16, device="cuda"))
    with pytest.raises(H.HoardError, match="page 24"):
        attn.attn_decode(q, odd, pages, lens)

"""8-bit caches whose rows of values have scales far apart: each row of queries keeps the digits of what it weighs."""
import math

import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, BF16, I8 = torch.float32, torch.bfloat16, torch.int8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def cache_of(pages, heads, d, seed):
    from hoard_amd import attn
    c = attn.KVCache.new(pages, 16, heads, d, I8)
    x = torch.randn((2, pages * 16, heads, d), generator=gen(seed)).cuda()
    attn.kv_write(c, torch.arange(pages * 16, dtype=torch.int32, device="cuda"), x[0], x[1])
    return c


def dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def held(q, c, pages, lens, scale):
    """How far off a result may be as products of weights and scales are held to 2^-37 of the row's largest, where that
    is more than their own digits: the largest, brought to 2^12 or more, is formed of 16-bit floats whose steps end at
    2^-24, so half a step is 2^-25; it meets a code of up to 127 of each key.  (A column in which the largest product's
    key has the code 0 keeps no more of the others: far below that key's step, by which it may be off.)"""
    kk, vs = A.values(c.k, c.k_scale), A.t64(c.v_scale)
    out = torch.zeros(q.shape[:2], dtype=A.D)
    pages, lens = pages.cpu(), lens.cpu().reshape(len(pages), -1)
    for r in range(len(q)):
        n = int(lens[r // lens.shape[1], r % lens.shape[1]])
        p, o, _ = A.gathered(pages[r // lens.shape[1]], n, 16, len(kk))
        for h in range(q.shape[1]):
            kv = h * kk.shape[1] // q.shape[1]
            w = torch.softmax(scale * (kk[p, kv, o] @ A.t64(q[r, h])), 0)
            out[r, h] = n * 127 * 2.0 ** -37 * (w * vs[p, kv, o]).max()
    return out.unsqueeze(-1)


def check(q, c, pages, lens, scale):
    from hoard_amd import attn
    got = attn.attn_decode(q, c, pages, lens, scale=scale, want_lse=True)
    want, bound, lse, lse_bound = A.attention(q, c.k, c.v, c.k_scale, c.v_scale, pages, lens, scale, q.dtype)
    bound = bound + held(q, c, pages, lens, scale)
    A.close(got.out, want, A.stored(want, bound, q.dtype), "out")
    A.close(got.lse, lse, A.stored(lse, lse_bound, F32), "lse")
    return got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("power", [8, 22, 30, 40, 100, math.inf])
def test_a_scale_that_one_draft_sees(power, d, dtype):
    """Two drafts of 36 and 37 keys, key 36's values 2^power times the others': the first draft's row is untouched."""
    from hoard_amd import attn
    c = cache_of(4, 2, d, 1)
    pages, lens = dev([[2, 0, 3]]), dev([[36, 37]])
    q = torch.randn((2, 4, d), generator=gen(2)).to(dtype).cuda()
    clean = attn.attn_decode(q, c, pages, lens, want_lse=True)
    c.v_scale[3, :, 4] *= 2.0 ** power
    if power < math.inf:
        got = check(q, c, pages, lens, float(torch.tensor(d ** -0.5)))
    else:
        got = attn.attn_decode(q, c, pages, lens, want_lse=True)
    assert torch.equal(got.out[0], clean.out[0]) and torch.equal(got.lse, clean.lse)
    assert power < math.inf or got.out[1].isnan().all()


def sloped(n, d, bits, step, seed):
    """A cache of one key head whose value rows' scales and keys' first elements follow the tiles of 32 keys: the values
    of tile i are 2^(bits i) times the first's (those in the middle of size one), its keys (step i, 0, ..) and some noise."""
    from hoard_amd import attn
    c = attn.KVCache.new(n // 16 + 1, 16, 1, d, I8)
    tile = torch.arange(c.n_pages * 16) // 32
    k = 0.02 * torch.randn((c.n_pages * 16, 1, d), generator=gen(seed))
    k[:, 0, 0] = step * tile
    v = torch.randn((c.n_pages * 16, 1, d), generator=gen(seed + 1)) * (2.0 ** (bits * (tile.double() - n / 64))).float().view(-1, 1, 1)
    attn.kv_write(c, torch.arange(c.n_pages * 16, dtype=torch.int32, device="cuda"), k.cuda(), v.cuda())
    return c, torch.arange(c.n_pages, dtype=torch.int32, device="cuda").view(1, -1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [3, -3, 10, -10])
@pytest.mark.parametrize("n", [320, 1000])
def test_scales_against_weights(n, bits, dtype):
    """Scales that rise (fall) from tile to tile, and in one row scores that fall (rise) by as much, so that every tile
    counts the same there; in others they rise together, do not change, or fall twice as fast."""
    if n == 1000:
        bits = bits / 4  # 31 tiles, some of them in other waves and workgroups
    d, step = 64, 4.0
    c, pages = sloped(n, d, bits, step, 11)
    unit = -bits * math.log(2.0) / step
    q = 0.02 * torch.randn((1, 8, d), generator=gen(13))
    q[0, :, 0] = unit * torch.tensor([1.0, 0.0, -0.5, 2.0, 0.9, 1.1, 0.25, 1.0])
    check(q.to(dtype).cuda(), c, pages, dev([n]), 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("power", [30, 60])
def test_a_large_scale_of_no_weight(power, dtype):
    """One key's values are 2^power times the others' and its weight 2^-power / 1000 of theirs, or next to nothing."""
    d = 128
    c = cache_of(5, 1, d, 21)
    pages = dev([[4, 1, 0, 3]])
    c.v_scale[1, 0, 4] *= 2.0 ** power  # key 20
    c.k[1, 0, 4] = 0
    c.k[1, 0, 4, 0] = 127
    c.k_scale[1, 0, 4] = 1.0
    q = 0.1 * torch.randn((2, 4, d), generator=gen(22))
    q[0, :, 0] = -(power * math.log(2.0) + math.log(1000.0)) / 127
    q[1, :, 0] = -150.0 / 127
    check(q.to(dtype).cuda(), c, pages, dev([[50, 64]]), 1.0)


def test_scales_of_zero_and_below_the_normal_range():
    """Rows of zeros among others, and all scales tiny or none at all."""
    from hoard_amd import attn
    c = cache_of(4, 1, 64, 31)
    pages, lens = dev([[0, 1, 2, 3]]), dev([[40, 64]])
    q = torch.randn((2, 4, 64), generator=gen(32)).cuda()
    c.v_scale[1] = 0.0
    check(q, c, pages, lens, 0.125)
    c.v_scale *= 2.0 ** -126
    check(q, c, pages, lens, 0.125)
    c.v_scale.zero_()
    assert not attn.attn_decode(q, c, pages, lens).out.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e20, 1e36])
def test_queries_and_keys_of_opposite_sizes(size, dtype):
    """Scores of order 4 of queries and keys each far from one."""
    c = cache_of(5, 2, 128, 41)
    c.k_scale /= size
    q = size * torch.randn((2, 8, 128), generator=gen(42))
    check(q.to(dtype).cuda(), c, dev([[4, 0, 2, 1, 3]]), dev([[70, 71]]), float(torch.tensor(4.0 / 128 ** 0.5)))

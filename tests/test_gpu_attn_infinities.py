"""Infinities and NaN that a row of queries sees in a 16-bit cache: the same wherever they lie, and in their columns only."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = math.inf, math.nan


def gen(seed):
    return torch.Generator().manual_seed(seed)


def setup(n, d, ct, dtype, t=2):
    """A cache in order of its pages, and t drafts of n - t + 1 .. n keys; 1 key head."""
    from hoard_amd import attn
    c = attn.KVCache.new(-(-n // 16), 16, 1, d, ct)
    x = torch.randn((2, c.n_pages * 16, 1, d), generator=gen(1)).cuda()
    attn.kv_write(c, torch.arange(c.n_pages * 16, dtype=torch.int32, device="cuda"), x[0], x[1])
    pages = torch.arange(c.n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    lens = torch.arange(n - t + 1, n + 1, dtype=torch.int32, device="cuda").view(1, t)
    q = torch.randn((t, 4, d), generator=gen(2)).to(dtype).cuda()
    return c, pages, lens, q


@pytest.mark.parametrize("ct", [F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 80, 256])
@pytest.mark.parametrize("n,places", [(38, [0, 31, 33, 36, 37]), (300, [5, 100, 200, 298, 299]), (1500, [0, 700, 1499])])
def test_values(n, places, d, dtype, ct):
    from hoard_amd import attn
    c, pages, lens, q = setup(n, d, ct, dtype)
    clean = attn.attn_decode(q, c, pages, lens, want_lse=True)
    col = d - 3
    for j in places:
        kept = c.v[j // 16, 0, j % 16, col].clone()
        c.v[j // 16, 0, j % 16, col] = 0.0
        zero = attn.attn_decode(q, c, pages, lens).out
        for bad in (INF, -INF, NAN):
            c.v[j // 16, 0, j % 16, col] = bad
            got = attn.attn_decode(q, c, pages, lens, want_lse=True)
            assert torch.equal(got.lse, clean.lse)
            want = zero.clone()
            for r in range(2):
                if j < int(lens[0, r]):
                    want[r, :, col] = bad
            assert torch.equal(got.out.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)), (j, bad)
        c.v[j // 16, 0, j % 16, col] = kept
    # opposite ones in one column are NaN there; in two columns each is its own
    c.v[0, 0, 3, 1], c.v[0, 0, 9, 1], c.v[1, 0, 2, 2], c.v[0, 0, 9, 4] = INF, -INF, -INF, INF
    got = attn.attn_decode(q, c, pages, lens).out
    assert got[..., 1].isnan().all() and (got[..., 2] == -INF).all() and (got[..., 4] == INF).all()
    others = [i for i in range(d) if i not in (1, 2, 4)]
    assert torch.equal(got[..., others], clean.out[..., others])


@pytest.mark.parametrize("ct", [F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,places", [(38, [0, 31, 36, 37]), (300, [100, 298]), (1500, [0, 1499])])
def test_keys(n, places, dtype, ct):
    """A key of infinity: a score of minus infinity weighs nothing, one of plus infinity makes its row NaN."""
    from hoard_amd import attn
    c, pages, lens, q = setup(n, 64, ct, dtype)
    q[:, 0, 5], q[:, 1, 5], q[:, 2, 5] = 1.5, -1.5, 0.0
    q[:, 3, 5] = 1.1 if dtype == F32 else 1.25  # with and without a second plane
    big = 60000.0
    for j in places:
        key = c.k[j // 16, 0, j % 16]
        kept = key[5].clone()
        for sign in (1.0, -1.0):
            key[5] = sign * big  # scores of magnitude 8000, whose weight is zero where it is negative
            want = attn.attn_decode(q, c, pages, lens, want_lse=True)
            key[5] = sign * INF
            got = attn.attn_decode(q, c, pages, lens, want_lse=True)
            for r in range(2):
                seen = j < int(lens[0, r])
                for h, s in ((0, 1.0), (1, -1.0), (2, 0.0), (3, 1.0)):
                    if seen and s * sign >= 0:
                        assert got.out[r, h].isnan().all(), (j, sign, r, h)
                    else:
                        assert torch.equal(got.out[r, h], want.out[r, h]) and torch.equal(got.lse[r, h], want.lse[r, h]), (j, sign, r, h)
        key[5] = NAN
        got = attn.attn_decode(q, c, pages, lens)
        for r in range(2):
            assert bool(got.out[r].isnan().all()) == (j < int(lens[0, r]))
        key[5] = kept


@pytest.mark.parametrize("ct", [F16, BF16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_every_score_minus_infinity(dtype, ct):
    """Such a row is as one that sees no key."""
    from hoard_amd import attn
    c, pages, lens, q = setup(70, 64, ct, dtype)
    c.k[:, 0, :, 7] = INF
    q[1, 2, 7] = -1.25
    q[1, 3, 7] = 1.25
    got = attn.attn_decode(q, c, pages, lens, want_lse=True)
    assert not got.out[1, 2].any() and got.lse[1, 2] == -INF and got.out[1, 3].isnan().all()


@pytest.mark.parametrize("ct", [F16, BF16, torch.int8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_queries(dtype, ct):
    """A query that is not finite makes its row NaN, whatever the signs of the keys, and no other; where it sees no key
    its row is zero."""
    from hoard_amd import attn
    c, pages, lens, q = setup(70, 64, ct, dtype, 3)
    lens[0, 2] = 0
    want = attn.attn_decode(q, c, pages, lens, want_lse=True)
    for bad in (INF, -INF, NAN):
        q2 = q.clone()
        q2[0, 1, 9], q2[1, 3, 0], q2[2, :, 63] = bad, bad, bad
        got = attn.attn_decode(q2, c, pages, lens, want_lse=True)
        assert got.out[0, 1].isnan().all() and got.out[1, 3].isnan().all() and got.lse[0, 1].isnan()
        got.out[0, 1], got.out[1, 3] = want.out[0, 1], want.out[1, 3]
        assert torch.equal(got.out, want.out) and not got.out[2].any() and (got.lse[2] == -INF).all()

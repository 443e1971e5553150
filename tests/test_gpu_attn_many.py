"""Attention of more sequences than one launch takes."""
import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16 = torch.float16


def test_more_lanes_than_a_grid():
    """2^21 + 5 sequences by 4 key heads: two launches, whose rows are those of calls of few sequences."""
    from hoard_amd import attn
    n, hkv, d = (1 << 21) + 5, 4, 16
    g = torch.Generator().manual_seed(1)
    c = attn.KVCache.new(50, 16, hkv, d, F16)
    x = torch.randn((2, 800, hkv, d), generator=g).cuda()
    attn.kv_write(c, torch.arange(800, dtype=torch.int32, device="cuda"), x[0], x[1])
    pages = torch.randint(0, 50, (n, 1), generator=g, dtype=torch.int32).cuda()
    lens = torch.randint(0, 17, (n,), generator=g, dtype=torch.int32).cuda()
    q = torch.randn((n, hkv, d), generator=g).to(F16).cuda()
    got = attn.attn_decode(q, c, pages, lens, want_lse=True)
    for at in (slice(0, 3000), slice((1 << 21) - 1500, (1 << 21) + 5), slice(1000003, 1003003)):
        few = attn.attn_decode(q[at], c, pages[at], lens[at], want_lse=True)
        assert torch.equal(got.out[at], few.out) and torch.equal(got.lse[at], few.lse)
    last = slice(n - 40, n)
    want, bound, _, _ = A.attention(q[last], c.k, c.v, None, None, pages[last], lens[last], float(torch.tensor(d ** -0.5)), F16)
    A.close(got.out[last], want, A.stored(want, bound, F16), "out")
    step = (1 << 19)
    for i in range(0, n, step):
        at = slice(i, min(i + step, n))
        assert torch.equal(got.out[at], attn.attn_decode(q[at], c, pages[at], lens[at]).out)

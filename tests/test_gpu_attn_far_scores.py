"""Scores so large that neighbouring numbers of 32 bits lie far apart."""
import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [240, 1300])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 10, 2.0 ** 16, 2.0 ** 40])
def test_the_largest_alone(size, n, dtype, ct):
    """Keys whose scores are 0, 16 size, 32 size, .. in turns of 100: the result is the mean of the values of the largest.
    The others weigh e^-16 of each of them at most, all of them together less than 2e-7 of the result's terms; the mean's
    weights and sum round a few times."""
    from hoard_amd import attn
    c = attn.KVCache.new(n // 16 + 1, 16, 1, 64, ct)
    x = torch.randn((c.n_pages * 16, 1, 64), generator=torch.Generator().manual_seed(1))
    k = torch.zeros_like(x)
    k[:, 0, 0] = 127.0 * (torch.arange(len(k)) % 100)
    attn.kv_write(c, torch.arange(len(k), dtype=torch.int32, device="cuda"), k.cuda(), x.cuda())
    pages = torch.arange(c.n_pages, dtype=torch.int32, device="cuda").view(1, -1)
    q = torch.zeros((1, 2, 64))
    q[0, 0, 0], q[0, 1, 0] = 128.0, -128.0
    scale = 16.0 / (127 * 128) * size
    got = attn.attn_decode(q.to(dtype).cuda(), c, pages, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=scale, want_lse=True)
    v = A.values(c.v, c.v_scale).transpose(1, 2).reshape(-1, 64)[:n]
    at = torch.arange(n) % 100
    for h, best in ((0, 99), (1, 0)):
        rows = v[at == best]
        want = rows.mean(0)
        bound = rows.abs().mean(0) * 16 * A.U32 + 3e-7 * v.abs().amax(0)
        A.close(got.out[0, h], want, A.stored(want, bound, dtype), h)
    # the key as the cache rounds it
    top = float(torch.tensor(scale)) * 128.0 * float(A.values(c.k, c.k_scale)[6, 0, 3, 0])
    assert abs(float(got.lse[0, 0]) - top) <= 8 * A.U32 * top + 3


@pytest.mark.parametrize("ct", [BF16, I8])
@pytest.mark.parametrize("seqs,n", [(1, 6000), (66, 1200), (140, 1200)])
def test_large_values_in_many_parts(seqs, n, ct):
    """Values of 1e36 and all keys alike: their mean, of which no sum of parts may be larger than 32 bits hold.  A term a
    key rounds a few times, each to 2^-15 for its weight."""
    from hoard_amd import attn
    c = attn.KVCache.new(n // 16 + 1, 16, 1, 64, ct)
    x = torch.randn((c.n_pages * 16, 1, 64), generator=torch.Generator().manual_seed(1)).abs()
    attn.kv_write(c, torch.arange(len(x), dtype=torch.int32, device="cuda"), x.cuda(), 1e36 * x.cuda())
    pages = torch.arange(c.n_pages, dtype=torch.int32, device="cuda").expand(seqs, -1).contiguous()
    lens = (n - torch.arange(seqs)).to(torch.int32).cuda()
    got = attn.attn_decode(torch.zeros((seqs, 8, 64), dtype=BF16, device="cuda"), c, pages, lens).out
    v = A.values(c.v, c.v_scale).transpose(1, 2).reshape(-1, 64)
    want = torch.stack([v[:int(m)].mean(0) for m in lens]).unsqueeze(1).expand(seqs, 8, 64)
    A.close(got, want, A.stored(want, want * (2.0 ** -15 + 2 * n * A.U32), BF16), "out")

"""The logarithms of the sums in all of their digits."""
import pytest

import attnref as A

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16, I8 = torch.float32, torch.float16, torch.bfloat16, torch.int8


@pytest.mark.parametrize("ct", [F16, BF16, I8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("longest", [300, 6000])
def test_of_counts(longest, dtype, ct):
    """Queries of zeros: the logarithm of the number of keys.  Its sum is exact, in parts too; its base 2 logarithm rounds
    by 2 u, it is added to a maximum of 0, the factor and the product round by a u each."""
    from hoard_amd import attn
    n = 48
    c = attn.KVCache.new(longest // 16 + 1, 16, 1, 64, ct)
    x = torch.randn((c.n_pages * 16, 1, 64), generator=torch.Generator().manual_seed(1)).cuda()
    attn.kv_write(c, torch.arange(c.n_pages * 16, dtype=torch.int32, device="cuda"), x, x)
    pages = torch.arange(c.n_pages, dtype=torch.int32, device="cuda").expand(n, -1).contiguous()
    g = torch.Generator().manual_seed(2)
    lens = torch.cat([torch.arange(1, 25), torch.randint(25, longest + 1, (n - 24,), generator=g)]).to(torch.int32).cuda()
    got = attn.attn_decode(torch.zeros((n, 2, 64), dtype=dtype, device="cuda"), c, pages, lens, want_lse=True)
    want = torch.log(A.t64(lens)).view(n, 1).expand(n, 2)
    A.close(got.lse, want, 4 * A.U32 * want, "lse")

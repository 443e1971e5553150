"""Arrays of more than 2^31 elements or 2^32 bytes: what lies behind those offsets is read and written where it is."""
import pytest

import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def test_rows_far():
    """Gather, combine and its gradient over 2^31 elements of sorted rows, checked at both ends."""
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather, sort_pairs
    tokens, k, n, experts = 132000, 8, 2048, 8
    assert tokens * k * n > 2**31
    ids = torch.arange(k, dtype=torch.int32).repeat(tokens, 1).cuda()  # expert j holds slot j of every token
    s = sort_pairs(ids, experts)
    assert s.offsets.tolist() == [j * tokens for j in range(k + 1)]
    x = torch.randint(-8, 8, (tokens, n), device="cuda", dtype=torch.int8).to(BF16)
    xs = sort_gather(x, s.place)
    for j in range(k):
        assert torch.equal(xs[j * tokens], x[0]) and torch.equal(xs[(j + 1) * tokens - 1], x[-1])
    w = torch.ones((tokens, k), device="cuda")
    out = sort_combine(xs, s.place, w)
    assert torch.equal(out[-3:], x[-3:] * 8) and torch.equal(out[:3], x[:3] * 8)
    dy, dw = sort_combine_grad(x, xs, s.place, w, dy=xs)  # in place of y: a pair's row is read before it is written
    assert torch.equal(dy[-2:], x[-2:])
    sums = (x[-4:].double() ** 2).sum(1, keepdim=True).expand(4, k)
    assert ((dw[-4:].double() - sums).abs() <= (n + 1) * R.U32 * sums).all()


def test_norm_far():
    from hoard_amd.ops import norm_backward, norm_forward
    m, n = 132000, 16384
    assert m * n > 2**31
    r = torch.ones((m, n), dtype=BF16, device="cuda")
    r[-1] = torch.randn(n, device="cuda").to(BF16)
    w = torch.ones(n, device="cuda")
    st = norm_forward(r, w_pre=w, eps=1e-6, want_stats=True)
    want = R.norm(r[-1:].cpu().double(), 1e-6)
    R.close(st.h[-1:], want, R.stored(want, 40 * R.U32 * want.abs(), BF16), "h")
    assert (st.h[: m // 2].float() - 1).abs().max() < 1e-2
    g = norm_backward(st, None, st.h, w_pre=w, eps=1e-6)
    # dh = h = v rho: dr = rho (h - v rho^2 mean(h v)) = rho h (1 - rho^2 mean v^2), which eps alone keeps from 0
    assert g.dr[-1].float().abs().max() < 0.05 and torch.isfinite(g.dr[-1]).all()


def test_q4_far():
    """Codes behind 2^32 bytes, by ids and by offsets."""
    from hoard_amd.ops import Q4Weight, q4_matmul
    mats, rows, cols, group = 1100, 1024, 8192, 128
    assert mats * rows * cols // 2 > 2**32
    codes = torch.full((mats, rows, cols // 2), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.full((mats, rows, cols // group), 0.01, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(3)
    for e in (0, mats - 1):
        codes[e] = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8).cuda()
    w = Q4Weight(codes, scales)
    x = torch.randn((6, cols), generator=g).to(BF16).cuda()
    ids = torch.tensor([mats - 1, 5, 0, mats - 1, 1099, 7], dtype=torch.int32).cuda()
    y = q4_matmul(x, w, ids=ids)
    offsets = torch.zeros(mats + 1, dtype=torch.int32)
    offsets[1:] = 2
    offsets[mats] = 6
    z = q4_matmul(x, w, offsets=offsets.cuda())
    for e, got, rows_of in ((mats - 1, y, [0, 3, 4]), (0, y, [2]), (0, z, [0, 1]), (mats - 1, z, [2, 3, 4, 5])):
        v, b = R.product(x[rows_of], (codes[e], scales[e], None), None)
        R.close(got[rows_of], v, R.stored(v, b, BF16), (e, rows_of))
    assert (y[[1, 5]] == 0).all()

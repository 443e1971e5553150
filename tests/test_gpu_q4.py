"""hoard_q4_matmul and its forms by ids and by offsets against a 64-bit product, within bounds that count roundings."""
import numpy as np
import pytest

import hoard_amd as H
import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def weights(seed, n_mat, rows, cols, group, scales=F16, zeros=False, wild=False):
    """(codes, scales, zeros) on the device; wild: any zero byte and scales of either sign and of zero."""
    g = torch.Generator().manual_seed(seed)
    lead = (n_mat, rows) if n_mat else (rows,)
    codes = torch.randint(0, 256, (*lead, cols // 2), generator=g, dtype=torch.uint8)
    s = torch.rand((*lead, cols // group), generator=g) * 0.02
    if wild:
        s = torch.where(torch.rand(s.shape, generator=g) < 0.2, torch.zeros_like(s), s - 0.01)
    z = None
    if zeros:
        z = torch.randint(0, 256 if wild else 16, s.shape, generator=g, dtype=torch.uint8).cuda()
    return codes.cuda(), s.to(scales).cuda(), z


def rows_of(seed, n, cols, dtype, scale=1.0):
    return (torch.randn((n, cols), generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def op(m):
    from hoard_amd.ops import Q4Weight
    return Q4Weight(*m)


def expect(x, w, up, e=None):
    """Value and bound (stored) of the rows x by matrix e (None: the only one)."""
    v, b = R.product(x, w, e)
    if up is not None:
        v, b = R.swiglu(v, b, *R.product(x, up, e))
    return v, R.stored(v, b, x.dtype)


DENSE = [
    # rows of x, rows of w, cols, group, type, scales, zeros, up
    (1, 1, 32, 32, F32, F16, False, False), (1, 5, 64, 64, BF16, BF16, True, False),
    (1, 64, 128, 128, F16, F32, False, True), (1, 257, 2048, 128, F32, F16, True, False),
    (1, 512, 4096, 64, BF16, BF16, False, True), (1, 1000, 8192, 128, F16, F16, True, True),
    (2, 333, 1056, 32, F32, F32, True, True), (2, 64, 2048, 128, BF16, F16, False, False),
    (3, 96, 640, 128, F16, BF16, True, False), (4, 130, 1024, 64, BF16, BF16, False, False),
    (5, 63, 2080, 32, F32, F16, True, False), (6, 256, 2048, 64, F32, BF16, False, True),
    (8, 17, 8192, 128, BF16, F32, False, True), (13, 300, 4096, 32, F16, F16, True, False),
    (16, 128, 2048, 128, BF16, BF16, False, False), (17, 129, 544, 32, F32, F16, False, False),
    (31, 65, 192, 64, F16, F16, True, True), (33, 200, 256, 128, F32, F32, True, False),
    (64, 64, 2048, 64, BF16, BF16, False, True), (65, 80, 96, 32, BF16, F16, True, False),
    (100, 250, 1024, 128, F16, F16, False, False), (127, 31, 384, 128, F32, F16, True, True),
    (128, 128, 512, 64, BF16, BF16, True, False), (200, 513, 2048, 128, BF16, F16, False, True),
    (513, 96, 256, 32, F16, BF16, True, False),
]


@pytest.mark.parametrize("n,rows,cols,group,dtype,scales,zeros,up", DENSE)
def test_dense(n, rows, cols, group, dtype, scales, zeros, up):
    from hoard_amd.ops import q4_matmul
    print("q4 dense", n, rows, cols, group, dtype, flush=True)
    w = weights(1, 0, rows, cols, group, scales, zeros)
    # the second matrix has its own scale type and zeros
    u = weights(2, 0, rows, cols, group, F32, not zeros) if up else None
    x = rows_of(3, n, cols, dtype)
    y = q4_matmul(x, op(w), op(u) if up else None)
    R.close(y, *expect(x, w, u), "y")


@pytest.mark.parametrize("n", [1, 4, 16, 70])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_dense_wild(n, dtype):
    """Zero points of any byte, scales of either sign and of zero, x over many orders of magnitude."""
    from hoard_amd.ops import q4_matmul
    rows, cols = 48, 512
    w = weights(5, 0, rows, cols, 64, F32, True, wild=True)
    x = rows_of(6, n, cols, F32) * torch.exp2(torch.randint(-12, 8, (n, cols), generator=torch.Generator().manual_seed(7))).cuda()
    x = x.to(dtype)
    y = q4_matmul(x, op(w))
    R.close(y, *expect(x, w, None), "y")


def routing(seed, tokens, k, experts, bad=()):
    g = np.random.default_rng(seed)
    ids = np.stack([g.permutation(experts)[:k] for _ in range(tokens)]).astype(np.int32)
    for t, j, e in bad:
        ids[t, j] = e
    return torch.from_numpy(ids)


@pytest.mark.parametrize("tokens,k,experts,rows,cols,group,dtype,up", [
    (1, 1, 1, 33, 64, 32, F32, False), (1, 8, 16, 96, 512, 128, F32, True), (1, 2, 3, 256, 2048, 64, BF16, True),
    (3, 4, 9, 65, 256, 32, F16, False), (7, 10, 12, 40, 1024, 128, BF16, False), (32, 3, 5, 24, 128, 64, F32, True)])
def test_ids(tokens, k, experts, rows, cols, group, dtype, up):
    from hoard_amd.ops import q4_matmul
    w = weights(11, experts, rows, cols, group, F16, True)
    u = weights(12, experts, rows, cols, group, BF16) if up else None
    x = rows_of(13, tokens, cols, dtype)
    ids = routing(14, tokens, k, experts)
    y = q4_matmul(x, op(w), op(u) if up else None, ids=ids.cuda())
    flat, xr = ids.reshape(-1), x.repeat_interleave(k, 0)
    for e in range(experts):
        r = torch.nonzero(flat == e).view(-1)
        R.close(y[r.cuda()], *expect(xr[r.cuda()], w, u, e), f"expert {e}")


def test_ids_out_of_range_and_repeated():
    from hoard_amd.ops import q4_matmul
    experts, k = 4, 3
    w = weights(21, experts, 50, 256, 64)
    x = rows_of(22, 3, 256, F32)
    ids = routing(23, 3, k, experts, [(0, 1, -1), (1, 0, experts), (1, 2, 2**31 - 1), (2, 0, 2), (2, 1, 2)])
    y = q4_matmul(x, op(w), ids=ids.cuda())
    for p, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < experts:
            R.close(y[p:p + 1], *expect(x[p // k:p // k + 1], w, None, e), p)
        else:
            assert y[p].isnan().all()


@pytest.mark.parametrize("counts,rows,cols,group,dtype,up", [
    ([1], 40, 64, 32, F32, False), ([0, 0, 3, 0], 70, 256, 64, BF16, True), ([1, 1, 1, 1, 1, 1, 1, 1], 96, 512, 128, F32, True),
    ([5, 0, 17, 1, 64, 2], 130, 512, 128, BF16, True), ([200, 3, 0, 65], 64, 256, 32, F16, False),
    ([33, 31, 0, 0, 129], 48, 320, 64, F32, True), ([2] * 40 + [0] * 30, 33, 128, 128, BF16, False),
    ([16, 15, 17, 32, 31, 33, 48, 0, 1], 100, 1024, 128, F16, True)])
@pytest.mark.parametrize("tail", [0, 5])
def test_sorted(counts, rows, cols, group, dtype, up, tail):
    """Rows by offsets; `tail` rows behind the last range stay as they were."""
    from hoard_amd.ops import q4_matmul
    experts = len(counts)
    w = weights(31, experts, rows, cols, group, BF16, True)
    u = weights(32, experts, rows, cols, group, F16) if up else None
    n = sum(counts) + tail
    x = rows_of(33, n, cols, dtype)
    x[sum(counts):] = float("nan")
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    out = torch.full((n, rows), 7.0, dtype=dtype, device="cuda")
    y = q4_matmul(x, op(w), op(u) if up else None, offsets=torch.from_numpy(offsets).cuda(), out=out)
    assert y is out
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        R.close(y[a:b], *expect(x[a:b], w, u, e), f"expert {e}")
    assert (y[sum(counts):] == 7.0).all()


def test_sorted_offsets_are_clamped():
    """Offsets past the rows, negative, and ranges that do not start at 0: no row outside [0, n_rows) is read or written."""
    from hoard_amd.ops import q4_matmul
    w = weights(41, 3, 40, 128, 64)
    x = rows_of(42, 20, 128, BF16)
    out = torch.full((24, 40), 7.0, dtype=BF16, device="cuda")
    for offsets, ranges in (([-5, 4, 9, 1000], [(0, 4, 0), (4, 9, 1), (9, 20, 2)]), ([3, 3, 8, 8], [(3, 8, 1)]),
                            ([20, 30, 40, 50], []), ([-9, -4, -1, 6], [(0, 6, 2)])):
        out.fill_(7.0)
        q4_matmul(x, op(w), offsets=torch.tensor(offsets, dtype=torch.int32).cuda(), out=out[:20])
        left = torch.ones(24, dtype=torch.bool)
        for a, b, e in ranges:
            R.close(out[a:b], *expect(x[a:b], w, None, e), (offsets, e))
            left[a:b] = False
        assert (out[left.cuda()] == 7.0).all(), offsets


@pytest.mark.parametrize("n", [1, 3, 20, 80])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rows_apart(n, dtype):
    """A row with an infinity or a NaN spoils no other row, and a row of zeros is exactly zero."""
    from hoard_amd.ops import q4_matmul
    w = weights(51, 0, 64, 256, 64, F16, True)
    x = rows_of(52, n + 3, 256, dtype)
    clean = q4_matmul(x, op(w))
    bad = x.clone()
    bad[0, 3], bad[1, 200], bad[2] = float("inf"), float("nan"), 0.0
    y = q4_matmul(bad, op(w))
    assert not y[0].isfinite().any() and not y[1].isfinite().any()
    assert (y[2] == 0).all()
    assert torch.equal(y[3:], clean[3:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens,k,experts,rows,cols,group,up", [
    (3, 2, 40, 96, 256, 64, False), (40, 4, 16, 200, 384, 128, True), (300, 2, 5, 130, 256, 32, True),
    (64, 3, 200, 64, 160, 32, False), (1200, 1, 6, 256, 128, 64, False), (200, 4, 100, 600, 128, 64, False),
    (900, 4, 20, 1000, 96, 32, False), (100, 4, 20, 2000, 128, 128, False), (130, 4, 60, 500, 224, 32, True),
    (500, 4, 10, 520, 128, 128, True)])
def test_sorted_routed(tokens, k, experts, rows, cols, group, up, dtype):
    """The sizes at which a sorted call takes another form: few rows, many small runs, long runs, many matrices."""
    from hoard_amd.ops import q4_matmul, sort_pairs
    w = weights(91, experts, rows, cols, group, BF16, True)
    u = weights(92, experts, rows, cols, group, F16) if up else None
    s = sort_pairs(routing(93, tokens, k, experts).cuda(), experts)
    x = rows_of(94, tokens * k, cols, dtype)
    y = q4_matmul(x, op(w), op(u) if up else None, offsets=s.offsets)
    off = s.offsets.tolist()
    for e in range(experts):
        if off[e + 1] > off[e]:
            R.close(y[off[e]:off[e + 1]], *expect(x[off[e]:off[e + 1]], w, u, e), f"expert {e}")


@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("n,rows,cols,group,dtype", [
    (16, 12400, 128, 64, BF16), (9, 12400, 128, 64, F32), (30, 4200, 160, 32, BF16), (48, 2100, 256, 128, F16),
    (150, 700, 256, 64, BF16), (300, 600, 384, 128, F16), (600, 520, 128, 32, BF16), (700, 3000, 64, 32, F32),
    (1, 4100, 96, 32, F32), (90, 1100, 224, 32, F32), (1100, 2050, 64, 64, F16), (600, 1100, 352, 32, BF16),
    (800, 2050, 320, 64, F16), (300, 1000, 288, 32, F32), (300, 560, 1152, 128, BF16)])
def test_dense_forms(n, rows, cols, group, dtype, up):
    """The sizes at which a dense call takes another form, and odd ones beside them."""
    from hoard_amd.ops import q4_matmul
    w = weights(95, 0, rows, cols, group, F32, True)
    u = weights(90, 0, rows, cols, group, F16) if up else None
    x = rows_of(96, n, cols, dtype)
    R.close(q4_matmul(x, op(w), op(u) if up else None), *expect(x, w, u), "y")


def near_fp32(x, m):
    """(value, bound) of fp32 products whose terms (q - z) x are formed without an offset.

    x is held to 2^-24 of itself or 2^-39 of its group's largest magnitude.  A group's sum takes two terms a column,
    each adding at most a whole step (twice U32) of the sum of their magnitudes; its scaling, the groups' sum and the
    parts of a split row round a few times more.  Below the normal range every term and sum rounds to 2^-149."""
    codes, s, z = m
    w = R.dense(codes, s, z)[0]
    group, groups = w.shape[-1] // s.shape[-1], s.shape[-1]
    x = x.cpu().to(torch.float64)
    most = x.abs().view(len(x), groups, group).amax(dim=2).repeat_interleave(group, dim=1)
    held = torch.maximum(2.0 ** -24 * x.abs(), 2.0 ** -39 * most)
    size = x.abs() @ w.abs().t()
    step = 2.0 ** -149 * (groups + 20 + 2 * group * s.cpu().to(torch.float64).abs().sum(-1))
    return x @ w.t(), held @ w.abs().t() + (4 * group + groups + 24) * R.U32 * size + step


F32_FORMS = [(1, 512, 2048, 128), (1, 4100, 256, 32), (3, 64, 640, 64), (16, 100, 1024, 32), (20, 96, 2080, 32),
             (40, 2048, 512, 128), (70, 65, 1920, 64), (300, 1500, 384, 32)]


@pytest.mark.parametrize("scale", [1e-40, 1e-37, 1.0, 1e34])
@pytest.mark.parametrize("n,rows,cols,group", F32_FORMS)
def test_f32_magnitudes(n, rows, cols, group, scale):
    from hoard_amd.ops import q4_matmul
    print("q4 f32 magnitudes", n, rows, cols, group, scale, flush=True)
    w = weights(61, 0, rows, cols, group, F32, True)
    x = (torch.randn((n, cols), generator=torch.Generator().manual_seed(62), dtype=torch.float64) * scale).to(F32)
    x[0, :group] = 0.0  # a group of nothing
    R.close(q4_matmul(x.cuda(), op(w)), *near_fp32(x, w), "y")


@pytest.mark.parametrize("n,rows,cols,group", F32_FORMS)
def test_f32_small_beside_large(n, rows, cols, group):
    """Values 2^-25 of the group's largest, which itself meets a weight of zero, keep their digits."""
    from hoard_amd.ops import q4_matmul
    print("q4 f32 small beside large", n, rows, cols, group, flush=True)
    codes, s, z = weights(63, 0, rows, cols, group, F32, False)
    codes = codes.clone()
    codes[:, ::group // 2] = codes[:, ::group // 2] & 0xF0 | 8  # a group's first code: the zero point
    x = torch.randn((n, cols), generator=torch.Generator().manual_seed(64)) * 2.0 ** -25
    x[:, ::group] = 1.9
    w = (codes, s, z)
    R.close(q4_matmul(x.cuda(), op(w)), *near_fp32(x, w), "y")


@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("n,rows,cols,group,dtype", [
    (20, 700, 1184, 32, F32), (70, 2500, 672, 32, F32), (70, 1200, 1088, 64, F32), (130, 2500, 320, 64, F32),
    (400, 1500, 416, 32, F32), (700, 1800, 288, 32, F32), (33, 4100, 640, 128, F32), (100, 2000, 1312, 32, BF16),
    (50, 1300, 640, 128, F16), (17, 8200, 1216, 64, BF16)])
def test_dense_splits(n, rows, cols, group, dtype, up):
    """Sizes on both sides of where a dense call's columns are split over fewer waves, none a multiple of a step."""
    from hoard_amd.ops import q4_matmul
    print("q4 splits", n, rows, cols, group, dtype, up, flush=True)
    w = weights(97, 0, rows, cols, group, BF16, True)
    u = weights(98, 0, rows, cols, group, F32) if up else None
    x = rows_of(99, n, cols, dtype)
    R.close(q4_matmul(x, op(w), op(u) if up else None), *expect(x, w, u), "y")


def test_graphs():
    """Three forms captured and replayed with eager work between, each replay the eager result."""
    from hoard_amd.ops import q4_matmul
    w, many = op(weights(97, 0, 300, 512, 128)), op(weights(98, 4, 300, 512, 128))
    ids = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32).cuda()
    offsets = torch.tensor([0, 5, 5, 80, 99], dtype=torch.int32).cuda()
    x = {n: rows_of(99 + n, n, 512, BF16) for n in (1, 2, 30, 99)}
    calls = [lambda: q4_matmul(x[1], w), lambda: q4_matmul(x[30], w), lambda: q4_matmul(x[2], many, ids=ids),
             lambda: q4_matmul(x[99], many, many, offsets=offsets)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [c() for c in calls]
    for r in range(4):
        for t in got:
            t.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), r
        calls[r]()
        torch.empty(1 << 16, device="cuda").normal_().sum().item()


def test_deterministic_and_streams():
    from hoard_amd.ops import q4_matmul
    w, u = op(weights(61, 0, 300, 1024, 128)), op(weights(62, 0, 300, 1024, 128))
    for n in (1, 9, 90):
        xs = [rows_of(63 + i, n, 1024, BF16) for i in range(2)]
        want = [q4_matmul(x, w, u) for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in xs]
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append([q4_matmul(x, w, u) for _ in range(4)])
        torch.cuda.synchronize()
        for g, e in zip(got, want):
            assert all(torch.equal(y, e) for y in g)


def test_largest_rows():
    """More rows than a grid's second dimension holds, few columns."""
    from hoard_amd.ops import q4_matmul
    w = weights(71, 0, 3, 32, 32)
    x = rows_of(72, 70001, 32, BF16)
    y = q4_matmul(x, op(w))
    R.close(y, *expect(x, w, None), "y")


def test_python_refusals():
    from hoard_amd.ops import Q4Weight, q4_matmul
    codes, scales, _ = weights(81, 0, 8, 128, 64)
    w = Q4Weight(codes, scales)
    x = rows_of(82, 4, 128, F32)
    for call in (lambda: q4_matmul(x.cpu(), w), lambda: q4_matmul(x[:, :64], w), lambda: q4_matmul(x.double(), w),
                 lambda: q4_matmul(rows_of(1, 4, 64, F32), w), lambda: q4_matmul(x, w, out=torch.empty((4, 7), device="cuda")),
                 lambda: q4_matmul(x, w, ids=torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: q4_matmul(x, w, offsets=torch.zeros(3, dtype=torch.int32, device="cuda")),
                 lambda: q4_matmul(x, w, ids=torch.zeros(4, dtype=torch.int64, device="cuda")),
                 lambda: Q4Weight(codes.to(torch.int8), scales), lambda: Q4Weight(codes, scales[:4]),
                 lambda: Q4Weight(codes, scales, scales), lambda: q4_matmul(x, Q4Weight(codes[:4], scales[:4]), w)):
        with pytest.raises(H.HoardError):
            call()

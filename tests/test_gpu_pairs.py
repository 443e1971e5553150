"""The pairs sorted by expert, their rows laid out and taken back, and the gradients, against plain forms."""
import numpy as np
import pytest

import hoard_amd as H
import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make_ids(seed, tokens, k, experts, drop=0.0, skew=False):
    g = np.random.default_rng(seed)
    hi = max(1, experts // 8) if skew else experts
    ids = g.integers(0, hi, (tokens, k)).astype(np.int32)
    if drop:
        out = g.random((tokens, k)) < drop
        ids[out] = g.choice([-1, experts, -2**31, 2**31 - 1], out.sum())
    return torch.from_numpy(ids)


SORTS = [(0, 8, 4, 0.0), (1, 1, 1, 0.0), (1, 8, 128, 0.0), (1, 64, 3, 0.1), (5, 3, 1024, 0.0), (16, 8, 128, 0.3),
         (127, 8, 64, 0.0), (128, 8, 64, 0.0), (129, 8, 64, 0.0), (341, 3, 1000, 0.2), (512, 10, 512, 0.0),
         (700, 7, 2, 0.5), (2048, 8, 127, 0.0), (8192, 8, 1000, 0.1), (8193, 8, 3, 0.0), (66000, 1, 65, 0.2), (5001, 8, 1024, 0.1), (20000, 4, 60, 0.0), (40000, 5, 256, 1.0)]


@pytest.mark.parametrize("tokens,k,experts,drop", SORTS)
@pytest.mark.parametrize("skew", [False, True])
def test_sort(tokens, k, experts, drop, skew):
    from hoard_amd.ops import sort_pairs
    print("sort", tokens, k, experts, flush=True)
    ids = make_ids(1, tokens, k, experts, drop, skew)
    got = sort_pairs(ids.cuda(), experts)
    for name, g, w in zip(got._fields, got, R.sort_pairs(ids, experts)):
        assert torch.equal(g.cpu(), w), name


def test_sort_many_pairs():
    from hoard_amd.ops import sort_pairs
    ids = make_ids(2, 300000, 8, 128, 0.05)
    place, order, offsets = sort_pairs(ids.cuda(), 128)
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat < 0) | (flat >= 128), 128, flat)
    ranked, by = torch.sort(key, stable=True)
    by = torch.where(ranked < 128, by, -1).to(torch.int32)
    assert torch.equal(order.cpu(), by)
    assert torch.equal(offsets.cpu().to(torch.int64), torch.searchsorted(ranked, torch.arange(129)))
    kept = key < 128
    assert torch.equal(order.cpu()[place.cpu().reshape(-1)[kept].to(torch.int64)].to(torch.int64), torch.nonzero(kept).view(-1))
    assert (place.cpu().reshape(-1)[~kept] == -1).all()


def data(seed, *size, dtype, off=0):
    """A dense tensor whose first element lies `off` elements after a 16-byte boundary."""
    t = torch.randn(int(np.prod(size)), generator=torch.Generator().manual_seed(seed)).to(dtype)
    buf = torch.empty(t.numel() + off, dtype=dtype, device="cuda")
    buf[off:] = t.cuda()
    return buf[off:].view(*size)


ROWS = [
    # tokens, k, experts, n, type, share dropped, elements off alignment
    (1, 1, 1, 1, F32, 0.0, 0), (1, 8, 128, 2048, BF16, 0.0, 0), (1, 3, 4, 7, F16, 0.4, 1), (2, 64, 5, 100, F32, 0.2, 0),
    (5, 2, 3, 8, BF16, 1.0, 0), (16, 8, 128, 2048, F32, 0.0, 0), (33, 10, 512, 513, BF16, 0.1, 1),
    (64, 4, 8, 4096, F16, 0.0, 0), (100, 6, 16, 1023, F32, 0.3, 3), (257, 8, 64, 264, BF16, 0.0, 1),
    (300, 1, 7, 2049, F16, 0.2, 0), (1000, 8, 32, 65, F32, 0.0, 0), (3, 17, 40, 9000, BF16, 0.1, 0),
]


@pytest.mark.parametrize("tokens,k,experts,n,dtype,drop,off", ROWS)
@pytest.mark.parametrize("weighted", [False, True])
def test_gather(tokens, k, experts, n, dtype, drop, off, weighted):
    from hoard_amd.ops import sort_gather
    ids = make_ids(3, tokens, k, experts, drop)
    place = R.sort_pairs(ids, experts)[0]
    x = data(4, tokens, n, dtype=dtype, off=off)
    w = data(5, tokens, k, dtype=F32, off=off) if weighted else None
    out = data(6, tokens * k, n, dtype=dtype, off=off).fill_(7.0)
    assert sort_gather(x, place.cuda(), w, out=out) is out
    want = torch.full((tokens * k, n), 7.0, dtype=torch.float64)
    bound = torch.zeros_like(want)
    at = place.reshape(-1).to(torch.int64)
    p = torch.nonzero(at >= 0).view(-1)
    rows = x.cpu().to(torch.float64)[p // k]
    if weighted:
        rows = rows * w.cpu().to(torch.float64).reshape(-1)[p].unsqueeze(1)
        bound[at[p]] = R.stored(rows, R.U32 * rows.abs(), dtype)
    want[at[p]] = rows
    R.close(out, want, bound, "xs")


@pytest.mark.parametrize("tokens,k,experts,n,dtype,drop,off", ROWS)
@pytest.mark.parametrize("weighted,residual", [(False, False), (True, False), (True, True), (False, True)])
def test_combine(tokens, k, experts, n, dtype, drop, off, weighted, residual):
    from hoard_amd.ops import sort_combine
    ids = make_ids(7, tokens, k, experts, drop)
    place, _, offsets = R.sort_pairs(ids, experts)
    y = data(8, tokens * k, n, dtype=dtype, off=off)
    y[int(offsets[-1]):] = float("nan")  # rows that no pair names
    w = data(9, tokens, k, dtype=F32, off=off) if weighted else None
    res = data(10, tokens, n, dtype=dtype, off=off) if residual else None
    if weighted and drop:
        w[(place < 0).cuda()] = float("inf")  # weights of dropped pairs
    out = sort_combine(y, place.cuda(), w, res)
    at = place.reshape(-1).to(torch.int64)
    rows = torch.where((at >= 0).unsqueeze(1), y.cpu().to(torch.float64)[at.clamp(min=0)], 0.0).view(tokens, k, n)
    if weighted:
        rows = rows * torch.where(place >= 0, w.cpu().to(torch.float64), 0.0).unsqueeze(2)
    want, mag = rows.sum(1), rows.abs().sum(1)
    if residual:
        want, mag = want + res.cpu().to(torch.float64), mag + res.cpu().to(torch.float64).abs()
    R.close(out, want, R.stored(want, (k + 1) * R.U32 * mag, dtype), "out")
    if residual:  # in place
        assert sort_combine(y, place.cuda(), w, res, out=res) is res
        assert torch.equal(res, out)


@pytest.mark.parametrize("tokens,k,experts,n,dtype,drop,off", ROWS)
def test_combine_grad(tokens, k, experts, n, dtype, drop, off):
    from hoard_amd.ops import sort_combine_grad
    ids = make_ids(11, tokens, k, experts, drop)
    place, _, offsets = R.sort_pairs(ids, experts)
    y = data(12, tokens * k, n, dtype=dtype, off=off)
    y[int(offsets[-1]):] = float("nan")
    w, dout = data(13, tokens, k, dtype=F32, off=off), data(14, tokens, n, dtype=dtype, off=off)
    dy = data(15, tokens * k, n, dtype=dtype, off=off).fill_(7.0)
    got, dw = sort_combine_grad(dout, y, place.cuda(), w, dy=dy)
    assert got is dy
    at = place.reshape(-1).to(torch.int64)
    p = torch.nonzero(at >= 0).view(-1)
    d, y64, w64 = dout.cpu().to(torch.float64)[p // k], y.cpu().to(torch.float64)[at[p]], w.cpu().to(torch.float64).reshape(-1)[p]
    want, bound = torch.full((tokens * k, n), 7.0, dtype=torch.float64), torch.zeros((tokens * k, n), dtype=torch.float64)
    want[at[p]] = w64.unsqueeze(1) * d
    bound[at[p]] = R.stored(want[at[p]], R.U32 * want[at[p]].abs(), dtype)
    R.close(dy, want, bound, "dy")
    ww, wb = torch.zeros(tokens * k, dtype=torch.float64), torch.zeros(tokens * k, dtype=torch.float64)
    ww[p] = (d * y64).sum(1)
    wb[p] = (n + 1) * R.U32 * (d * y64).abs().sum(1)
    R.close(dw.reshape(-1), ww, wb, "dw")


@pytest.mark.parametrize("n", [5, 64, 2047, 2049, 5003])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_combine_grad_in_place(n, dtype):
    """dy over y."""
    from hoard_amd.ops import sort_combine_grad, sort_pairs
    tokens, k = 30, 5
    s = sort_pairs(make_ids(50, tokens, k, 9, 0.1).cuda(), 9)
    y, w, dout = data(51, tokens * k, n, dtype=dtype), data(52, tokens, k, dtype=F32), data(53, tokens, n, dtype=dtype)
    dy, dw = sort_combine_grad(dout, y, s.place, w, dy=y.clone())
    got, dw2 = sort_combine_grad(dout, y, s.place, w, dy=y)
    assert got is y and torch.equal(got, dy) and torch.equal(dw, dw2)


def test_gather_and_combine_are_adjoint():
    """<gather(x), g> = <x, combine(g)>, the gradient of each by the other, and dw against differences."""
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather, sort_pairs
    tokens, k, experts, n = 60, 6, 20, 300
    s = sort_pairs(make_ids(16, tokens, k, experts, 0.2).cuda(), experts)
    x, g = data(17, tokens, n, dtype=F32), data(18, tokens * k, n, dtype=F32)
    xs = sort_gather(x, s.place, out=torch.zeros_like(g))
    live = torch.arange(tokens * k, device="cuda") < s.offsets[-1]
    left = (xs.double() * g.double())[live].sum()
    right = (x.double() * sort_combine(g, s.place).double()).sum()
    scale = (xs.double() * g.double()).abs().sum()
    assert abs(float(left - right)) <= (k + 2) * R.U32 * float(scale)
    w, dout = data(19, tokens, k, dtype=F32), data(20, tokens, n, dtype=F32)
    dy, dw = sort_combine_grad(dout, g, s.place, w)
    # the combine is linear in w and in y: a difference of any step is the derivative
    dirw = data(21, tokens, k, dtype=F32)
    diff = (sort_combine(g, s.place, w + dirw).double() - sort_combine(g, s.place, w).double()) * dout.double()
    want = (dw.double() * dirw.double()).sum()
    # both combines round k + 1 times relative to the sum of magnitudes of at most sum |w| |y|, w + dirw once more
    mag = (sort_combine(g.abs(), s.place, w.abs() * 2 + dirw.abs()).double() * dout.double().abs()).sum()
    assert abs(float(diff.sum() - want)) <= (2 * k + 4 + n) * R.U32 * float(mag)
    diry = data(22, tokens * k, n, dtype=F32)
    diff = (sort_combine(g + diry, s.place, w).double() - sort_combine(g, s.place, w).double()) * dout.double()
    want = (dy.double() * diry.double())[live].sum()
    mag = (sort_combine(2 * g.abs() + diry.abs(), s.place, w.abs()).double() * dout.double().abs()).sum()
    assert abs(float(diff.sum() - want)) <= (2 * k + 6) * R.U32 * float(mag)


def test_places_out_of_range_are_dropped():
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather
    place = torch.tensor([[0, 6, -7], [2**31 - 1, 1, -2**31]], dtype=torch.int32).cuda()
    x = data(23, 2, 40, dtype=F32)
    xs = sort_gather(x, place, out=torch.full((6, 40), 7.0, device="cuda"))
    assert torch.equal(xs[0], x[0]) and torch.equal(xs[1], x[1]) and (xs[2:] == 7.0).all()
    y, w = data(24, 6, 40, dtype=F32), torch.ones((2, 3), device="cuda")
    assert torch.equal(sort_combine(y, place, w), y[:2])
    dy, dw = sort_combine_grad(x, y, place, w)
    assert torch.equal(dy[:2], x) and (dy[2:] == 0).all()
    assert ((dw != 0).cpu() == torch.tensor([[True, False, False], [False, True, False]])).all()


def test_streams_and_graph():
    """Two calls at once on their own workspaces, and a captured chain replayed with eager work between."""
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather, sort_pairs
    tokens, k, experts, n = 400, 8, 64, 256
    cases = [(make_ids(30 + i, tokens, k, experts, 0.1).cuda(), data(32 + i, tokens, n, dtype=BF16), data(34 + i, tokens, k, dtype=F32))
             for i in range(2)]

    def chain(ids, x, w):
        s = sort_pairs(ids, experts)
        xs = sort_gather(x, s.place, out=torch.zeros((tokens * k, n), dtype=BF16, device="cuda"))
        out = sort_combine(xs, s.place, w, x)
        return (*s, xs, out, *sort_combine_grad(out, xs, s.place, w, dy=torch.zeros_like(xs)))

    want = [[t.clone() for t in chain(*c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, st in zip(cases, streams):
        with torch.cuda.stream(st):
            got.append([chain(*c) for _ in range(3)])
    torch.cuda.synchronize()
    for g, e in zip(got, want):
        for once in g:
            assert all(torch.equal(a, b) for a, b in zip(once, e))
    graphs = []
    for c, st in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs = chain(*c)
        graphs.append((g, outs))
    for r in range(4):
        for (g, outs), e in zip(graphs, want):
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, e)), r
        chain(*cases[r % 2])
        torch.empty(1 << 16, device="cuda").normal_().sum().item()


def test_python_refusals():
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather, sort_pairs
    ids = make_ids(40, 4, 2, 8).cuda()
    s = sort_pairs(ids, 8)
    x, y, w = data(41, 4, 16, dtype=F32), data(42, 8, 16, dtype=F32), data(43, 4, 2, dtype=F32)
    for call in (lambda: sort_pairs(ids.cpu(), 8), lambda: sort_pairs(ids.long(), 8), lambda: sort_pairs(ids, 0),
                 lambda: sort_pairs(ids, 1025), lambda: sort_pairs(ids.view(-1), 8), lambda: sort_pairs(ids.t(), 8),
                 lambda: sort_gather(x[:3], s.place), lambda: sort_gather(x.double(), s.place),
                 lambda: sort_gather(x, s.place, w[:2]), lambda: sort_combine(y[:7], s.place),
                 lambda: sort_combine(y, s.place, w, x[:, :8]), lambda: sort_combine(y, s.place, w.half()),
                 lambda: sort_combine_grad(x, y, s.place, None), lambda: sort_combine_grad(y, y, s.place, w),
                 lambda: sort_combine(y, s.place, out=y)):
        with pytest.raises(H.HoardError):
            call()

"""fp32 4-bit products in all their forms, by offsets, by ids and with a second matrix, within the mean square error
that two f16 planes of x and exact codes allow."""
import pytest

import opsbounds as B

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16, F16 = torch.bfloat16, torch.float16


def matrix(seed, lead, rows, cols, group, scales):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, rows, cols // 2), generator=g, dtype=torch.uint8)
    s = (torch.rand((*lead, rows, cols // group), generator=g) * 0.01).to(scales)
    return codes.cuda(), s.cuda(), torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8).cuda()


def one(m, e):
    return tuple(t[e] for t in m)


def check(parts):
    """parts: (results, value, mean square) of some rows each."""
    got, value, square = (torch.cat([p[i].cpu() for p in parts]) for i in range(3))
    ratio = B.rms_ratio(got, value, square)
    print("rms ratio", ratio, flush=True)
    assert ratio <= 1.0


def expect(x, w, u):
    v = B.fp32_product(x, w)
    return v if u is None else B.fp32_swiglu(*v, *B.fp32_product(x, u))


def routing(tokens, k, experts):
    g = torch.Generator().manual_seed(7)
    return torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(tokens)]).to(torch.int32)


@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("tokens,k,experts,rows,cols,group", [
    (10, 4, 16, 200, 384, 128), (3, 2, 40, 96, 256, 64), (80, 4, 40, 1000, 320, 64), (40, 4, 40, 1000, 512, 128),
    (160, 4, 64, 1900, 160, 32), (600, 4, 20, 1000, 256, 128), (500, 4, 10, 520, 224, 32)])
def test_sorted(tokens, k, experts, rows, cols, group, up):
    from hoard_amd.ops import Q4Weight, q4_matmul, sort_pairs
    print("q4 fp32 sorted", tokens, k, experts, rows, cols, group, up, flush=True)
    w = matrix(1, (experts,), rows, cols, group, BF16)
    u = matrix(2, (experts,), rows, cols, group, F16) if up else None
    s = sort_pairs(routing(tokens, k, experts).cuda(), experts)
    x = torch.randn((tokens * k, cols), generator=torch.Generator().manual_seed(3)).cuda()
    y = q4_matmul(x, Q4Weight(*w), Q4Weight(*u) if up else None, offsets=s.offsets)
    off = s.offsets.tolist()
    check([(y[a:b], *expect(x[a:b], one(w, e), one(u, e) if up else None))
           for e, (a, b) in enumerate(zip(off, off[1:])) if b > a])


@pytest.mark.parametrize("up", [False, True])
def test_ids(up):
    from hoard_amd.ops import Q4Weight, q4_matmul
    tokens, k, experts, rows, cols, group = 9, 4, 12, 130, 768, 64
    w = matrix(1, (experts,), rows, cols, group, BF16)
    u = matrix(2, (experts,), rows, cols, group, F16) if up else None
    ids = routing(tokens, k, experts)
    x = torch.randn((tokens, cols), generator=torch.Generator().manual_seed(3)).cuda()
    y = q4_matmul(x, Q4Weight(*w), Q4Weight(*u) if up else None, ids=ids.cuda())
    check([(y[p:p + 1], *expect(x[p // k:p // k + 1], one(w, e), one(u, e) if up else None))
           for p, e in enumerate(ids.view(-1).tolist())])


@pytest.mark.parametrize("up", [False, True])
@pytest.mark.parametrize("n,rows,cols,group", [
    (1, 512, 2048, 128), (1, 4200, 1024, 32), (5, 200, 640, 64), (40, 2048, 512, 128), (130, 2500, 320, 64),
    (300, 1500, 384, 32), (700, 1800, 512, 128)])
def test_dense(n, rows, cols, group, up):
    from hoard_amd.ops import Q4Weight, q4_matmul
    print("q4 fp32 dense", n, rows, cols, group, up, flush=True)
    w = matrix(1, (), rows, cols, group, BF16)
    u = matrix(2, (), rows, cols, group, F16) if up else None
    x = torch.randn((n, cols), generator=torch.Generator().manual_seed(3)).cuda()
    y = q4_matmul(x, Q4Weight(*w), Q4Weight(*u) if up else None)
    check([(y, *expect(x, w, u))])

"""How often a 16-bit result of a 4-bit product is not the rounded 64-bit one, and silu far below zero."""
import pytest

import opsbounds as B

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F16, BF16 = torch.float16, torch.bfloat16


def matrix(seed, lead, rows, cols, group):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (*lead, rows, cols // 2), generator=g, dtype=torch.uint8)
    return codes.cuda(), (torch.rand((*lead, rows, cols // group), generator=g) * 0.01).to(BF16).cuda(), None


# prompts: the sizes of each form that takes x in its own order, by rows of x and of W
PROMPTS = [(128, 4096, 128), (130, 4096, 32), (256, 4096, 64), (512, 4096, 128), (700, 4096, 128), (700, 2080, 32)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,rows,group", PROMPTS)
def test_prompt(n, rows, group, dtype):
    from hoard_amd.ops import Q4Weight, q4_matmul
    print("q4 rounding", n, rows, group, dtype, flush=True)
    m = matrix(1, (), rows, 2048, group)
    x = torch.randn((n, 2048), generator=torch.Generator().manual_seed(2)).to(dtype)
    value, expected = B.expected_over_border(x, m, dtype)
    over = B.over_border(q4_matmul(x.cuda(), Q4Weight(*m)), value)
    print("over a border", over, "expected", expected, "of", value.numel(), flush=True)
    assert over <= B.allowed(expected)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,rows,group", [(1, 4096, 128), (13, 2048, 32), (20, 2048, 64), (60, 2048, 128)])
def test_few_rows(n, rows, group, dtype):
    """Dots and the tiles of few rows sum codes with an offset of 16 (f16 tiles none)."""
    from hoard_amd.ops import Q4Weight, q4_matmul
    print("q4 rounding", n, rows, group, dtype, flush=True)
    m = matrix(5, (), rows, 2048, group)
    x = torch.randn((n, 2048), generator=torch.Generator().manual_seed(6)).to(dtype)
    value, expected = B.expected_over_border(x, m, dtype, 0 if dtype == F16 and n > 1 else 16)
    over = B.over_border(q4_matmul(x.cuda(), Q4Weight(*m)), value)
    print("over a border", over, "expected", expected, "of", value.numel(), flush=True)
    assert over <= B.allowed(expected)


@pytest.mark.parametrize("tokens,k,experts,rows,group", [(16, 8, 64, 512, 128), (120, 4, 20, 768, 64), (512, 4, 20, 768, 128)])
def test_sorted(tokens, k, experts, rows, group):
    from hoard_amd.ops import Q4Weight, q4_matmul, sort_pairs
    g = torch.Generator().manual_seed(3)
    ids = torch.stack([torch.randperm(experts, generator=g)[:k] for _ in range(tokens)]).to(torch.int32).cuda()
    s = sort_pairs(ids, experts)
    m = matrix(4, (experts,), rows, 2048, group)
    x = torch.randn((tokens * k, 2048), generator=g).to(BF16)
    y = q4_matmul(x.cuda(), Q4Weight(*m), offsets=s.offsets)
    off, over, expected = s.offsets.tolist(), 0, 0.0
    for e in range(experts):
        a, b = off[e], off[e + 1]
        if b > a:
            value, more = B.expected_over_border(x[a:b], (m[0][e], m[1][e], None), BF16)
            over += B.over_border(y[a:b], value)
            expected += more
    print("over a border", over, "expected", expected, "of", y.numel(), flush=True)
    assert over <= B.allowed(expected)


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("n", [1, 20, 400])
def test_silu_of_far_negatives(n, dtype):
    """silu(g) down to g = -88, where 1 / (1 + e^-g) is below the normal range, times an u that brings it back."""
    from hoard_amd.ops import Q4Weight, q4_matmul
    rows = 4096
    ones = torch.full((rows, 16), 0x99, dtype=torch.uint8, device="cuda")  # codes of 9: weights of one scale
    scale = torch.linspace(0.25, 1.0, rows).to(BF16).to(torch.float32).view(rows, 1)
    w, u = Q4Weight(ones, scale.cuda()), Q4Weight(ones, torch.full((rows, 1), 1e34, device="cuda"))
    x = torch.full((n, 32), -2.75, dtype=dtype, device="cuda")
    y = q4_matmul(x, w, u)
    g = -88.0 * scale.double().view(1, rows)
    want = (g / (1 + torch.exp(-g)) * (-88.0 * float(torch.tensor(1e34)))).expand(n, rows)
    # g rounds once as a product of its scale, u once; e^-g is off by that of g and 2^-24 |g| of its exponent's product;
    # the exponential, the sum, the reciprocal and the products 8 more; half a step of the type
    bound = want.abs() * (2.0 ** -24 * (3 * g.abs() + 16) + torch.finfo(dtype).eps / 2)
    off = (y.cpu().double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())

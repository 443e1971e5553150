"""The bounds of the 4-bit products' tests refuse what they are there to refuse: mistakes planted in a model, on the CPU."""
import pytest

torch = pytest.importorskip("torch")

import opsbounds as B  # noqa: E402


def model(x, m, bias):
    """A product as the matrix tiles form it, codes plus `bias`: 32 columns an instruction, each result rounded to 32 bits."""
    codes, scales, _ = m
    q = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.float64) + bias
    groups = scales.shape[-1]
    group = q.shape[-1] // groups
    x, s = x.to(torch.float64), scales.to(torch.float64)
    f32 = lambda t: t.to(torch.float32).to(torch.float64)  # noqa: E731
    acc = torch.zeros((x.shape[0], q.shape[0]), dtype=torch.float64)
    for g in range(groups):
        d, sums = torch.zeros_like(acc), torch.zeros((x.shape[0], 1), dtype=torch.float64)
        for c in range(g * group, (g + 1) * group, 32):
            d = f32(d + x[:, c:c + 32] @ q[:, c:c + 32].t())
            sums = f32(sums + x[:, c:c + 32].sum(1, keepdim=True))
        acc = f32(acc + s[:, g] * f32(d - (8 + bias) * sums))
    return acc


def matrix(seed, rows, cols, group):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8)
    return codes, (torch.rand((rows, cols // group), generator=g) * 0.01).to(torch.bfloat16), None


def test_offset_of_128_is_refused():
    m = matrix(1, 512, 2048, 128)
    x = torch.randn((128, 2048), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    value, expected = B.expected_over_border(x, m, torch.bfloat16)
    over = {bias: B.over_border(model(x, m, bias).to(torch.bfloat16), value) for bias in (0, 128)}
    assert over[0] <= B.allowed(expected) < over[128], (over, expected)


def planes(x, group, low=True):
    """fp32 x as the matrix tiles hold it: two f16 planes of x times a power of two a group."""
    most = x.abs().view(len(x), -1, group).amax(dim=2, keepdim=True)
    power = torch.exp2(14 - torch.floor(torch.log2(most.to(torch.float64))))
    v = x.to(torch.float64).view(len(x), -1, group) * power
    high = v.to(torch.float16).to(torch.float64)
    held = high + (v - high).to(torch.float16).to(torch.float64) if low else high
    return (held / power).view(x.shape)


def test_two_planes_hold_23_bits():
    x = torch.randn((4096, 128), generator=torch.Generator().manual_seed(3))
    off = ((planes(x, 128) - x.to(torch.float64)).abs() / x.to(torch.float64).abs())
    near = x.abs() >= 2.0 ** -15 * x.abs().amax(dim=1, keepdim=True)
    assert 2.0 ** -24 < off[near].max() <= 2.0 ** -23


@pytest.mark.parametrize("tokens,rows,cols,group", [(8, 96, 512, 128), (33, 48, 320, 64), (4, 40, 96, 32), (64, 64, 4096, 128)])
def test_one_plane_is_refused(tokens, rows, cols, group):
    """fp32 products with x in f16 stay far outside what the two planes may be off, with a second matrix too."""
    m, up = matrix(4, rows, cols, group), matrix(5, rows, cols, group)
    x = torch.randn((tokens, cols), generator=torch.Generator().manual_seed(6))
    (g, vg), (u, vu) = B.fp32_product(x, m), B.fp32_product(x, up)
    both, v = B.fp32_swiglu(g, vg, u, vu)
    for low in (True, False):
        held = planes(x, group, low)
        g1, u1 = B.fp32_product(held, m)[0], B.fp32_product(held, up)[0]
        for ratio in (B.rms_ratio(g1, g, vg), B.rms_ratio(g1 / (1 + torch.exp(-g1)) * u1, both, v)):
            assert ratio <= 1.0 if low else ratio > 10.0, (low, ratio)

"""Mistakes planted in the plain forms of the attention half, on the CPU: the bounds of the tests refuse each."""
import math

import pytest

import attnref as A

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def off(got, want, bound):
    """Whether a result misses its bound somewhere."""
    return bool(((got - want).abs() > bound).any())


@pytest.mark.parametrize("dtype", [F32, torch.float16, BF16])
def test_heads(dtype):
    x = torch.randn((5, 3, 64), generator=gen(1)).to(dtype)
    w = 1 + 0.2 * torch.randn(64, generator=gen(2))
    pos, freq = torch.randint(0, 100000, (5,), generator=gen(3)), 10000.0 ** (-torch.arange(16, dtype=A.D) / 16)
    rope = (pos, freq, None, False)
    want, bound, _ = A.heads(x, w, rope, 1e-6, 0.0)
    bound = A.stored(want, bound, dtype)
    assert not off(want.to(dtype).to(A.D), want, bound)
    mistakes = {
        "no norm": A.heads(x, None, rope, 1e-6, 0.0)[0] * w,
        "weight's offset": A.heads(x, w, rope, 1e-6, 1.0)[0],
        "pairs": A.heads(x, w, (pos, freq, None, True), 1e-6, 0.0)[0],
        "next position": A.heads(x, w, (pos + 1, freq, None, False), 1e-6, 0.0)[0],
        "angle backwards": A.rotate(A.head_norm(A.t64(x), A.t64(w), 1e-6, 0.0)[0], torch.zeros(x.shape, dtype=A.D), rope, True)[0],
        "norm behind the rotation": A.head_norm(A.rotate(A.t64(x), torch.zeros(x.shape, dtype=A.D), rope)[0], A.t64(w), 1e-6, 0.0)[0],
        "another head's sum": A.heads(x, w, rope, 1e-6, 0.0)[0].roll(1, 1),
    }
    if dtype == F32:
        mistakes["angles in 32 bits"] = A.heads(x, w, (pos, (freq.to(F32) * (1 + 1e-6)).to(A.D), None, False), 1e-6, 0.0)[0]
    for name, got in mistakes.items():
        assert off(got, want, bound), name


def test_heads_grad():
    x, dz = torch.randn((40, 2, 32), generator=gen(4)), torch.randn((40, 2, 32), generator=gen(5))
    w = 1 + 0.2 * torch.randn(32, generator=gen(6))
    pos, freq = torch.arange(40), 100.0 ** (-torch.arange(8, dtype=A.D) / 8)
    rope = (pos, freq, None, True)
    rho = A.head_norm(A.t64(x), A.t64(w), 1e-6, 0.0)[2]
    dx, ex, dw, ew = A.heads_grad(dz, x, w, rope, rho, 0.0)
    ex = A.stored(dx, ex, F32)
    leaf, wl = A.t64(x).requires_grad_(True), A.t64(w).requires_grad_(True)
    y = leaf / torch.sqrt(leaf.square().mean(-1, keepdim=True) + 1e-6) * wl
    gx, gw = torch.autograd.grad(A.rotate(y, torch.zeros(x.shape, dtype=A.D), rope)[0], [leaf, wl], A.t64(dz))
    assert not off(gx, dx, ex) and not off(gw, dw, ew)
    assert off(A.heads_grad(dz, x, w, (pos + 1, freq, None, True), rho, 0.0)[0], dx, ex)
    assert off(rho.unsqueeze(-1) * A.t64(w) * A.rotate(A.t64(dz), torch.zeros(x.shape, dtype=A.D), rope, True)[0], dx, ex)
    assert off(A.heads_grad(dz[1:], x[1:], w, (pos[1:], freq, None, True), rho[1:], 0.0)[2], dw, ew)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention(dtype):
    k, v = (torch.randn((6, 1, 16, 64), generator=gen(s)).to(torch.float16) for s in (7, 8))
    q = (2.0 * torch.randn((2, 4, 64), generator=gen(9))).to(dtype)
    pages = torch.tensor([[4, 0, 5, 1]], dtype=torch.int32)
    lens = torch.tensor([[49, 50]], dtype=torch.int32)
    run = lambda **kw: A.attention(**{**dict(q=q, k=k, v=v, ks=None, vs=None, pages=pages, lens=lens, scale=0.125, dtype=dtype), **kw})  # noqa: E731
    want, bound, lse, lse_bound = run()
    bound, lse_bound = A.stored(want, bound, dtype), A.stored(lse, lse_bound, F32)
    assert not off(want.to(dtype).to(A.D), want, bound)
    moved = pages.clone()
    moved[0, 3] = 2
    mistakes = {"one key more": run(lens=lens + 1), "one key less": run(lens=lens - 1), "another page": run(pages=moved),
                "rows exchanged": run(lens=lens.flip(1)), "scale": run(scale=0.1255 if dtype == F32 else 0.13),
                "keys for values": run(v=k), "cache as fp8": run(k=k.to(torch.float8_e4m3fn).to(torch.float16))}
    for name, got in mistakes.items():
        assert off(got[0], want, bound) or off(got[2], lse, lse_bound), name
    if dtype == F32:  # weights and queries of one 16-bit plane
        assert off(run(q=q.to(torch.float16).to(F32))[0], want, bound)
    assert math.isinf(float(run(lens=lens * 0)[2][0, 0]))


def test_quantised():
    x = torch.randn((9, 4, 32), generator=gen(10))
    x[3, 1] = 0.0
    q, step = A.quantised(x)
    assert ((A.values(q, step) - A.t64(x)).abs() <= 0.5001 * A.t64(step).unsqueeze(-1)).all() and not q[3, 1].any() and step[3, 1] == 0
    assert int(q.abs().amax()) == 127

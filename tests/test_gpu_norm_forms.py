"""The norms' kernels by row length and count: several rows a group, rows past the caches, odd lengths, all types."""
import pytest

import test_gpu_norm as N

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# rows, columns: for each length of row more rows than groups, without and with the rows going past the caches
SIZES = [(1500, 1021), (4300, 1021), (15001, 301), (900, 2040), (2300, 2043), (300, 4093), (1100, 4093), (270, 8190), (700, 8189)]
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32), (F16, F16)]
GATES = [dict(gate="channel"), dict(gate="token", sigmoid=True, scale=0.5), dict(gate="full", sigmoid=True, offset=1.0), dict(post=False)]
CASES = [dict(m=m, n=n, dtype=t, res=r, **GATES[(i + j) % 4]) for i, (m, n) in enumerate(SIZES) for j, (t, r) in enumerate(TYPES)]
IDS = ["-".join(str(v).replace("torch.", "") for v in c.values()) for c in CASES]


@pytest.mark.parametrize("kw", CASES, ids=IDS)
def test_forward(kw):
    N.test_forward(kw)


@pytest.mark.parametrize("kw", CASES, ids=IDS)
def test_backward(kw):
    N.test_backward(kw, "both")


@pytest.mark.parametrize("n", [1021, 4093, 8189])
def test_in_place(n):
    """r_out over r, and the same result on a second call, at rows past the caches."""
    from hoard_amd.ops import norm_forward
    case = N.Case(m=(9 << 20) // (2 * n), n=n, dtype=BF16, res=F32, gate="channel")
    want = case.forward()
    r = case.r.clone()
    got = norm_forward(r, **case.par, **case.kw, r_out=r)
    assert torch.equal(got.r_out, want.r_out) and torch.equal(got.h, want.h)

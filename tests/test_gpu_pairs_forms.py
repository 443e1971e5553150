"""Sorted rows beyond 16 MB, which go past the caches, at a length that is no multiple of 8, in every type and in place."""
import pytest

import test_gpu_pairs as P

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SIZES = [(600, 8, 40, 2045), (4001, 3, 9, 701)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,k,experts,n", SIZES)
def test_rows(tokens, k, experts, n, dtype):
    size = (tokens, k, experts, n, dtype, 0.1, 1)
    assert tokens * k * n * dtype.itemsize >= 16 << 20
    for weighted in (False, True):
        print("gather", size, weighted, flush=True)
        P.test_gather(*size, weighted)
        print("combine", size, weighted, flush=True)
        P.test_combine(*size, weighted, True)
    print("combine_grad", size, flush=True)
    P.test_combine_grad(*size)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,k,experts,n", SIZES)
def test_gradient_in_place(tokens, k, experts, n, dtype):
    from hoard_amd.ops import sort_combine_grad, sort_pairs
    s = sort_pairs(P.make_ids(50, tokens, k, experts, 0.1).cuda(), experts)
    y, w = P.data(51, tokens * k, n, dtype=dtype), P.data(52, tokens, k, dtype=F32)
    dout = P.data(53, tokens, n, dtype=dtype)
    dy, dw = sort_combine_grad(dout, y, s.place, w, dy=y.clone())
    got, dw2 = sort_combine_grad(dout, y, s.place, w, dy=y)
    assert got is y and torch.equal(got, dy) and torch.equal(dw, dw2)

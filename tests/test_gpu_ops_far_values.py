"""Arrays of more than 2^31 elements, with values that differ from what the buffers held before the call."""
import ctypes

import pytest

import hoard_amd as H
import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16
D = torch.float64


def test_combine_and_gradient_far():
    """Weights that differ by slot and gradients other than the rows: every pair's row is its own, at both ends of each
    expert's rows and around the element 2^31, in place of y."""
    from hoard_amd.ops import sort_combine, sort_combine_grad, sort_gather, sort_pairs
    tokens, k, n = 132000, 8, 2048
    assert tokens * k * n > 2**31
    ids = torch.arange(k, dtype=torch.int32).repeat(tokens, 1).cuda()  # expert j holds slot j of every token
    s = sort_pairs(ids, k)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dout = (torch.randint(-8, 8, (tokens, n), device="cuda", dtype=torch.int8, generator=g).to(BF16) for _ in range(2))
    w = torch.arange(1, k + 1, dtype=torch.float32, device="cuda").repeat(tokens, 1)
    far = 2**31 // n  # the row of element 2^31, of expert far // tokens
    at = sorted({j * tokens + t for j in range(k) for t in (0, tokens - 1)} | {far - 1, far, far + 1})
    xs = sort_gather(x, s.place, w)
    for row in at:
        assert torch.equal(xs[row], x[row % tokens] * (row // tokens + 1)), row
    out = sort_combine(xs, s.place, w)
    ends = torch.tensor([0, 1, 65999, tokens - 2, tokens - 1], device="cuda")
    squares = sum((j + 1) ** 2 for j in range(k))  # 204 |x|: exact before it is stored
    assert torch.equal(out[ends], (x[ends].float() * squares).to(BF16))
    kept = xs[torch.tensor(at, device="cuda")].clone()
    dy, dw = sort_combine_grad(dout, xs, s.place, w, dy=xs)
    for i, row in enumerate(at):
        t, j = row % tokens, row // tokens
        assert torch.equal(dy[row], dout[t] * (j + 1)), row
        terms = dout[t].double() * kept[i].double()
        assert abs(float(dw[t, j]) - float(terms.sum())) <= (n + 1) * R.U32 * float(terms.abs().sum()), row


def test_norm_gradient_far():
    """dr of a last row and of none beside it, and the sums over the rows, into arrays that held NaN."""
    from hoard_amd.ops import norm_forward
    m, n = 132000, 16384
    assert m * n > 2**31
    g = torch.Generator().manual_seed(2)
    last = torch.randn((2, n), generator=g).to(BF16).cuda()
    r = torch.ones((m, n), dtype=BF16, device="cuda")
    r[-1] = last[0]
    w = (1 + 0.1 * torch.randn(n, generator=g)).cuda()
    st = norm_forward(r, w_pre=w, eps=1e-6, want_stats=True)
    dh = torch.zeros((m, n), dtype=BF16, device="cuda")
    dh[-1] = last[1]
    dr, dw = torch.full((m, n), float("nan"), dtype=BF16, device="cuda"), torch.full((n,), float("nan"), device="cuda")
    a = H.NormArgs(H.TYPE_BF16, H.TYPE_BF16, H.GATE_NONE, 0, m, n, 1e-6, 1.0, 0.0, None, None, None, None, w.data_ptr(),
                   r.data_ptr(), None, st.stats.data_ptr())
    grads = H.NormGrads(None, dh.data_ptr(), dr.data_ptr(), None, None, None, dw.data_ptr())
    lib, need = H.load_library(), ctypes.c_size_t()
    H.check(lib.hoard_norm_workspace(ctypes.byref(a), ctypes.byref(need)))
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    H.check(lib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(grads), work.data_ptr(), need.value,
                                    torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    v, d, wd = last[0].cpu().to(D), last[1].cpu().to(D), w.cpu().to(D)
    rho = float(st.stats[-1, 1])
    u, part = d * wd, v * rho ** 2
    want = rho * (u - part * (u * v).mean())
    size = rho * (u.abs() + part.abs() * (u * v).abs().mean())
    R.close(dr[-1], want, R.stored(want, 56 * R.U32 * size, BF16), "dr")
    for row in (0, 1, m // 2, m - 2):
        assert (dr[row] == 0).all(), row
    assert not any(dr[i:i + 1000].isnan().any() for i in range(0, m, 1000))
    terms = d * v * rho
    R.close(dw, terms, 8 * R.U32 * terms.abs(), "dw_pre")  # the other rows add zeros, which round nothing

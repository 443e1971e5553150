"""The operators together, as a layer uses them: norm, the stage's router, the pairs sorted by expert, 4-bit expert
products, the rows taken back with the router's weights, and the norm after the block with gate and residual."""
import numpy as np
import pytest

import opsref as R
from hoard_amd import workloads as W

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

D = torch.float64
EPS = 1e-6


def weights(seed, n_mat, rows, cols, group):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n_mat, rows, cols // 2), generator=g, dtype=torch.uint8).cuda()
    return codes, (torch.rand((n_mat, rows, cols // group), generator=g) * 0.01).to(torch.float16).cuda(), None


@pytest.fixture(scope="module")
def layer():
    from hoard_amd.runtime import MoEStage
    shape = W.Shape("small", 90, 256, 12, 4, 256, 1, 12, 12, 12, 1)
    st = MoEStage(shape, n_layer=1, layers={0: W.make_layer(shape, 5, 0)})
    n, f, e = shape.n_embd, shape.n_ff, shape.n_expert
    mats = {"gate": weights(1, e, f, n, 64), "up": weights(2, e, f, n, 64), "down": weights(3, e, n, f, 128)}
    g = torch.Generator().manual_seed(4)
    par = {k: (1.0 + 0.1 * torch.randn(n, generator=g)).cuda() for k in ("first", "post", "next")}
    yield shape, st, mats, par
    st.close()


def run(layer, r, gate, one_token):
    from hoard_amd import ops
    shape, st, mats, par = layer
    q = {k: ops.Q4Weight(*m) for k, m in mats.items()}
    h = ops.norm_forward(r, w_pre=par["first"], eps=EPS).h
    picks = [st.route(0, t.cpu().numpy()) for t in h]
    ids = torch.from_numpy(np.stack([p[0] for p in picks])).cuda()
    w = torch.from_numpy(np.stack([p[1] for p in picks])).cuda()
    if one_token:  # no sort: every pair's row is at its own number
        place = torch.arange(ids.numel(), dtype=torch.int32, device="cuda").view(ids.shape)
        hid = ops.q4_matmul(h, q["gate"], q["up"], ids=ids)
        y = ops.q4_matmul(hid, q["down"], ids=ids.view(-1))
    else:
        s = ops.sort_pairs(ids, shape.n_expert)
        place = s.place
        xs = ops.sort_gather(h, place)
        hid = ops.q4_matmul(xs, q["gate"], q["up"], offsets=s.offsets)
        y = ops.q4_matmul(hid, q["down"], offsets=s.offsets)
    b = ops.sort_combine(y, place, w)
    st2 = ops.norm_forward(r, b, par["post"], gate, par["next"], eps=EPS, scale=0.5, gate_sigmoid=True, want_stats=True)
    return ids, w, place, y, b, st2


def plain(layer, r, gate, ids, w):
    shape, _, mats, par = layer
    p = {k: t.cpu().to(D) for k, t in par.items()}
    r = r.cpu().to(D)
    h = R.norm(r, EPS) * p["first"]
    ww = {k: R.dense(*m)[0] for k, m in mats.items()}
    b = torch.zeros_like(r)
    for t in range(r.shape[0]):
        for j, e in enumerate(ids[t].tolist()):
            g, u = ww["gate"][e] @ h[t], ww["up"][e] @ h[t]
            b[t] += float(w[t, j]) * (ww["down"][e] @ (g / (1 + torch.exp(-g)) * u))
    v = r + 0.5 * torch.sigmoid(gate.cpu().to(D)) * (R.norm(b, EPS) * p["post"])
    return b, v, R.norm(v, EPS) * p["next"]


@pytest.mark.parametrize("tokens,one", [(1, True), (1, False), (3, True), (16, False), (75, False)])
def test_layer(layer, tokens, one):
    g = torch.Generator().manual_seed(tokens)
    n = layer[0].n_embd
    r = torch.randn((tokens, n), generator=g).cuda()
    gate = torch.randn((tokens, 1), generator=g).cuda()
    ids, w, place, y, b, st = run(layer, r, gate, one)
    want_b, want_v, want_h = plain(layer, r, gate, ids, w)
    # three products of 256 terms, whose bound is (256 + 8) roundings of magnitudes some 40 times the sum's own size
    # (codes of up to 15 by up to 32 over sums of 256 random signs), each passing through the next: 3 * 264 * 40
    # roundings, and a fourth for the norms and the gate
    tol = 4 * 264 * 40 * R.U32
    for got, want in ((b, want_b), (st.r_out, want_v), (st.h, want_h)):
        rows = want.norm(dim=1, keepdim=True)
        assert ((got.cpu().to(D) - want).norm(dim=1, keepdim=True) <= tol * rows).all()


def test_forms_agree(layer):
    """The form for single tokens and the sorted one give each pair the same row, within their bounds."""
    r = torch.randn((9, layer[0].n_embd), generator=torch.Generator().manual_seed(9)).cuda()
    gate = torch.zeros((9, 1), device="cuda")
    a, b = run(layer, r, gate, True), run(layer, r, gate, False)
    assert torch.equal(a[0], b[0])
    ya, yb = a[3][a[2].reshape(-1).long()].double(), b[3][b[2].reshape(-1).long()].double()
    assert ((ya - yb).norm(dim=1) <= 2 * 264 * 40 * 3 * R.U32 * ya.norm(dim=1)).all()


def test_gradients_through_sort_and_norm(layer):
    """The gradient of the combine, the norm and the gather chained, against a 64-bit difference along a direction."""
    from hoard_amd import ops
    shape = layer[0]
    m, k, n = 20, 4, shape.n_embd
    g = torch.Generator().manual_seed(77)
    rand = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
    ids = torch.stack([torch.randperm(shape.n_expert, generator=g)[:k] for _ in range(m)]).to(torch.int32).cuda()
    s = ops.sort_pairs(ids, shape.n_expert)
    x, w, r, wp, wq = rand(m, n), rand(m, k), rand(m, n), rand(n), rand(n)
    e = torch.bucketize(torch.arange(m * k, device="cuda"), s.offsets[1:], right=True)
    scale = rand(shape.n_expert)[e].unsqueeze(1)  # the experts: each scales its rows
    xs = ops.sort_gather(x, s.place)
    y = xs * scale
    b = ops.sort_combine(y, s.place, w)
    st = ops.norm_forward(r, b, wp, None, wq, eps=EPS, want_stats=True)
    dr, dh = rand(m, n), rand(m, n)
    grads = ops.norm_backward(st, dr, dh, b, wp, None, wq, eps=EPS)
    dy, dw = ops.sort_combine_grad(grads.db, y, s.place, w)
    dx = ops.sort_combine(dy * scale, s.place)
    t64 = lambda t: t.cpu().to(D)  # noqa: E731
    place, sc = t64(s.place).long().view(-1), t64(scale)
    dir_x, dir_w = torch.randn(m, n, generator=g, dtype=D), torch.randn(m, k, generator=g, dtype=D)

    def loss(t):
        rows = torch.empty(m * k, n, dtype=D)
        rows[place] = (t64(x) + t * dir_x).repeat_interleave(k, 0)
        y = rows * sc
        b = (y[place].view(m, k, n) * (t64(w) + t * dir_w).unsqueeze(2)).sum(1)
        v = t64(r) + R.norm(b, EPS) * t64(wp)
        return (v * t64(dr)).sum() + (R.norm(v, EPS) * t64(wq) * t64(dh)).sum()

    diff = float(loss(1e-5) - loss(-1e-5)) / 2e-5
    tx, tw = t64(dx) * dir_x, t64(dw) * dir_w
    want, mag = float(tx.sum() + tw.sum()), float(tx.abs().sum() + tw.abs().sum())
    # some 300 roundings of magnitudes up to 10 times the gradients', and the step's square
    assert abs(diff - want) <= (3000 * R.U32 + 1e-6) * mag

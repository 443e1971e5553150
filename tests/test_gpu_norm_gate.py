"""The gradient of a gate behind a sigmoid keeps its digits where the sigmoid is close to 1 or to 0."""
import pytest

import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

D = torch.float64


@pytest.mark.parametrize("kind", ["channel", "token", "full"])
@pytest.mark.parametrize("n", [600, 2047, 9001])
def test_far_gates(kind, n):
    from hoard_amd.ops import norm_backward, norm_forward
    m = 3 if kind == "full" else 1 if kind == "channel" else 61
    g = torch.Generator().manual_seed(n)
    r, b, dr = (torch.randn((m, n), generator=g) for _ in range(3))
    size = {"channel": (n,), "token": (m, 1), "full": (m, n)}[kind]
    gate = torch.linspace(-60.0, 60.0, n if kind == "channel" else m * n if kind == "full" else m).view(size)
    st = norm_forward(r.cuda(), b.cuda(), gate=gate.cuda(), eps=1e-6, gate_sigmoid=True, want_stats=True)
    got = norm_backward(st, dr.cuda(), None, b.cuda(), gate=gate.cuda(), eps=1e-6, gate_sigmoid=True)
    q = gate.to(D)
    slope = torch.exp(-q.abs()) / (1 + torch.exp(-q.abs())) ** 2
    terms = dr.to(D) * b.to(D) * slope
    # a term: its factors 4, e^-x by 2 (1.5 steps of 32 bits), a sum, a quotient by 2, two products; a row's sum 40
    steps, want, mag = 14, terms, terms.abs()
    if kind == "channel":
        want, mag = terms.sum(0), terms.abs().sum(0)
    if kind == "token":
        steps, want, mag = 14 + 44, terms.sum(1, keepdim=True), terms.abs().sum(1, keepdim=True)
    R.close(got.dgate, want, steps * R.U32 * mag + 2.0 ** -149, "dgate")
    db = torch.sigmoid(q) * dr.to(D)
    R.close(got.db, db.expand(m, n), 14 * R.U32 * db.abs().expand(m, n) + 2.0 ** -149, "db")

"""The norms around a block and their gradients against 64-bit forms, within bounds that count roundings.

A row's sums are formed by threads of at most 16 values each, then over the 64 lanes in 6 steps and over at most 16
waves: a value passes at most 16 + 6 + 16 additions, so a sum is off by 40 roundings of its terms' magnitudes, two
more for each term's own factors; rho = 1 / sqrt(mean + eps) halves that and adds a product, a sum, a root and a quotient.
"""
import pytest

import hoard_amd as H
import opsref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
D = torch.float64
U = R.U32
EPS = 1e-6


def rand(seed, *size, dtype=F32, off=0, std=1.0, mean=0.0):
    t = (torch.randn(size, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype)
    buf = torch.empty(t.numel() + off, dtype=dtype, device="cuda")
    buf[off:] = t.reshape(-1).cuda()
    return buf[off:].view(*size)


def c64(t):
    return None if t is None else t.detach().cpu().to(D)


class Case:
    def __init__(self, m, n, dtype, res, gate="none", sigmoid=False, post=True, pre=True, block=True, scale=1.0, offset=0.0,
                 off=0, zero_row=False):
        self.m, self.n, self.kind, self.pre = m, n, gate, pre
        self.r = rand(1, m, n, dtype=res, off=off)
        self.kw = dict(eps=EPS, scale=scale, w_offset=offset, gate_sigmoid=sigmoid)
        self.dtype, self.res = dtype, res
        self.par = {}
        if block:
            b = rand(2, m, n, dtype=dtype, off=off, std=0.5)
            if zero_row:
                b[m // 2] = 0
                self.r[m // 3] = 0
            self.par["b"] = b
            if post:
                self.par["w_post"] = rand(3, n, off=off, std=0.1, mean=1.0 - offset)
            if gate != "none":
                self.par["gate"] = {"channel": lambda: rand(4, n, off=off), "token": lambda: rand(4, m, 1, off=off),
                                    "full": lambda: rand(4, m, n, dtype=dtype, off=off)}[gate]()
        if pre:
            self.par["w_pre"] = rand(5, n, off=off, std=0.1, mean=1.0 - offset)

    def forward(self, **kw):
        from hoard_amd.ops import norm_forward
        return norm_forward(self.r, **self.par, dtype=self.dtype, want_stats=True, **self.kw, **kw)

    def p64(self):
        return {k: c64(t) for k, t in self.par.items()}


def gate64(case, gate):
    if gate is None:
        return 1.0
    return torch.sigmoid(gate) if case.kw["gate_sigmoid"] else gate


CASES = [
    dict(m=1, n=1, dtype=F32, res=F32), dict(m=1, n=2048, dtype=F32, res=F32, gate="token", sigmoid=True),
    dict(m=3, n=7, dtype=BF16, res=F32, gate="channel", off=1), dict(m=5, n=64, dtype=F16, res=F16, gate="full", scale=0.3),
    dict(m=2, n=512, dtype=BF16, res=BF16, offset=1.0), dict(m=4, n=513, dtype=F16, res=F32, gate="full", sigmoid=True),
    dict(m=7, n=1000, dtype=F32, res=F32, gate="channel", sigmoid=True, scale=-0.5, off=1),
    dict(m=3, n=1025, dtype=BF16, res=F32, gate="token"), dict(m=9, n=2048, dtype=BF16, res=BF16, gate="channel", offset=1.0),
    dict(m=6, n=2049, dtype=F16, res=F16, gate="token", sigmoid=True), dict(m=5, n=4095, dtype=BF16, res=F32, gate="channel", scale=0.22, off=3),
    dict(m=3, n=4097, dtype=F32, res=F32, gate="full", sigmoid=True), dict(m=2, n=8192, dtype=BF16, res=BF16, gate="full"),
    dict(m=3, n=8193, dtype=F16, res=F32, gate="channel"), dict(m=2, n=16383, dtype=F32, res=F32, gate="token", off=1),
    dict(m=2, n=16384, dtype=BF16, res=F32, gate="full", sigmoid=True, offset=1.0),
    dict(m=700, n=96, dtype=BF16, res=F32, gate="channel"), dict(m=1500, n=40, dtype=F32, res=F32, gate="token"),
    # parts of it: a plain norm, a plain addition, an addition and a norm, a norm of the block's output alone
    dict(m=4, n=300, dtype=BF16, res=F32, block=False), dict(m=4, n=300, dtype=F32, res=F32, block=False, offset=1.0),
    dict(m=4, n=300, dtype=BF16, res=BF16, post=False, pre=False), dict(m=4, n=300, dtype=F16, res=F16, post=False, gate="token"),
    dict(m=4, n=300, dtype=BF16, res=F32, pre=False, gate="channel", sigmoid=True), dict(m=4, n=2048, dtype=F32, res=F32, post=False),
    # one row, whose sums over the rows need none
    dict(m=1, n=1500, dtype=F32, res=F32, gate="channel"), dict(m=1, n=9001, dtype=BF16, res=F32, gate="channel", sigmoid=True),
    # more rows than groups
    dict(m=3000, n=24, dtype=F32, res=F32, gate="channel"), dict(m=1600, n=1100, dtype=BF16, res=BF16, gate="channel"),
    # rows of zeros
    dict(m=6, n=320, dtype=BF16, res=F32, gate="channel", zero_row=True),
]
IDS = ["-".join(str(v).replace("torch.", "") for v in c.values()) for c in CASES]


def forward64(case):
    """(value of r_out before storing, its bound, rho_b, relative bound of a rho)."""
    p = case.p64()
    v, bound, rho_b = c64(case.r), torch.zeros(case.m, case.n, dtype=D), torch.ones(case.m, dtype=D)
    rel_rho = 28 * U
    if "b" in p:
        c = p["b"]
        if "w_post" in p:
            rho_b = 1.0 / torch.sqrt((c * c).mean(1) + EPS)
            c = c * rho_b.unsqueeze(1) * (case.kw["w_offset"] + p["w_post"])
        add = case.kw["scale"] * gate64(case, p.get("gate")) * c
        # rho, four products, the weight's sum, a sigmoid of up to 8 (e^-x by 2, a sum, a quotient, with room)
        mag = add.abs()
        if "w_post" in p:
            mag = mag + (case.kw["scale"] * gate64(case, p.get("gate")) * p["b"] * rho_b.unsqueeze(1)).abs() * abs(case.kw["w_offset"])
        bound = mag * (rel_rho + 16 * U) + (v + add).abs() * U
        v = v + add
    return v, bound, rho_b, rel_rho


@pytest.mark.parametrize("kw", CASES, ids=IDS)
def test_forward(kw):
    print("norm", kw, flush=True)
    case = Case(**kw)
    st = case.forward()
    v, bound, rho_b, rel = forward64(case)
    if "b" in case.par:
        R.close(st.r_out, v, R.stored(v, bound, case.res), "r_out")
    else:
        assert st.r_out is case.r
    R.close(st.stats[:, 0], rho_b, rho_b * rel, "rho_b")
    if not case.pre:
        assert st.h is None and (st.stats[:, 1] == 1).all()
        return
    v = c64(st.r_out)  # of the stream as stored
    rho = 1.0 / torch.sqrt((v * v).mean(1) + EPS)
    R.close(st.stats[:, 1], rho, rho * rel, "rho_v")
    w = c64(case.par["w_pre"])
    h = v * rho.unsqueeze(1) * (case.kw["w_offset"] + w)
    mag = (v * rho.unsqueeze(1)).abs() * (abs(case.kw["w_offset"]) + w.abs())
    R.close(st.h, h, R.stored(h, mag * (rel + 4 * U), case.dtype), "h")


def backward64(case, v, stats, dr_out, dh):
    """The formulas, and the same with every term's magnitude."""
    p, o = case.p64(), case.kw["w_offset"]
    n = case.n
    rho_b, rho_v = stats[:, :1], stats[:, 1:]
    out, mag = {}, {}
    zero = torch.zeros(case.m, n, dtype=D)
    dv = dr_out if dr_out is not None else zero
    m_dv = dv.abs()
    if dh is not None:
        u, m_u = dh * (o + p["w_pre"]), dh.abs() * (abs(o) + p["w_pre"].abs())
        dv = dv + rho_v * (u - v * rho_v ** 2 * (u * v).mean(1, keepdim=True))
        m_dv = m_dv + rho_v * (m_u + v.abs() * rho_v ** 2 * (m_u * v.abs()).mean(1, keepdim=True))
        out["dw_pre"], mag["dw_pre"] = (dh * v * rho_v).sum(0), (dh * v * rho_v).abs().sum(0)
    out["dr"], mag["dr"] = dv, m_dv
    if "b" not in p:
        return out, mag
    g = gate64(case, p.get("gate"))
    g = g if torch.is_tensor(g) else torch.ones(1, 1, dtype=D)
    slope = g * (1 - g) if case.kw["gate_sigmoid"] else torch.ones_like(g)
    wp = o + p["w_post"] if "w_post" in p else torch.ones(n, dtype=D)
    m_wp = abs(o) + p["w_post"].abs() if "w_post" in p else wp
    s, b = case.kw["scale"], p["b"]
    d, m_d = s * dv, abs(s) * m_dv
    if "gate" in p:
        # a sigmoid close to 1 leaves 1 - g with the rounding of 1
        m_slope = g if case.kw["gate_sigmoid"] else slope
        dg, m_dg = d * b * rho_b * wp * slope, m_d * (b * rho_b).abs() * m_wp * m_slope
        if case.kind == "channel":
            dg, m_dg = dg.sum(0), m_dg.sum(0)
        if case.kind == "token":
            dg, m_dg = dg.sum(1, keepdim=True), m_dg.sum(1, keepdim=True)
        out["dgate"], mag["dgate"] = dg, m_dg
    dc, m_dc = d * g, m_d * g.abs()
    if "w_post" in p:
        out["dw_post"], mag["dw_post"] = (dc * b * rho_b).sum(0), (m_dc * (b * rho_b).abs()).sum(0)
        u2, m_u2 = dc * wp, m_dc * m_wp
        dc = rho_b * (u2 - b * rho_b ** 2 * (u2 * b).mean(1, keepdim=True))
        m_dc = rho_b * (m_u2 + b.abs() * rho_b ** 2 * (m_u2 * b.abs()).mean(1, keepdim=True))
    out["db"], mag["db"] = dc, m_dc
    return out, mag


def grad_bounds(case, out, mag):
    # dv: a row's sum (42 roundings, three factors more) and six of its own; db: that, another row's sum, a gate of 8
    # roundings and eight products; sums over the rows: those of a term and one for each row
    steps = {"dr": 56, "dw_pre": 8 + case.m, "dgate": 80 + (case.m if case.kind == "channel" else 44), "dw_post": 80 + case.m,
             "db": 136}
    kind = {"dr": case.res, "db": case.dtype, "dgate": case.dtype if case.kind == "full" else F32}
    return {k: R.stored(out[k], steps[k] * U * mag[k], kind.get(k, F32)) for k in out}


@pytest.mark.parametrize("given", ["both", "dr_out", "dh"])
@pytest.mark.parametrize("kw", CASES, ids=IDS)
def test_backward(kw, given):
    from hoard_amd.ops import norm_backward
    print("norm grad", kw, given, flush=True)
    case = Case(**kw)
    if given == "dh" and not case.pre:
        return
    st = case.forward()
    off = kw.get("off", 0)
    dr_out = rand(6, case.m, case.n, dtype=case.res, off=off) if given != "dh" else None
    dh = rand(7, case.m, case.n, dtype=case.dtype, off=off) if case.pre and given != "dr_out" else None
    if "b" not in case.par and dh is None and case.dtype != case.res:
        return  # nothing of that type takes part
    got = norm_backward(st, dr_out, dh, **case.par, **case.kw)
    out, mag = backward64(case, c64(st.r_out), c64(st.stats), c64(dr_out), c64(dh))
    bounds = grad_bounds(case, out, mag)
    for name, t in got._asdict().items():
        assert (t is not None) == (name in out), name
        if t is not None:
            R.close(t, out[name], bounds[name], name)


@pytest.mark.parametrize("given", ["both", "dr_out", "dh"])
@pytest.mark.parametrize("kw", [dict(m=600, n=8200, dtype=BF16, res=F32, gate="channel", sigmoid=True),
                                dict(m=520, n=9003, dtype=F32, res=F32, gate="channel"),
                                dict(m=300, n=16384, dtype=F16, res=F16, gate="token", offset=1.0)], ids=str)
def test_backward_long_rows(kw, given):
    """The longest rows, several of them a group."""
    test_backward(kw, given)


@pytest.mark.parametrize("kw", [c for c in CASES if c["dtype"] == F32], ids=[i for i, c in zip(IDS, CASES) if c["dtype"] == F32])
def test_backward_against_differences(kw):
    """Along a random direction: the gradients' inner product against a central difference of the 64-bit forward."""
    from hoard_amd.ops import norm_backward
    case = Case(**kw)
    st = case.forward()
    dr_out = rand(6, case.m, case.n) if "b" in case.par else None
    dh = rand(7, case.m, case.n) if case.pre else None
    got = norm_backward(st, dr_out, dh, **case.par, **case.kw)
    p, o = dict(case.p64(), r=c64(case.r)), case.kw["w_offset"]
    dirs = {k: torch.randn(t.shape, generator=torch.Generator().manual_seed(50 + i), dtype=D) for i, (k, t) in enumerate(p.items())}

    def loss(t):
        q = {k: x + t * dirs[k] for k, x in p.items()}
        v = q["r"]
        if "b" in q:
            c = R.norm(q["b"], EPS) * (o + q["w_post"]) if "w_post" in q else q["b"]
            v = v + case.kw["scale"] * gate64(case, q.get("gate")) * c
        s = (v * c64(dr_out)).sum() if dr_out is not None else 0.0
        return s + ((R.norm(v, EPS) * (o + q["w_pre"]) * c64(dh)).sum() if dh is not None else 0.0)

    step = 1e-5 if case.n > 1 else 1e-7  # one column's norm is a sign: nearly a step where x is small
    diff = (loss(step) - loss(-step)) / (2 * step)
    names = {"r": "dr", **{k: "d" + k for k in case.par}}
    terms = [(c64(getattr(got, names[k])) * dirs[k]) for k in p]
    want, mag = sum(float(t.sum()) for t in terms), sum(float(t.abs().sum()) for t in terms)
    # a gradient is off by at most (200 + rows) roundings of its terms' magnitudes (above), which exceed the gradients'
    # by what cancels in a norm's, at most a factor of about n^0.5 for random values; the difference itself by step^2
    assert abs(float(diff) - want) <= (200 + case.m) * U * mag * 10 + 1e-6 * mag


def test_in_place():
    from hoard_amd.ops import norm_forward
    for n in (100, 2048, 9000):
        case = Case(m=5, n=n, dtype=BF16, res=F32, gate="channel")
        want = case.forward()
        r = case.r.clone()
        got = norm_forward(r, **case.par, **case.kw, r_out=r)
        assert got.r_out is r and torch.equal(r, want.r_out) and torch.equal(got.h, want.h)


def test_gradient_in_place():
    """dr over dr_out, through the C ABI."""
    import ctypes
    from hoard_amd import ops
    for n in (100, 2048, 9000):
        case = Case(m=6, n=n, dtype=F32, res=F32, gate="token")
        st = case.forward()
        dr_out, dh = rand(6, 6, n), rand(7, 6, n)
        want = ops.norm_backward(st, dr_out, dh, **case.par, **case.kw)
        p = {k: t.data_ptr() for k, t in case.par.items()}
        a = H.NormArgs(H.TYPE_F32, H.TYPE_F32, H.GATE_TOKEN, 0, 6, n, EPS, 1.0, 0.0, None, p["b"], p["gate"], p["w_post"],
                       p["w_pre"], st.r_out.data_ptr(), None, st.stats.data_ptr())
        g = H.NormGrads(dr_out.data_ptr(), dh.data_ptr(), dr_out.data_ptr())
        work = torch.empty(3 * 6 * n, device="cuda")
        lib = H.load_library()
        H.check(lib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(g), work.data_ptr(), work.numel() * 4,
                                        torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert torch.equal(dr_out, want.dr)


def test_no_rows():
    """No rows: nothing to write but the sums over them."""
    from hoard_amd.ops import norm_backward, norm_forward
    r, b, w = (torch.empty((0, 50), device="cuda") for _ in range(3))
    wp, wq, gate = rand(1, 50), rand(2, 50), rand(3, 50)
    st = norm_forward(r, b, wp, gate, wq, eps=EPS, want_stats=True)
    assert st.r_out.shape == (0, 50)
    got = norm_backward(st, r, w, b, wp, gate, wq, eps=EPS)
    for t in (got.dw_post, got.dw_pre, got.dgate):
        assert (t == 0).all()


def test_bad_rows_stay_apart():
    """A row with a NaN or an infinity spoils no other row."""
    case = Case(m=8, n=700, dtype=BF16, res=F32, gate="full")
    want = case.forward()
    case.par["b"][2, 5], case.r[4, 600] = float("nan"), float("inf")
    got = case.forward()
    rest = [0, 1, 3, 5, 6, 7]
    for a, b in ((got.r_out, want.r_out), (got.h, want.h), (got.stats, want.stats)):
        assert torch.equal(a[rest], b[rest])
    assert got.h[2].isnan().all() and got.h[4].isnan().any()


def test_streams_and_graph():
    from hoard_amd.ops import norm_backward
    cases = [Case(m=600, n=256, dtype=BF16, res=F32, gate="channel", scale=s) for s in (1.0, 0.5)]
    dr, dh = rand(6, 600, 256), rand(7, 600, 256, dtype=BF16)

    def chain(case):
        st = case.forward()
        return [st.r_out, st.h, st.stats, *norm_backward(st, dr, dh, **case.par, **case.kw)]

    want = [[t.clone() for t in chain(c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append([chain(c) for _ in range(3)])
    torch.cuda.synchronize()
    for g, e in zip(got, want):
        for once in g:
            assert all(torch.equal(a, b) for a, b in zip(once, e))
    graphs = []
    for c, s in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = chain(c)
        graphs.append((g, outs))
    for r in range(4):
        for (g, outs), e in zip(graphs, want):
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, e)), r
        chain(cases[r % 2])
        torch.empty(1 << 16, device="cuda").normal_().sum().item()


def test_python_refusals():
    from hoard_amd.ops import norm_backward, norm_forward
    r, b, w = rand(1, 4, 32), rand(2, 4, 32), rand(3, 32)
    st = norm_forward(r, b, w, w_pre=w, eps=EPS, want_stats=True)
    for call in (lambda: norm_forward(r.cpu(), w_pre=w, eps=EPS), lambda: norm_forward(r, eps=EPS), lambda: norm_forward(r, w_pre=w, eps=0.0),
                 lambda: norm_forward(r, b[:3], eps=EPS), lambda: norm_forward(r, b, w[:8], eps=EPS), lambda: norm_forward(r, w_post=w, w_pre=w, eps=EPS),
                 lambda: norm_forward(r, gate=w, w_pre=w, eps=EPS), lambda: norm_forward(r, b, gate=w[:4], eps=EPS),
                 lambda: norm_forward(r.half(), b, eps=EPS), lambda: norm_forward(r, b, w.half(), eps=EPS),
                 lambda: norm_forward(r.t(), w_pre=w, eps=EPS), lambda: norm_forward(r, w_pre=w, eps=EPS, r_out=b),
                 lambda: norm_backward(st, b=b, w_post=w, w_pre=w, eps=EPS), lambda: norm_backward(st._replace(stats=None), r, b=b, eps=EPS),
                 lambda: norm_backward(st, r[:2], b=b, w_post=w, eps=EPS)):
        with pytest.raises(H.HoardError):
            call()

"""A layer's attention half together, as a decode loop and a verify step use it: the 4-bit projection to queries, keys and
values, heads normed and rotated into the cache, attention over it, the output projection, the norm that adds the residual
and the stage after it."""
import pytest

import attnref as A
import opsref as R
from hoard_amd import workloads as W

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

D = torch.float64
EPS = 1e-6
HQ, HKV, DIM, N = 8, 2, 64, 256


def gen(seed):
    return torch.Generator().manual_seed(seed)


def q4(seed, rows, cols):
    from hoard_amd import ops
    codes = torch.randint(0, 256, (rows, cols // 2), generator=gen(seed), dtype=torch.uint8).cuda()
    return ops.Q4Weight(codes, (torch.rand((rows, cols // 64), generator=gen(seed + 1)) * 0.02).cuda())


class Layer:
    """Weights of one layer and its plain 64-bit form over whole sequences."""

    def __init__(self, rot=32, pairs=False):
        from hoard_amd import attn
        self.qkv, self.out = q4(1, (HQ + 2 * HKV) * DIM, N), q4(3, N, HQ * DIM)
        self.w_q, self.w_k = (1 + 0.2 * torch.randn(DIM, generator=gen(s)) for s in (5, 6))
        self.first, self.next = (1 + 0.1 * torch.randn(N, generator=gen(s)) for s in (7, 8))
        self.freq, self.pairs = attn.rope_freq(rot, 10000.0), pairs
        self.dev = {k: getattr(self, k).cuda() for k in ("w_q", "w_k", "first", "next")}

    def step(self, x, pos, cache, slots, pages, lens):
        """(residual after the attention, the next block's input, attention's rows) of the new tokens' rows x."""
        from hoard_amd import attn, ops
        h = ops.norm_forward(x, w_pre=self.dev["first"], eps=EPS).h
        q, k, v = attn.split_heads(ops.q4_matmul(h, self.qkv), HQ, HKV, DIM)
        st = attn.heads_forward(q, k, v, w_q=self.dev["w_q"], w_k=self.dev["w_k"], cache=cache, slots=slots, eps=EPS,
                                rope=attn.Rope(pos, self.freq, pairs=self.pairs), q_out=q)
        o = attn.attn_decode(st.q_out, cache, pages, lens).out
        b = ops.q4_matmul(o.view(len(x), HQ * DIM), self.out)
        n = ops.norm_forward(x, b, w_pre=self.dev["next"], eps=EPS)
        return n.r_out, n.h, o

    def plain(self, x, held):
        """The same of a whole sequence x [tokens, N] in 64 bits; held: what the cache does to a row."""
        x = x.cpu().to(D)
        w, wo = (R.dense(m.codes, m.scales, None)[0] for m in (self.qkv, self.out))
        h = R.norm(x, EPS) * self.first.to(D)
        qkv = (h @ w.t()).view(len(x), -1, DIM)
        pos = torch.arange(len(x))
        rope = (pos, self.freq.cpu(), None, self.pairs)
        q = A.heads(qkv[:, :HQ], self.w_q, rope, EPS, 0.0)[0]
        k = held(A.heads(qkv[:, HQ:HQ + HKV], self.w_k, rope, EPS, 0.0)[0])
        v = held(qkv[:, HQ + HKV:])
        k, v = (t.repeat_interleave(HQ // HKV, dim=1).transpose(0, 1) for t in (k, v))
        s = (q.transpose(0, 1) @ k.transpose(1, 2)) * DIM ** -0.5
        s = s.masked_fill(torch.ones(len(x), len(x)).triu(1).bool(), float("-inf"))
        o = (torch.softmax(s, 2) @ v).transpose(0, 1)
        r = x + o.reshape(len(x), HQ * DIM) @ wo.t()
        return r, R.norm(r, EPS) * self.next.to(D), o


@pytest.fixture(scope="module")
def layer():
    return Layer()


def i8(x):
    step = x.abs().amax(-1, keepdim=True) / 127.0
    return torch.round(x / step) * step


@pytest.mark.parametrize("ct,held,tol", [
    # three products of 256 to 512 columns in 32 bits, whose bounds are some 300 roundings of sums 40 times the result's
    # size, and one rounding of keys and values to the cache's type, which the scores (of order 8) carry on
    (torch.float16, lambda x: x.to(torch.float32).to(torch.float16).to(D), 1e-3 + 2 * 8 * 2.0 ** -11),
    # codes that differ where a value lies next to a border: one of 127 steps of the largest value for a few of the values
    (torch.int8, i8, 1e-3 + 8 * 2.0 / 127)])
def test_prompt_then_decode_then_verify(layer, ct, held, tol):
    """Two sequences: prompts written at once, tokens one by one, then a verify step of 3 and 4 drafts."""
    from hoard_amd import attn
    page = 16
    cache = attn.KVCache.new(12, page, HKV, DIM, ct)
    pages = torch.tensor([[3, 7, 0, 11], [5, 1, 9, 2]], dtype=torch.int32)
    total = [45, 26]
    xs = [0.5 * torch.randn((t, N), generator=gen(20 + i)) for i, t in enumerate(total)]
    want = [layer.plain(x, held) for x in xs]
    slot = lambda s, t: int(pages[s, t // page]) * page + t % page  # noqa: E731
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def run(rows, lens):
        """rows: (sequence, position) of each new token, or None; lens as attn_decode's."""
        x = torch.stack([xs[r[0]][r[1]] if r else torch.zeros(N) for r in rows]).cuda()
        got = layer.step(x, dev([r[1] if r else 0 for r in rows]), cache, dev([slot(*r) if r else -1 for r in rows]), pages.cuda(), lens)
        for i, r in enumerate(rows):
            if r is None:
                assert not got[2][i].any()
                continue
            for g, w in zip(got, want[r[0]]):
                g, w = g[i].cpu().to(D), w[r[1]]
                assert (g - w).norm() <= tol * w.norm(), (r, float((g - w).norm() / w.norm()))

    # the prompts: 9 and 5 tokens, each seeing those before it
    rows = [(0, t) for t in range(9)] + [(1, t) if t < 5 else None for t in range(9)]
    run(rows, dev([[t + 1 for t in range(9)], [t + 1 if t < 5 else 0 for t in range(9)]]))
    for i in range(18):
        run([(0, 9 + i), (1, 5 + i)], dev([10 + i, 6 + i]))
    # drafts: 4 and 3 tokens, the last row of the second padded
    for i in range(0, 18, 4):
        a, b = 27 + i, 23
        second = [(1, b + j) if i == 0 and j < 3 else None for j in range(4)]
        run([(0, a + j) if a + j < total[0] else None for j in range(4)] + second,
            dev([[a + j + 1 if a + j < total[0] else 0 for j in range(4)], [b + j + 1 if i == 0 and j < 3 else 0 for j in range(4)]]))


def test_decode_in_a_graph(layer):
    """A captured decode step, replayed token by token, equals the eager one."""
    from hoard_amd import attn
    x = 0.5 * torch.randn((12, N), generator=gen(40)).cuda()
    pages = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")

    def state():
        return attn.KVCache.new(2, 16, HKV, DIM, torch.int8), *(torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(3))

    def put(t, pos, slots, lens):
        pos.fill_(t)
        slots.fill_((16 if t < 16 else 0) + t % 16)
        lens.fill_(t + 1)

    cache, pos, slots, lens = state()
    want = []
    for t in range(12):
        put(t, pos, slots, lens)
        want.append([r.clone() for r in layer.step(x[t:t + 1], pos, cache, slots, pages, lens)])
    cache, pos, slots, lens = state()
    now = x[:1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.step(now, pos, cache, slots, pages, lens)
    for t in range(12):
        put(t, pos, slots, lens)
        now.copy_(x[t:t + 1])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want[t]):
            assert torch.equal(a, b), t


def test_before_the_stage():
    """The stage takes the attention half's rows: hoard_moe_layer's fx and residual."""
    from hoard_amd import attn, ops
    from hoard_amd.runtime import MoEStage
    shape = W.Shape("small", 90, 256, 12, 4, 256, 1, 12, 12, 12, 1)
    st = MoEStage(shape, n_layer=1, layers={0: W.make_layer(shape, 5, 0)})
    layer = Layer(rot=64, pairs=True)
    cache = attn.KVCache.new(2, 16, HKV, DIM, torch.float16)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x = 0.5 * torch.randn((1, N), generator=gen(50)).cuda()
    r, h, _ = layer.step(x, dev([0]), cache, dev([16]), dev([[1]]), dev([1]))
    out = st.layer(0, h[0].cpu().numpy(), r[0].cpu().numpy())
    out = out[0] if isinstance(out, tuple) else out
    assert out.shape == (N,) and bool((out == out).all())
    assert ops.norm_forward(r, w_pre=layer.dev["next"], eps=EPS).h.equal(h)
    st.close()

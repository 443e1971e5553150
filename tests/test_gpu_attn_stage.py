"""A layer's attention half over the codes that its 8-bit cache holds, and the stage behind it against the oracle."""
import numpy as np
import pytest

import attnref as A
import opsref as R
import parity
from hoard_amd import workloads as W
from test_gpu_attn_layer import D, DIM, EPS, HKV, HQ, N, Layer, gen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def dev(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rot,pairs", [(32, False), (64, True)])
def test_over_the_codes_held(rot, pairs):
    """Prompts, then tokens one by one, then drafts of two sequences; the 64-bit form attends to the codes that the cache
    holds, each within half a step of the 64-bit key or value.

    Three products of 256 to 512 columns in 32 bits are some 300 roundings of sums 40 times the result's size: 7e-4."""
    from hoard_amd import attn
    layer, page, tol = Layer(rot, pairs), 16, 1e-3
    cache = attn.KVCache.new(12, page, HKV, DIM, torch.int8)
    pages = torch.tensor([[3, 7, 0, 11], [5, 1, 9, 2]], dtype=torch.int32)
    total = [47, 33]
    xs = [0.5 * torch.randn((t, N), generator=gen(20 + i)) for i, t in enumerate(total)]
    slot = lambda s, t: int(pages[s, t // page]) * page + t % page  # noqa: E731
    got = [[None] * t for t in total]

    def run(first, new):
        """new[s] tokens of each sequence from first[s] on."""
        n = max(new)
        rows = [(s, first[s] + j) if j < new[s] else None for s in range(2) for j in range(n)]
        x = torch.stack([xs[r[0]][r[1]] if r else torch.zeros(N) for r in rows]).cuda()
        out = layer.step(x, dev([r[1] if r else 0 for r in rows]), cache, dev([slot(*r) if r else -1 for r in rows]),
                         pages.cuda(), dev([r[1] + 1 if r else 0 for r in rows]).view(2, n))
        for i, r in enumerate(rows):
            if r:
                got[r[0]][r[1]] = [t[i].cpu().to(D) for t in out]

    run([0, 0], [21, 7])
    for i in range(22):
        run([21 + i, 7 + i], [1, 1])
    run([43, 29], [4, 4])
    for s, t in enumerate(total):
        slots = dev([slot(s, i) for i in range(t)])
        read = [A.t64(r) for r in attn.kv_read(cache, slots, torch.float32)]
        steps = [A.t64(c[slots.long() // page, :, slots.long() % page]).unsqueeze(-1) for c in (cache.k_scale, cache.v_scale)]
        order = iter(zip(read, steps))

        def held(x):
            values, step = next(order)
            # half a step, and the product's roundings of a value of up to 127 of them
            assert ((values - x).abs() <= (0.5 + 127 * tol) * step).all() and ((values - x).abs() <= 0.51 * step).double().mean() > 0.99
            return values

        want = layer.plain(xs[s], held)
        for i in range(t):
            for name, g, w in zip(("r", "h", "attention"), got[s][i], want):
                assert (g - w[i]).norm() <= tol * w[i].norm(), (s, i, name, float((g - w[i]).norm() / w[i].norm()))
        # with a key less the attention's rows are further off
        less = attended(layer, xs[s], *read, 1)[1:]
        assert ((less - want[2][1:]).flatten(1).norm(dim=1) > 3 * tol * want[2][1:].flatten(1).norm(dim=1)).double().mean() > 0.9
        same = attended(layer, xs[s], *read, 0)
        assert (same - want[2]).norm() <= 1e-12 * same.norm()


def attended(layer, x, k, v, less):
    """The attention of x's rows over keys and values [tokens, HKV, DIM], each row's last `less` left out."""
    h = R.norm(x.to(D), EPS) * layer.first.to(D)
    q = (h @ R.dense(layer.qkv.codes, layer.qkv.scales, None)[0].t()).view(len(x), -1, DIM)[:, :HQ]
    q = A.heads(q, layer.w_q, (torch.arange(len(x)), layer.freq.cpu(), None, layer.pairs), EPS, 0.0)[0].transpose(0, 1)
    k, v = (t.repeat_interleave(HQ // HKV, dim=1).transpose(0, 1) for t in (k, v))
    s = (q @ k.transpose(1, 2)) * DIM ** -0.5
    s = s.masked_fill(torch.ones(len(x), len(x)).triu(1 - less).bool(), float("-inf"))
    return (torch.softmax(s, 2) @ v).transpose(0, 1)


def test_the_stage_behind_it(orc):
    """Rows of three sequences go on to the stage: its output is the oracle's for those rows, and no other's."""
    from hoard_amd import attn
    from hoard_amd.runtime import MoEStage
    shape = W.Shape("small", 90, 256, 12, 4, 256, 1, 12, 12, 12, 1)
    hl = W.make_layer(shape, 5, 0)
    st = MoEStage(shape, n_layer=1, layers={0: hl})
    try:
        layer = Layer(rot=64, pairs=True)
        cache = attn.KVCache.new(3, 16, HKV, DIM, torch.float16)
        x = 0.5 * torch.randn((3, N), generator=gen(50))
        pages, r, h = dev([[1], [2], [0]]), None, None
        r, h, _ = layer.step(x.cuda(), dev([0, 0, 0]), cache, dev([16, 32, 0]), pages, dev([1, 1, 1]))
        for i in range(3):
            r64, h64, _ = layer.plain(x[i:i + 1], lambda t: t.to(torch.float32).to(torch.float16).to(D))
            for g, w in ((r[i], r64[0]), (h[i], h64[0])):
                assert (A.t64(g) - w).norm() <= (1e-3 + 2.0 ** -11) * w.norm()
            out, sel, _ = st.layer(0, h[i].cpu().numpy(), r[i].cpu().numpy())
            ref, sel_o, _ = orc.moe_layer(hl, h[i].cpu().numpy(), r[i].cpu().numpy())
            assert np.array_equal(sel, sel_o)
            parity.assert_parity(out, ref, f"row {i}")
            other = lambda a, b: orc.moe_layer(hl, a.cpu().numpy(), b.cpu().numpy())[0]  # noqa: E731
            for row in (r[i], h[(i + 1) % 3]):  # another row shows
                assert parity.metrics(out, other(row, r[i]))["max_rel"] > 2 * parity.MAX_REL
            # and so does another residual, brought to the size of these experts' sum, which is far above it
            big = np.abs(ref).max() / float(r[i].abs().max())
            out = st.layer(0, h[i].cpu().numpy(), (big * r[i]).cpu().numpy())[0]
            parity.assert_parity(out, other(h[i], big * r[i]), f"row {i} with its residual")
            for res in (h[i], r[(i + 1) % 3]):
                assert parity.metrics(out, other(h[i], big * res))["max_rel"] > 2 * parity.MAX_REL
    finally:
        st.close()

"""The operators around the expert stage, as cases to time and to compare.

A layer whose experts come as 4-bit codes with group scales runs them in this order: the norm before the block,
the router, the (token, slot) pairs sorted by expert, the products with the experts' 4-bit weights, the rows taken
back to their tokens with the router's weights, and the norm after the block with its gate and the residual.

Operators ("op"):
  q4            rows times one 4-bit matrix (an attention or output projection, a dense layer);
  q4_ids        every row times the matrix its id names (one token, or a few, through their chosen experts);
  q4_sorted     rows sorted by expert times their experts' matrices (a prompt);
                with "up" two matrices at once and silu(gate) * up of their products;
  sort          the pairs sorted by expert, stable, ids outside the experts dropped;
  dispatch      the sort, then the tokens' rows laid out in that order;
  gather        the tokens' rows laid out in a given order;
  combine       the sorted rows back to their tokens, weighted, plus a residual;
  gather_grad   the gradient of "gather" (a combine with weights of one);
  combine_grad  the gradients of "combine" with respect to the rows and the weights;
  norm          v = r + scale * gate * norm(b), h = norm(v as stored), any part of it;
  norm_grad     the gradients of "norm" from its saved statistics.

Where `own` is false, run() computes them in elementary torch operations; where it is true, through the C ABI
(include/hoard_ops.h).
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _q4(name, op, tokens, k, experts, rows, cols, group, dtype, scales, zeros=False, up=False):
    """tokens rows of x (q4), or tokens that take k of `experts` matrices each; rows x cols is a matrix's size."""
    c = {"op": op, "tokens": tokens, "k": k, "experts": experts, "rows": rows, "cols": cols, "group": group,
         "dtype": dtype, "scales": scales, "zeros": zeros, "up": up}
    return dict(c, name=name) if name else c


def _pairs(name, op, tokens, k, experts, n, dtype, drop=0.0, res=False):
    """drop: the share of pairs whose id lies outside the experts (padding, experts held elsewhere)."""
    c = {"op": op, "tokens": tokens, "k": k, "experts": experts, "n": n, "dtype": dtype, "drop": drop, "res": res}
    return dict(c, name=name) if name else c


def _norm(name, op, tokens, n, dtype, res, gate="none", sigmoid=False, post=True, pre=True, block=True, scale=1.0,
          offset=0.0):
    c = {"op": op, "tokens": tokens, "n": n, "dtype": dtype, "res": res, "gate": gate, "sigmoid": sigmoid,
         "post": post, "pre": pre, "block": block, "scale": scale, "offset": offset}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token through a small projection in fp32, the stage's activation type: latency
        _q4("q4_one_f32", "q4", 1, 1, 1, 512, 2048, 128, "f32", "f16"),
        # one token through a large projection: reading the weights is all there is
        _q4("q4_one_large", "q4", 1, 1, 1, 16384, 8192, 128, "bf16", "bf16"),
        # a verify step of odd length through a projection with small groups and zero points
        _q4("q4_verify_13", "q4", 13, 1, 1, 4096, 4096, 32, "f16", "f16", zeros=True),
        # one token through the gate and up matrices of its 8 of 128 experts
        _q4("q4_ids_gateup", "q4_ids", 1, 8, 128, 768, 2048, 64, "f32", "f16", up=True),
        # a prompt's 512 tokens, sorted, through the gate and up matrices of their experts
        _q4("q4_sorted_512", "q4_sorted", 512, 8, 128, 768, 2048, 128, "bf16", "bf16", up=True),
        # the sort of a verify step: nothing but latency
        _pairs("sort_16", "sort", 16, 8, 128, 0, "f32"),
        # a prompt's pairs sorted and its rows laid out, where a third of the experts live on another device
        _pairs("dispatch_1021", "dispatch", 1021, 10, 512, 2048, "bf16", drop=0.33),
        # expert outputs back to their tokens with weights and residual, a long prompt
        _pairs("combine_4096", "combine", 4096, 8, 128, 2048, "bf16", res=True),
        # training: the gradients of that for a batch of 8192 tokens, the largest call
        _pairs("combine_grad_8192", "combine_grad", 8192, 8, 128, 2048, "bf16"),
        # one token between two blocks: norm after, sigmoid gate of the token, residual, norm before, fp32
        _norm("norm_one", "norm", 1, 2048, "f32", "f32", gate="token", sigmoid=True),
        # a prompt's rows of odd length between two blocks, bf16 block, fp32 residual stream, a gate a channel
        _norm("norm_511_odd", "norm", 511, 4095, "bf16", "f32", gate="channel", scale=0.22),
        # training: the gradients of the same for a batch, the weights stored around zero
        _norm("norm_grad_4096", "norm_grad", 4096, 2048, "bf16", "bf16", gate="channel", offset=1.0),
    ]


MOST = 600e6  # of _cost, the largest listed case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: an operator, its types, and sizes over the logarithm of their range."""
    while True:
        op = rng.choice(["q4", "q4", "q4", "q4_ids", "q4_ids", "q4_sorted", "q4_sorted", "sort", "dispatch", "gather",
                         "combine", "gather_grad", "combine_grad", "norm", "norm", "norm_grad", "norm_grad"])
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        if op.startswith("q4"):
            group = rng.choice([32, 64, 128])
            cols = group * _log(rng, 1, 8192 // group)
            form = dict(dtype=dtype, scales=rng.choice(["f16", "bf16", "f32"]), zeros=rng.random() < 0.4,
                        up=rng.random() < 0.4)
            if op == "q4":
                case = _q4("", op, _log(rng, 1, 512), 1, 1, _log(rng, 64, 16384), cols, group, **form)
            else:
                experts = _log(rng, 4, 512)
                tokens = _log(rng, 1, 32 if op == "q4_ids" else 512)
                case = _q4("", op, tokens, rng.randint(1, min(10, experts)), experts, _log(rng, 64, 4096), cols, group,
                           **form)
            one = case["rows"] * case["cols"]
            if case["experts"] * one > 2 ** 29 or (op == "q4_ids" and case["tokens"] * case["k"] * one > 2 ** 29):
                continue  # the plain form holds these matrices in 32 bits
        elif op in ("norm", "norm_grad"):
            block = rng.random() < 0.8
            case = _norm("", op, _log(rng, 1, 8192), _log(rng, 64, 16384), dtype, rng.choice(["f32", dtype]),
                         gate=rng.choice(["none", "channel", "token", "full"]) if block else "none",
                         sigmoid=block and rng.random() < 0.5, post=block and rng.random() < 0.7,
                         pre=not block or rng.random() < 0.8, block=block,
                         scale=rng.choice([1.0, 0.22, 0.5]) if block else 1.0, offset=rng.choice([0.0, 0.0, 1.0]))
            case["sigmoid"] = case["sigmoid"] and case["gate"] != "none"
        else:
            experts = _log(rng, 4, 512)
            case = _pairs("", op, _log(rng, 1, 16384), rng.randint(1, min(10, experts)), experts, _log(rng, 64, 8192),
                          dtype, drop=rng.choice([0.0, 0.0, 0.1, 0.33]), res=op == "combine" and rng.random() < 0.5)
            if op == "sort":
                case["n"] = 0
        if _cost(case) <= MOST:
            return case


# --- inputs ------------------------------------------------------------------

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(((seed & 0xFFFFFFFF) * 1000003 + what) & 0x7FFFFFFFFFFF)


def _randn(seed, what, *size):
    return torch.randn(size, device="cuda", generator=_gen(seed, what))


def _matrix(case, seed, what):
    """4-bit codes around their middle, scales that give weights of deviation about 0.02, zero points near 8."""
    e, n, k, g = case["experts"], case["rows"], case["cols"], case["group"]
    codes = torch.empty((e, n, k // 2), dtype=torch.uint8, device="cuda")
    flat = codes.view(-1)
    gen = _gen(seed, what)
    step = 1 << 26
    for at in range(0, flat.numel(), step):
        m = min(step, flat.numel() - at)
        q = (torch.randn((m, 2), device="cuda", generator=gen) * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
        flat[at:at + m] = q[:, 0] | (q[:, 1] << 4)
    scales = (0.004 + 0.008 * torch.rand((e, n, k // g), device="cuda", generator=gen)).to(DTYPES[case["scales"]])
    zeros = torch.randint(6, 11, (e, n, k // g), dtype=torch.uint8, device="cuda", generator=gen) if case["zeros"] else None
    return {"codes": codes, "scales": scales, "zeros": zeros}


def _ids(case, seed):
    """k distinct experts a token, some taken more often than others; a dropped pair's id is one past the experts or -1."""
    m, k, e = case["tokens"], case["k"], case["experts"]
    logits = _randn(seed, 20, m, e) + _randn(seed, 21, e)
    top, ids = torch.sort(logits, dim=1, descending=True)
    ids, w = ids[:, :k].to(torch.int32).contiguous(), torch.softmax(top[:, :k], dim=1)
    if case.get("drop"):
        u = torch.rand((m, k), device="cuda", generator=_gen(seed, 22))
        ids = torch.where(u < case["drop"], torch.where(u < case["drop"] / 2, -1, e).to(torch.int32), ids)
    return ids.contiguous(), w.contiguous()


def _sorted(ids, experts):
    """place, order, offsets of the ids' pairs, as the sort gives them."""
    flat = ids.reshape(-1).to(torch.int64)
    key = torch.where((flat < 0) | (flat >= experts), experts, flat)
    ranked, order = torch.sort(key, stable=True)
    rows = torch.arange(flat.numel(), device=ids.device)
    place = torch.empty_like(order)
    place[order] = rows
    place = torch.where(key < experts, place, -1)
    order = torch.where(ranked < experts, order, -1)
    offsets = torch.searchsorted(ranked, torch.arange(experts + 1, device=ids.device))
    return place.to(torch.int32).view(ids.shape), order.to(torch.int32), offsets.to(torch.int32)


def prepare(case, seed):
    op, dt, m = case["op"], DTYPES[case["dtype"]], case["tokens"]
    dev = {"device": "cuda"}
    s = {"case": case}
    if op.startswith("q4"):
        s["w"] = _matrix(case, seed, 1)
        s["up"] = _matrix(case, seed, 2) if case["up"] else None
        rows = m * case["k"]
        s["y"] = torch.empty((rows, case["rows"]), dtype=dt, **dev)
        s["x"] = _randn(seed, 3, rows if op == "q4_sorted" else m, case["cols"]).to(dt)
        if op == "q4_ids":
            s["ids"] = _ids(case, seed)[0]
        if op == "q4_sorted":
            s["offsets"] = _sorted(_ids(case, seed)[0], case["experts"])[2]
            s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # the longest run of one expert
        return s
    n = case["n"]
    if op in ("norm", "norm_grad"):
        rt, f32 = DTYPES[case["res"]], torch.float32
        r = _randn(seed, 4, m, n).to(rt)
        s["b"] = (_randn(seed, 5, m, n) * 0.5).to(dt) if case["block"] else None
        about = 1.0 - case["offset"]  # weights are stored as they are, or less their offset
        s["w_post"] = about + 0.1 * _randn(seed, 6, n) if case["post"] else None
        s["w_pre"] = about + 0.1 * _randn(seed, 7, n) if case["pre"] else None
        size = {"none": None, "channel": (n,), "token": (m,), "full": (m, n)}[case["gate"]]
        s["gate"] = _randn(seed, 8, *size).to(dt if case["gate"] == "full" else f32) if size else None
        s["stats"] = torch.empty((m, 2), **dev)
        s["r"], s["r_out"], s["h"] = r, torch.empty((m, n), dtype=rt, **dev), torch.empty((m, n), dtype=dt, **dev)
        if op == "norm":
            return s
        v, _, s["stats"] = _norm_plain(s)  # what the forward pass kept
        s["r_out"] = v if case["block"] else r
        s["dr_out"] = _randn(seed, 9, m, n).to(rt)
        s["dh"] = _randn(seed, 10, m, n).to(dt) if case["pre"] else None
        s["dr"] = torch.empty((m, n), dtype=rt, **dev)
        for name in ("b", "gate", "w_post", "w_pre"):
            s["d" + name] = torch.empty_like(s[name]) if s[name] is not None else None
        # the call's workspace, of the size that the library names
        s["work"] = torch.empty(_norm_work(m, n), dtype=torch.uint8, **dev)
        return s
    s["ids"], s["w"] = _ids(case, seed)
    s["place"], s["order"], s["offsets"] = _sorted(s["ids"], case["experts"])
    rows = m * case["k"]
    if op in ("sort", "dispatch"):
        s["work"] = torch.empty(_sort_work(rows, case["experts"]), dtype=torch.uint8, **dev)
    if op in ("gather", "dispatch"):
        s["x"] = _randn(seed, 11, m, n).to(dt)
        s["xs"] = torch.zeros((rows, n), dtype=dt, **dev)  # rows behind the last pair stay as they are
    elif op != "sort":
        s["y"] = _randn(seed, 12, rows, n).to(dt)
        s["res"] = _randn(seed, 13, m, n).to(dt) if case["res"] else None
        s["out"] = torch.empty((m, n), dtype=dt, **dev)
    if op == "combine_grad":
        s["dout"] = _randn(seed, 14, m, n).to(dt)
        s["dy"], s["dw"] = torch.zeros((rows, n), dtype=dt, **dev), torch.empty_like(s["w"])
    return s


def _sort_work(pairs, experts):
    """Bytes of workspace that cover hoard_sort_workspace's answer: a count an expert for every 1024 pairs."""
    return 4 * (experts + 1) * (pairs // 1024 + 2) + 256


def _norm_work(rows, n):
    """Bytes of workspace that cover hoard_norm_workspace's answer: three partial sums a column, 1024 groups of rows."""
    return 3 * 4 * n * min(1024, rows) + 256


# --- one pass ----------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    if op.startswith("q4"):
        return _q4_plain(state)
    if op in ("norm", "norm_grad"):
        if op == "norm_grad":
            return _norm_grad_plain(state)
        v, h, stats = _norm_plain(state)
        out = {"stats": stats}
        if v is not None:
            out["r_out"] = v
        if h is not None:
            out["h"] = h
        return out
    return _pairs_plain(state)


def _dense(w, e=None):
    """A matrix's values in 32 bits; e: those of the experts it names, one after the other."""
    codes, scales, zeros = w["codes"], w["scales"], w["zeros"]
    if e is not None:
        codes, scales, zeros = codes[e], scales[e], zeros[e] if zeros is not None else None
    q = torch.stack([codes & 15, codes >> 4], dim=-1).view(*scales.shape, -1).to(torch.float32)
    q = q - (8.0 if zeros is None else zeros.to(torch.float32).unsqueeze(-1))
    return (q * scales.to(torch.float32).unsqueeze(-1)).flatten(-2)


def _silu_mul(g, u):
    return g / (1.0 + torch.exp(-g)) * u


def _q4_plain(s):
    case, x = s["case"], s["x"].to(torch.float32)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "q4":
        product = lambda w: x @ _dense(w)[0].t()  # noqa: E731
    elif case["op"] == "q4_ids":
        ids = s["ids"].reshape(-1).to(torch.int64)
        rows = x.repeat_interleave(case["k"], dim=0).unsqueeze(-1)
        product = lambda w: torch.bmm(_dense(w, ids), rows).squeeze(-1)  # noqa: E731
    else:
        # every expert's rows in a batch of their own, padded to the longest
        off = s["offsets"].to(torch.int64)
        r = torch.arange(x.shape[0], device=x.device)
        e = torch.searchsorted(off, r, right=True) - 1
        at = r - off[e]
        batch = torch.zeros((case["experts"], s["most"], case["cols"]), device=x.device)
        batch[e, at] = x
        product = lambda w: torch.bmm(batch, _dense(w).transpose(1, 2).contiguous())[e, at]  # noqa: E731
    y = product(s["w"])
    if case["up"]:
        y = _silu_mul(y, product(s["up"]))
    return {"y": y.to(dt)}


def _pairs_plain(s):
    case, op = s["case"], s["case"]["op"]
    m, k, n, dt = case["tokens"], case["k"], case["n"], DTYPES[case["dtype"]]
    place = s["place"]
    out = {}
    if op in ("sort", "dispatch"):
        place, order, offsets = _sorted(s["ids"], case["experts"])
        out = {"place": place, "order": order, "offsets": offsets}
        if op == "sort":
            return out
    at = place.reshape(-1).to(torch.int64)
    kept = (at >= 0).view(m, k, 1)
    if op in ("gather", "dispatch"):
        xs = torch.zeros((m * k + 1, n), dtype=dt, device=at.device)  # the last row takes the dropped pairs
        xs[torch.where(at >= 0, at, m * k)] = s["x"].repeat_interleave(k, dim=0)
        return dict(out, xs=xs[:m * k])
    if op == "combine_grad":
        dout = s["dout"].to(torch.float32)
        rows = torch.where(kept, s["y"][at.clamp(min=0)].view(m, k, n).to(torch.float32), 0.0)
        dw = (rows * dout.unsqueeze(1)).sum(dim=2)
        dy = torch.zeros((m * k + 1, n), dtype=dt, device=at.device)
        dy[torch.where(at >= 0, at, m * k)] = (s["w"].unsqueeze(2) * dout.unsqueeze(1)).view(m * k, n).to(dt)
        return {"dy": dy[:m * k], "dw": dw}
    rows = torch.where(kept, s["y"][at.clamp(min=0)].view(m, k, n).to(torch.float32), 0.0)
    if op == "combine":
        rows = rows * s["w"].unsqueeze(2)
    y = rows.sum(dim=1)
    if s["res"] is not None:
        y = y + s["res"].to(torch.float32)
    return {"out": y.to(dt)}


def _gate_of(s, f):
    """The gate as it multiplies a row, in type f, and its derivative by what is stored."""
    case, gate = s["case"], s["gate"]
    if gate is None:
        return torch.ones((1, 1), dtype=f, device="cuda"), None
    g = gate.to(f)
    g = g.unsqueeze(1) if case["gate"] == "token" else g
    if not case["sigmoid"]:
        return g, torch.ones_like(g)
    g = 1.0 / (1.0 + torch.exp(-g))
    return g, g * (1.0 - g)


def _norm_plain(s):
    case, f = s["case"], torch.float32
    v = s["r"].to(f)
    stats = torch.ones((case["tokens"], 2), device="cuda")
    if case["block"]:
        b = s["b"].to(f)
        if case["post"]:
            rho = torch.rsqrt((b * b).mean(dim=1) + EPS)
            stats[:, 0] = rho
            b = b * rho.unsqueeze(1) * (case["offset"] + s["w_post"])
        v = v + case["scale"] * _gate_of(s, f)[0] * b
    stored = v.to(DTYPES[case["res"]])  # the second norm is the stored stream's, as its gradient needs it
    h = None
    if case["pre"]:
        v = stored.to(f)
        rho = torch.rsqrt((v * v).mean(dim=1) + EPS)
        stats[:, 1] = rho
        h = (v * rho.unsqueeze(1) * (case["offset"] + s["w_pre"])).to(DTYPES[case["dtype"]])
    return stored if case["block"] else None, h, stats


def _norm_grad_plain(s):
    case, f = s["case"], torch.float32
    out = {}
    dv = s["dr_out"].to(f)
    if case["pre"]:
        v, dh, rho = s["r_out"].to(f), s["dh"].to(f), s["stats"][:, 1:2]
        u = dh * (case["offset"] + s["w_pre"])
        out["dw_pre"] = (dh * v * rho).sum(dim=0)
        dv = dv + rho * (u - v * rho * rho * (u * v).mean(dim=1, keepdim=True))
    out["dr"] = dv.to(DTYPES[case["res"]])
    if not case["block"]:
        return out
    b, rho = s["b"].to(f), s["stats"][:, 0:1]
    g, slope = _gate_of(s, f)
    post = b * rho * (case["offset"] + s["w_post"]) if case["post"] else b
    d = case["scale"] * g * dv
    if slope is not None:
        dg = case["scale"] * dv * post * slope
        out["dgate"] = {"channel": lambda: dg.sum(dim=0), "token": lambda: dg.sum(dim=1),
                        "full": lambda: dg.to(DTYPES[case["dtype"]])}[case["gate"]]()
    if case["post"]:
        out["dw_post"] = (d * b * rho).sum(dim=0)
        u = d * (case["offset"] + s["w_post"])
        d = rho * (u - b * rho * rho * (u * b).mean(dim=1, keepdim=True))
    out["db"] = d.to(DTYPES[case["dtype"]])
    return out


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import hoard_amd as H
    lib, case, op = H.load_library(), s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    types = {"f32": H.TYPE_F32, "f16": H.TYPE_F16, "bf16": H.TYPE_BF16}
    dt, m, k = types[case["dtype"]], case["tokens"], case.get("k", 1)
    if op.startswith("q4"):
        def matrix(w):
            return ctypes.byref(H.Q4Matrix(_p(w["codes"]), _p(w["scales"]), _p(w["zeros"]), case["rows"], case["cols"],
                                           case["group"], case["experts"], types[case["scales"]]))
        w, up, x, y = matrix(s["w"]), matrix(s["up"]) if case["up"] else None, _p(s["x"]), _p(s["y"])
        if op == "q4":
            H.check(lib.hoard_q4_matmul(w, up, dt, m, x, y, stream))
        elif op == "q4_ids":
            H.check(lib.hoard_q4_matmul_ids(w, up, dt, m * k, x, k, _p(s["ids"]), y, stream))
        else:
            H.check(lib.hoard_q4_matmul_sorted(w, up, dt, m * k, x, _p(s["offsets"]), y, stream))
        return {"y": s["y"]}
    if op in ("norm", "norm_grad"):
        kinds = {"none": H.GATE_NONE, "channel": H.GATE_CHANNEL, "token": H.GATE_TOKEN, "full": H.GATE_FULL}
        a = H.NormArgs(dt, types[case["res"]], kinds[case["gate"]], int(case["sigmoid"]), m, case["n"], EPS,
                       case["scale"], case["offset"], _p(s["r"]), _p(s["b"]), _p(s["gate"]), _p(s["w_post"]),
                       _p(s["w_pre"]), _p(s["r_out"]) if case["block"] or op == "norm_grad" else None,
                       _p(s["h"]) if case["pre"] else None, _p(s["stats"]))
        if op == "norm":
            H.check(lib.hoard_norm_forward(ctypes.byref(a), stream))
            out = {"stats": s["stats"]}
            if case["block"]:
                out["r_out"] = s["r_out"]
            if case["pre"]:
                out["h"] = s["h"]
            return out
        names = ["dr", "db", "dgate", "dw_post", "dw_pre"]
        g = H.NormGrads(_p(s["dr_out"]), _p(s["dh"]), *(_p(s[name]) for name in names))
        H.check(lib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(g), _p(s["work"]), s["work"].numel(), stream))
        return {name: s[name] for name in names if s[name] is not None}
    n, place, out = case["n"], _p(s["place"]), {}
    if op in ("sort", "dispatch"):
        H.check(lib.hoard_sort_pairs(m, k, case["experts"], _p(s["ids"]), place, _p(s["order"]), _p(s["offsets"]),
                                     _p(s["work"]), s["work"].numel(), stream))
        out = {"place": s["place"], "order": s["order"], "offsets": s["offsets"]}
        if op == "sort":
            return out
    if op in ("gather", "dispatch"):
        H.check(lib.hoard_sort_gather(dt, m, k, n, _p(s["x"]), place, None, _p(s["xs"]), stream))
        return dict(out, xs=s["xs"])
    if op == "combine_grad":
        H.check(lib.hoard_sort_combine_grad(dt, m, k, n, _p(s["dout"]), _p(s["y"]), place, _p(s["w"]), _p(s["dy"]),
                                            _p(s["dw"]), stream))
        return {"dy": s["dy"], "dw": s["dw"]}
    H.check(lib.hoard_sort_combine(dt, m, k, n, _p(s["y"]), place, _p(s["w"]) if op == "combine" else None,
                                   _p(s["res"]), _p(s["out"]), stream))
    return {"out": s["out"]}


def work(case):
    """Every input read once, every output written once; of the experts' matrices the ones that a pair takes
    (for independent, uniform ids the expected number)."""
    op, m, z = case["op"], case["tokens"], SIZE[case["dtype"]]
    if op.startswith("q4"):
        e, k, n, c = case["experts"], case["k"], case["rows"], case["cols"]
        taken = 1 if op == "q4" else e * (1.0 - (1.0 - k / e) ** m)
        mats = 2 if case["up"] else 1
        one = n * c / 2 + n * (c // case["group"]) * (SIZE[case["scales"]] + case["zeros"])
        rows_in = m * k if op == "q4_sorted" else m
        return {"bytes": mats * taken * one + z * (rows_in * c + m * k * n), "flops": 2 * mats * m * k * n * c}
    n = case["n"]
    if op in ("norm", "norm_grad"):
        full, rz = m * n, SIZE[case["res"]]
        weights = 4 * n * (case["post"] + case["pre"])
        gate = {"none": 0, "channel": 4 * n, "token": 4 * m, "full": z * full}[case["gate"]]
        if op == "norm":
            bytes_ = full * (rz * (1 + case["block"]) + z * (case["block"] + case["pre"])) + weights + gate + 8 * m
            return {"bytes": bytes_, "flops": 12 * full}
        bytes_ = full * (rz * (2 + case["pre"]) + z * (case["pre"] + 2 * case["block"])) + 2 * (weights + gate) + 8 * m
        return {"bytes": bytes_, "flops": 24 * full}
    pairs, kept = m * case["k"], m * case["k"] * (1.0 - case["drop"])
    sort = 4 * (3 * pairs + case["experts"] + 1)
    gather = z * n * (m + kept) + 4 * pairs
    if op == "sort":
        return {"bytes": sort, "flops": 0}
    if op == "dispatch":
        return {"bytes": sort + gather, "flops": 0}
    if op in ("gather", "gather_grad"):
        return {"bytes": gather, "flops": kept * n if op == "gather_grad" else 0}
    if op == "combine":
        return {"bytes": gather + 4 * pairs + (z * m * n if case["res"] else 0), "flops": 2 * kept * n}
    return {"bytes": z * n * (m + 2 * kept) + 12 * pairs, "flops": 3 * kept * n}


# --- the same in 64 bits -------------------------------------------------------

def _row_block64(w, e, r0, r1, group):
    """Rows r0..r1 of matrix e as float64."""
    c = w["codes"][e, r0:r1].to(torch.int64)
    q = torch.empty((r1 - r0, 2 * c.shape[1]), dtype=torch.float64, device=c.device)
    q[:, 0::2] = (c % 16).to(torch.float64)
    q[:, 1::2] = (c // 16).to(torch.float64)
    wide = lambda t: t[e, r0:r1].to(torch.float64).repeat_interleave(group, dim=1)  # noqa: E731
    return (q - (wide(w["zeros"]) if w["zeros"] is not None else 8.0)) * wide(w["scales"])


def _product64(w, e, x, group):
    n = w["codes"].shape[1]
    return torch.cat([x @ _row_block64(w, e, r, min(n, r + 4096), group).t().contiguous() for r in range(0, n, 4096)], 1)


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], torch.float64
    if op.startswith("q4"):
        rows = case["tokens"] * case["k"]
        x = s["x"].to(d)
        if op == "q4":
            takes = [(0, torch.arange(rows, device="cuda"))]
        else:
            ids = _ids(case, seed)[0].reshape(-1)
            ids = torch.sort(ids)[0] if op == "q4_sorted" else ids
            takes = [(e, torch.nonzero(ids == e).view(-1)) for e in torch.unique(ids).tolist()]
        y = torch.zeros((rows, case["rows"]), dtype=d, device="cuda")
        for e, r in takes:
            xe = x[r // case["k"]] if op == "q4_ids" else x[r]
            g = _product64(s["w"], e, xe, case["group"])
            y[r] = torch.nn.functional.silu(g) * _product64(s["up"], e, xe, case["group"]) if case["up"] else g
        return {"y": y}
    if op in ("norm", "norm_grad"):
        return _norm64(case, s)
    if op == "sort":
        return None
    m, k, n = case["tokens"], case["k"], case["n"]
    # the sorted row of pair p, counted apart from any sort: the pairs of lower experts, and the earlier ones of its own
    ids = s["ids"].reshape(-1).to(torch.int64)
    at = torch.full((m * k,), -1, dtype=torch.int64, device="cuda")
    next_row = 0
    for e in range(case["experts"]):
        mine = torch.nonzero(ids == e).view(-1)
        at[mine] = next_row + torch.arange(mine.numel(), device="cuda")
        next_row += mine.numel()
    pair = torch.nonzero(at >= 0).view(-1)
    if op in ("gather", "dispatch"):
        xs = torch.zeros((m * k, n), dtype=d, device="cuda")
        xs[at[pair]] = s["x"].to(d)[pair // k]
        return {"place": None, "order": None, "offsets": None, "xs": xs} if op == "dispatch" else {"xs": xs}
    w = s["w"].to(d).reshape(-1)
    if op == "combine_grad":
        dy, dw = torch.zeros((m * k, n), dtype=d, device="cuda"), torch.zeros(m * k, dtype=d, device="cuda")
        dout = s["dout"].to(d)
        dy[at[pair]] = w[pair].unsqueeze(1) * dout[pair // k]
        dw[pair] = (dout[pair // k] * s["y"].to(d)[at[pair]]).sum(dim=1)
        return {"dy": dy, "dw": dw.view(m, k)}
    out = s["res"].to(d) if s["res"] is not None else torch.zeros((m, n), dtype=d, device="cuda")
    rows = s["y"].to(d)[at[pair]]
    out.index_add_(0, pair // k, rows * w[pair].unsqueeze(1) if op == "combine" else rows)
    return {"out": out}


def _norm64(case, s):
    """By automatic differentiation of the forward formula, the statistics recomputed, for the gradients."""
    d = torch.float64
    wide = {k: (t.to(d) if torch.is_tensor(t) else t) for k, t in s.items()}
    back = case["op"] == "norm_grad"
    keep = [k for k in ("b", "gate", "w_post", "w_pre") if wide.get(k) is not None]

    def after(b, gate, w_post):
        if case["post"]:
            b = b / torch.sqrt((b ** 2).sum(1, keepdim=True) / case["n"] + EPS) * (w_post + case["offset"])
        if gate is not None:
            gate = torch.sigmoid(gate) if case["sigmoid"] else gate
            b = b * (gate.view(-1, 1) if case["gate"] == "token" else gate)
        return case["scale"] * b

    def before(v, w_pre):
        return v / torch.sqrt((v ** 2).sum(1, keepdim=True) / case["n"] + EPS) * (w_pre + case["offset"])

    if not back:
        v = wide["r"] + (after(wide["b"], wide["gate"], wide["w_post"]) if case["block"] else 0.0)
        stored = v.to(DTYPES[case["res"]]).to(d) if case["res"] != "f32" else v
        rho = lambda t: 1.0 / torch.sqrt((t ** 2).sum(1) / case["n"] + EPS)  # noqa: E731
        one = torch.ones(case["tokens"], dtype=d, device="cuda")
        out = {"stats": torch.stack([rho(wide["b"]) if case["post"] else one, rho(stored) if case["pre"] else one],
                                    dim=1)}
        if case["block"]:
            out["r_out"] = v
        if case["pre"]:
            out["h"] = before(stored, wide["w_pre"])
        return out
    for name in keep:
        wide[name].requires_grad_(True)
    v = wide["r_out"].clone().requires_grad_(True)
    total = wide["dr_out"]
    out = {}
    if case["pre"]:
        got = torch.autograd.grad(before(v, wide["w_pre"]), [v, wide["w_pre"]], wide["dh"])
        total, out["dw_pre"] = total + got[0], got[1]
    out["dr"] = total
    if case["block"]:
        names = [name for name in ("b", "gate", "w_post") if name in keep]
        got = torch.autograd.grad(after(wide["b"], wide["gate"], wide["w_post"]), [wide[x] for x in names], total)
        out.update({"d" + name: t for name, t in zip(names, got)})
    return out

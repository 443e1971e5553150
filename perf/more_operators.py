"""The operators of a layer's attention half, as cases to time and to compare.

Between the projection to queries, keys and values and the output projection a layer runs: the norms of each query and
key head with the rotation by its position, keys and values written to a paged cache, and the attention of the new
tokens over that cache.

Operators ("op"):
  heads       q_out, k_out = rotate(norm(q)), rotate(norm(k)) for each head, from rows of a fused projection;
  heads_grad  the gradients of "heads" from its saved statistics;
  cache       "heads" with keys and values written to the cache's pages, then the same rows read back from it;
  attn        attention of a few new tokens a sequence over its pages of the cache, with the sums' logarithms.

Where `own` is false, run() computes them in elementary torch operations; where it is true, through the C ABI
(include/hoard_attn.h).
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
EPS = 1e-6
BASE = 1e6  # of the rotation's frequencies


def _heads(name, op, tokens, hq, hkv, dim, rot, dtype, pairs=False, axes=1, norm=True, offset=0.0, far=0, cache="",
           page=0, read=""):
    """hq query and hkv key heads of `dim` values, the first `rot` of which turn; far: the first position."""
    c = {"op": op, "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rot": rot, "dtype": dtype, "pairs": pairs,
         "axes": axes, "norm": norm, "offset": offset, "far": far}
    if op == "cache":
        c.update(cache=cache, page=page, read=read)
    return dict(c, name=name) if name else c


def _attn(name, seqs, new, hq, hkv, dim, length, dtype, cache, page, ragged=False):
    """seqs sequences of up to `length` cached tokens, `new` of them with a query."""
    c = {"op": "attn", "seqs": seqs, "new": new, "hq": hq, "hkv": hkv, "dim": dim, "length": length, "dtype": dtype,
         "cache": cache, "page": page, "ragged": ragged}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a decode step in fp32, the stage's activation type: latency
        _heads("heads_one", "heads", 1, 32, 4, 128, 128, "f32", far=8191),
        # a long prompt's queries and keys
        _heads("heads_4096", "heads", 4096, 32, 4, 128, 128, "bf16"),
        # training: an odd batch of wide heads of which a quarter turns, weights stored around zero, three position axes
        _heads("heads_grad_511", "heads_grad", 511, 16, 2, 256, 64, "f16", offset=1.0, axes=3),
        # training: the gradients for a batch of 8192 tokens
        _heads("heads_grad_8192", "heads_grad", 8192, 32, 4, 128, 128, "bf16"),
        # a decode step of 16 sequences: keys and values into an 8-bit cache
        _heads("cache_16", "cache", 16, 32, 4, 128, 128, "bf16", far=100000, cache="i8", page=64, read="bf16"),
        # a long prompt of odd length into pages of 16 tokens, as 8 bits, and back for its own attention
        _heads("cache_5003", "cache", 5003, 16, 16, 128, 128, "f32", cache="i8", page=16, read="f16"),
        # one short sequence in fp32 over a 16-bit cache: latency
        _attn("attn_257", 1, 1, 32, 4, 128, 257, "f32", "f16", 64),
        # one long sequence: split over its length, all of the card reads one cache
        _attn("attn_32768", 1, 1, 32, 4, 128, 32768, "bf16", "bf16", 64),
        # one very long sequence over an 8-bit cache
        _attn("attn_131071", 1, 1, 32, 4, 128, 131071, "bf16", "i8", 128),
        # serving: 64 sequences of different lengths over an 8-bit cache, the largest call
        _attn("attn_64_ragged", 64, 1, 32, 4, 128, 8192, "bf16", "i8", 64, ragged=True),
        # a verify step: 5 new tokens a sequence, wide heads, some sequences with fewer drafts
        _attn("attn_verify_5", 16, 5, 16, 2, 256, 3001, "bf16", "bf16", 32, ragged=True),
        # serving with a key head for every query head
        _attn("attn_8_mha", 8, 1, 16, 16, 128, 2048, "f16", "f16", 16),
    ]


MOST = 330e6  # of _cost, about the largest listed case


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    """One more case: an operator, its types, and sizes over the logarithm of their range."""
    while True:
        op = rng.choice(["heads", "heads_grad", "cache", "cache", "attn", "attn", "attn"])
        dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
        dim = rng.choice([64, 96, 128, 128, 192, 256])
        hkv = _log(rng, 1, 16)
        hq = hkv * rng.choice([1, 2, 4, 5, 8, 16])
        if hq > 64:
            continue
        page = rng.choice([16, 32, 64, 128])
        if op == "attn":
            case = _attn("", _log(rng, 1, 128), rng.choice([1, 1, 1, _log(rng, 2, 16)]), hq, hkv, dim, 1, dtype,
                         rng.choice(["i8", "i8", "f16", "bf16"]), page, ragged=rng.random() < 0.6)
            case["length"] = _log(rng, case["new"], 131072)
            if case["seqs"] * case["length"] * hkv * dim > 2 ** 28:
                continue  # the plain form holds keys and values in 32 bits, every sequence at the longest's length
        else:
            case = _heads("", op, _log(rng, 1, 16384), hq, hkv, dim, rng.choice([dim, dim, dim // 2, dim // 4, 0]), dtype,
                          pairs=rng.random() < 0.3, axes=rng.choice([1, 1, 3]), norm=rng.random() < 0.8,
                          offset=rng.choice([0.0, 0.0, 1.0]), far=rng.choice([0, _log(rng, 1, 1000000)]), page=page)
            if op == "cache":
                case["cache"] = rng.choice(["i8", "i8", "f16", "bf16"])
                case["read"] = case["cache"] if case["cache"] != "i8" else rng.choice(["f16", "bf16"])
            if not case["norm"] and case["rot"] == 0 and op != "cache":
                continue  # nothing to do
        if _cost(case) <= MOST:
            return case


# --- inputs ------------------------------------------------------------------

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed(((seed & 0xFFFFFFFF) * 1000003 + what) & 0x7FFFFFFFFFFF)


def _randn(seed, what, *size):
    return torch.randn(size, device="cuda", generator=_gen(seed, what))


def _positions(case, seed):
    """Positions of consecutive tokens; with three axes (time, height, width) those of an image's patches among text."""
    m = case["tokens"]
    t = case["far"] + torch.arange(m, device="cuda")
    if case["axes"] == 1:
        return t.to(torch.int32).view(1, m)
    hw = torch.randint(0, 64, (2, m), device="cuda", generator=_gen(seed, 20))
    return torch.cat([t.view(1, m), case["far"] + hw]).to(torch.int32).contiguous()


def _scatter_pages(seed, pages, pool):
    """`pages` page numbers of a pool in no order."""
    return torch.randperm(pool, device="cuda", generator=_gen(seed, 21))[:pages].to(torch.int32)


def _quantise(x):
    """8-bit codes of rows and what a step of each row is."""
    x = x.to(torch.float32)
    scale = x.abs().amax(dim=-1, keepdim=True) / 127.0
    codes = torch.where(scale > 0, torch.round(x / scale), 0.0).clamp(-127, 127)
    return codes.to(torch.int8), scale.squeeze(-1)


def prepare(case, seed):
    op, dt = case["op"], DTYPES[case["dtype"]]
    dev = {"device": "cuda"}
    s = {"case": case}
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    if op == "attn":
        return _prepare_attn(case, seed, s)
    m, rot = case["tokens"], case["rot"]
    # rows of the fused projection: queries, keys, values
    s["qkv"] = _randn(seed, 1, m, (hq + 2 * hkv) * dim).to(dt)
    about = 1.0 - case["offset"]
    s["w_q"] = about + 0.1 * _randn(seed, 2, dim) if case["norm"] else None
    s["w_k"] = about + 0.1 * _randn(seed, 3, dim) if case["norm"] else None
    s["pos"] = _positions(case, seed)
    i = torch.arange(rot // 2, dtype=torch.float64, **dev)
    s["freq"] = BASE ** (-2.0 * i / rot) if rot else None
    s["axis"] = (torch.arange(rot // 2, **dev) % 3).to(torch.uint8) if case["axes"] == 3 and rot else None
    s["stats"] = torch.empty((m, hq + hkv), **dev) if case["norm"] else None
    s["q_out"] = torch.empty((m, hq, dim), dtype=dt, **dev)
    s["k_out"] = torch.empty((m, hkv, dim), dtype=dt, **dev)
    if op == "heads_grad":
        q, k, _ = _parts(s)
        s["stats"] = torch.cat([_norm(s, q, s["w_q"])[1], _norm(s, k, s["w_k"])[1]], dim=1) if case["norm"] else None
        s["dq_out"] = _randn(seed, 4, m, hq, dim).to(dt)
        s["dk_out"] = _randn(seed, 5, m, hkv, dim).to(dt)
        s["dqkv"] = torch.empty_like(s["qkv"])  # the projection's gradient, whose last part is the values'
        s["dw_q"], s["dw_k"] = torch.empty(dim, **dev), torch.empty(dim, **dev)
        s["work"] = torch.empty(_heads_work(dim), dtype=torch.uint8, **dev)
    if op == "cache":
        page, ct = case["page"], DTYPES[case["cache"]]
        pages = -(-m // page)
        pool = pages + max(4, pages // 8)
        table = _scatter_pages(seed, pages, pool).to(torch.int64)
        t = torch.arange(m, **dev)
        s["slots"] = (table[t // page] * page + t % page).to(torch.int32)
        for name in ("k", "v"):
            s[name + "_cache"] = torch.zeros((pool, hkv, page, dim), dtype=ct, **dev)
            s[name + "_scale"] = torch.zeros((pool, hkv, page), **dev) if case["cache"] == "i8" else None
            s[name + "_read"] = torch.empty((m, hkv, dim), dtype=DTYPES[case["read"]], **dev)
    return s


def _prepare_attn(case, seed, s):
    dev = {"device": "cuda"}
    n, t, hq, hkv, dim, page = (case[x] for x in ("seqs", "new", "hq", "hkv", "dim", "page"))
    lengths = torch.full((n,), case["length"], dtype=torch.int64, **dev)
    if case["ragged"]:
        u = torch.rand(n, device="cuda", generator=_gen(seed, 10))
        lengths = (case["length"] * (1.0 + 15.0 * u) / 16.0).to(torch.int64)
        lengths = lengths.clamp(min(case["length"], t), case["length"])
    width = -(-case["length"] // page)
    pool = n * width + 4
    s["pages"] = _scatter_pages(seed, n * width, pool).view(n, width)
    # a row sees its own token and those before it
    lens = (lengths.view(n, 1) - t + 1 + torch.arange(t, **dev)).clamp(min=0)
    if case["ragged"] and t > 1:  # sequences with fewer new tokens: their last rows see nothing
        drafts = torch.randint(1, t + 1, (n, 1), device="cuda", generator=_gen(seed, 11))
        lens = torch.where(torch.arange(t, **dev) < drafts, lens, 0)
    s["lens"] = lens.to(torch.int32).contiguous()
    ct = DTYPES[case["cache"]]
    for what, name in ((12, "k"), (13, "v")):
        cache = torch.empty((pool, hkv, page, dim), dtype=ct, **dev)
        scale = torch.empty((pool, hkv, page), **dev) if case["cache"] == "i8" else None
        step, gen = max(1, 2 ** 26 // (hkv * page * dim)), _gen(seed, what)
        for at in range(0, pool, step):
            x = torch.randn(cache[at:at + step].shape, generator=gen, **dev)
            if scale is None:
                cache[at:at + step] = x.to(ct)
            else:
                cache[at:at + step], scale[at:at + step] = _quantise(x)
        s[name + "_cache"], s[name + "_scale"] = cache, scale
    # queries that single out some keys: scores of deviation 2
    s["q"] = (2.0 * _randn(seed, 14, n * t, hq, dim)).to(DTYPES[case["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((n * t, hq), **dev)
    s["work"] = torch.empty(_attn_work(case), dtype=torch.uint8, **dev)
    return s


def _heads_work(dim):
    """Bytes of workspace that cover hoard_heads_workspace's answer: two rows of partial sums a group, 1024 groups."""
    return 2 * 4 * dim * 1024 + 256


def _attn_work(case):
    """Bytes of workspace that cover hoard_attn_workspace's answer: up to 256 parts of every row, or 4096 parts of 16."""
    rows = case["seqs"] * case["new"] * case["hq"]
    return 4 * (case["dim"] + 2) * (min(256 * rows, 2 * rows + 16 * 4096) + 64)


# --- one pass ----------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    if op == "attn":
        return _attn_plain(state)
    if op == "heads_grad":
        return _heads_grad_plain(state)
    q, k, v = _heads_plain(state)
    dt = DTYPES[state["case"]["dtype"]]
    if op == "heads":
        out = {"q_out": q[0].to(dt), "k_out": k[0].to(dt)}
        if state["case"]["norm"]:
            out["stats"] = torch.cat([q[1], k[1]], dim=1)
        return out
    return dict(_cache_plain(state, k[0], v), q_out=q[0].to(dt))


def _parts(s):
    """The heads of a fused row, in 32 bits."""
    case = s["case"]
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    x = s["qkv"].view(case["tokens"], hq + 2 * hkv, dim).to(torch.float32)
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


def _norm(s, x, w):
    if w is None:
        return x, None
    rho = torch.rsqrt((x * x).mean(dim=-1) + EPS)
    return x * rho.unsqueeze(-1) * (s["case"]["offset"] + w), rho


def _turn(s):
    """Cosines and sines [tokens, 1, rot / 2], the angles in 64 bits."""
    case = s["case"]
    axis = s["axis"].to(torch.int64) if s["axis"] is not None else torch.zeros(case["rot"] // 2, dtype=torch.int64, device="cuda")
    angle = (s["pos"].to(torch.float64)[axis].t() * s["freq"]).unsqueeze(1)
    return torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)


def _rotate(s, x, cos, sin):
    case, rot = s["case"], s["case"]["rot"]
    out = x.clone()
    if case["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    return out


def _heads_plain(s):
    """((q_out, rho), (k_out, rho), v) in 32 bits."""
    q, k, v = _parts(s)
    q, k = _norm(s, q, s["w_q"]), _norm(s, k, s["w_k"])
    if s["case"]["rot"]:
        cos, sin = _turn(s)
        q, k = (_rotate(s, q[0], cos, sin), q[1]), (_rotate(s, k[0], cos, sin), k[1])
    return q, k, v


def _heads_grad_plain(s):
    case, dt = s["case"], DTYPES[s["case"]["dtype"]]
    q, k, _ = _parts(s)
    hq = case["hq"]
    dq, dk = s["dq_out"].to(torch.float32), s["dk_out"].to(torch.float32)
    if case["rot"]:
        cos, sin = _turn(s)
        dq, dk = _rotate(s, dq, cos, -sin), _rotate(s, dk, cos, -sin)
    if not case["norm"]:
        return {"dq": dq.to(dt), "dk": dk.to(dt)}
    rq, rk = s["stats"][:, :hq].unsqueeze(-1), s["stats"][:, hq:].unsqueeze(-1)

    def back(d, x, rho, w):
        u = d * (case["offset"] + w)
        return rho * (u - x * rho * rho * (u * x).mean(dim=-1, keepdim=True)), (d * x * rho).sum(dim=(0, 1))

    (dq, dw_q), (dk, dw_k) = back(dq, q, rq, s["w_q"]), back(dk, k, rk, s["w_k"])
    return {"dq": dq.to(dt), "dk": dk.to(dt), "dw_q": dw_q, "dw_k": dw_k}


def _cache_plain(s, k, v):
    case = s["case"]
    page, rt = case["page"], DTYPES[case["read"]]
    at = s["slots"].to(torch.int64)
    p, o = at // page, at % page
    out = {}
    for name, x in (("k", k), ("v", v)):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if scale is None:
            cache[p, :, o] = x.to(cache.dtype)
            out[name + "_read"] = cache[p, :, o].to(rt)
        else:
            cache[p, :, o], scale[p, :, o] = _quantise(x)
            out[name + "_read"] = (cache[p, :, o].to(torch.float32) * scale[p, :, o].unsqueeze(-1)).to(rt)
    return out


def _attn_plain(s):
    case = s["case"]
    n, t, hq, hkv, dim = (case[x] for x in ("seqs", "new", "hq", "hkv", "dim"))
    g, pages = hq // hkv, s["pages"].to(torch.int64)

    def values(cache, scale):
        """[n, hkv, keys, dim] in 32 bits."""
        x = cache[pages].to(torch.float32)
        if scale is not None:
            x = x * scale[pages].unsqueeze(-1)
        return x.transpose(1, 2).reshape(n, hkv, -1, dim)

    # the rows of a key head's queries: (token, query head of the group)
    q = s["q"].to(torch.float32).view(n, t, hkv, g, dim).transpose(1, 2).reshape(n, hkv, t * g, dim)
    scores = torch.matmul(q, values(s["k_cache"], s["k_scale"]).transpose(2, 3)) * dim ** -0.5
    seen = torch.arange(scores.shape[-1], device="cuda") < s["lens"].view(n, 1, t, 1, 1)
    seen = seen.expand(n, hkv, t, g, scores.shape[-1]).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    e = torch.exp(scores - top)
    total = e.sum(dim=-1, keepdim=True)
    values_v = values(s["v_cache"], s["v_scale"])
    out = torch.matmul(e, values_v) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).view(n, hkv, t, g)
    out = out.view(n, hkv, t, g, dim).transpose(1, 2).reshape(n * t, hq, dim)
    return {"out": out.to(DTYPES[case["dtype"]]), "lse": lse.transpose(1, 2).reshape(n * t, hq)}


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    import hoard_amd as H
    lib, case, op = H.load_library(), s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    types = {"f32": H.TYPE_F32, "f16": H.TYPE_F16, "bf16": H.TYPE_BF16, "i8": H.TYPE_I8}
    dt, hq, hkv, dim = types[case["dtype"]], case["hq"], case["hkv"], case["dim"]
    cache = None
    if "cache" in case:
        cache = H.KvCache(_p(s["k_cache"]), _p(s["v_cache"]), _p(s["k_scale"]), _p(s["v_scale"]), types[case["cache"]],
                          s["k_cache"].shape[0], case["page"], hkv, dim)
    if op == "attn":
        a = H.AttnArgs(dt, case["seqs"], case["new"], hq, s["pages"].shape[1], dim ** -0.5, hq * dim, _p(s["q"]),
                       _p(s["pages"]), _p(s["lens"]), _p(s["out"]), _p(s["lse"]))
        H.check(lib.hoard_attn_decode(ctypes.byref(cache), ctypes.byref(a), _p(s["work"]), s["work"].numel(), stream))
        return {"out": s["out"], "lse": s["lse"]}
    m, row, z = case["tokens"], (hq + 2 * hkv) * dim, SIZE[case["dtype"]]
    qkv = s["qkv"].data_ptr()
    k, v = qkv + hq * dim * z, qkv + (hq + hkv) * dim * z
    written = op == "cache"
    a = H.HeadsArgs(dt, m, hq, hkv, dim, case["rot"], H.ROPE_PAIRS if case["pairs"] else H.ROPE_HALVES, case["axes"], EPS,
                    case["offset"], row, row, row, hq * dim, hkv * dim, qkv, k, v if written else None, _p(s["w_q"]),
                    _p(s["w_k"]), _p(s["pos"]), _p(s["freq"]), _p(s["axis"]), _p(s["q_out"]),
                    None if written else _p(s["k_out"]), None if written else _p(s["stats"]),
                    ctypes.addressof(cache) if written else None, _p(s["slots"]) if written else None)
    if op == "heads_grad":
        dqkv = s["dqkv"].data_ptr()
        norm = case["norm"]
        g = H.HeadsGrads(_p(s["dq_out"]), _p(s["dk_out"]), dqkv, dqkv + hq * dim * z, _p(s["dw_q"]) if norm else None,
                         _p(s["dw_k"]) if norm else None)
        H.check(lib.hoard_heads_backward(ctypes.byref(a), ctypes.byref(g), _p(s["work"]), s["work"].numel(), stream))
        d = s["dqkv"].view(m, hq + 2 * hkv, dim)
        out = {"dq": d[:, :hq], "dk": d[:, hq:hq + hkv]}
        return dict(out, dw_q=s["dw_q"], dw_k=s["dw_k"]) if norm else out
    H.check(lib.hoard_heads_forward(ctypes.byref(a), stream))
    if op == "heads":
        out = {"q_out": s["q_out"], "k_out": s["k_out"]}
        return dict(out, stats=s["stats"]) if case["norm"] else out
    H.check(lib.hoard_kv_read(ctypes.byref(cache), types[case["read"]], m, _p(s["slots"]), _p(s["k_read"]), hkv * dim,
                              _p(s["v_read"]), hkv * dim, stream))
    return {"k_read": s["k_read"], "v_read": s["v_read"], "q_out": s["q_out"]}


def work(case):
    """Every input read once, every output written once; of a cache the keys and values that a row sees (for lengths
    that differ their expected number)."""
    op, z, hq, hkv, dim = case["op"], SIZE[case["dtype"]], case["hq"], case["hkv"], case["dim"]
    if op == "attn":
        keys = case["seqs"] * case["length"] * (17 / 32 if case["ragged"] else 1.0)
        row = dim * SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0)
        rows = case["seqs"] * case["new"] * hq
        return {"bytes": 2 * keys * hkv * row + 2 * z * rows * dim + 4 * rows, "flops": 4 * keys * case["new"] * hq * dim}
    m, values = case["tokens"], case["tokens"] * (hq + hkv) * dim
    small = 4 * m * case["axes"] + 8 * case["rot"] // 2 + (8 * dim + 4 * m * (hq + hkv) if case["norm"] else 0)
    if op == "heads":
        return {"bytes": 2 * z * values + small, "flops": 10 * values}
    if op == "heads_grad":
        return {"bytes": z * values * (3 if case["norm"] else 2) + small, "flops": 16 * values}
    kv = 2 * m * hkv
    held = kv * (dim * SIZE[case["cache"]] + (4 if case["cache"] == "i8" else 0))
    return {"bytes": z * (2 * m * hq * dim + kv * dim) + 2 * held + SIZE[case["read"]] * kv * dim + small,
            "flops": 10 * values + 6 * kv * dim}


# --- the same in 64 bits -------------------------------------------------------

def _turned64(case, s, y, back=False):
    """The rotation as a product with complex numbers of modulus one."""
    rot, m = case["rot"], case["tokens"]
    if not rot:
        return y
    pos = s["pos"].to(torch.float64)
    if s["axis"] is None:
        angle = pos[0].view(m, 1) * s["freq"].view(1, -1)
    else:
        angle = torch.stack([pos[int(a)] for a in s["axis"].tolist()], dim=1) * s["freq"].view(1, -1)
    w = torch.polar(torch.ones_like(angle), -angle if back else angle).view(m, 1, rot // 2)
    head = y[..., :rot]
    if case["pairs"]:
        c = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous()) * w
        head = torch.view_as_real(c).reshape(head.shape)
    else:
        c = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * w
        head = torch.cat([c.real, c.imag], dim=-1)
    return torch.cat([head, y[..., rot:]], dim=-1)


def _head64(case, s, x, w):
    if w is not None:
        x = x / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / case["dim"] + EPS) * (w + case["offset"])
    return _turned64(case, s, x)


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], torch.float64
    if op == "attn":
        return _attn64(case, s)
    hq, hkv, dim, m = case["hq"], case["hkv"], case["dim"], case["tokens"]
    q, k, v = (x.to(d) for x in torch.split(s["qkv"].view(m, -1, dim), [hq, hkv, hkv], dim=1))
    w_q, w_k = (s[x].to(d) if case["norm"] else None for x in ("w_q", "w_k"))
    if op == "heads_grad":
        out = {}
        for name, x, w in (("q", q, w_q), ("k", k, w_k)):
            x = x.clone().requires_grad_(True)
            leaves = [x] + ([w.requires_grad_(True)] if w is not None else [])
            got = torch.autograd.grad(_head64(case, s, x, w), leaves, s["d%s_out" % name].to(d))
            out["d" + name] = got[0]
            if w is not None:
                out["dw_" + name] = got[1]
        return out
    q_out, k_out = _head64(case, s, q, w_q), _head64(case, s, k, w_k)
    if op == "heads":
        out = {"q_out": q_out, "k_out": k_out}
        if case["norm"]:
            out["stats"] = (torch.cat([q, k], dim=1).square().sum(dim=-1) / dim + EPS) ** -0.5
        return out
    out = {"q_out": q_out}
    for name, x in (("k_read", k_out), ("v_read", v)):
        if case["cache"] == "i8":
            step = x.abs().max(dim=-1, keepdim=True).values / 127.0
            x = torch.round(x / step) * step
        out[name] = x
    return out


def _attn64(case, s):
    """Sequence by sequence and key head by key head."""
    n, t, hq, hkv, dim, page = (case[x] for x in ("seqs", "new", "hq", "hkv", "dim", "page"))
    d, g = torch.float64, hq // hkv
    if n * hkv > 1024:
        return None  # of many small products: the loop's own time
    out = torch.zeros((n * t, hq, dim), dtype=d, device="cuda")
    lse = torch.full((n * t, hq), -math.inf, dtype=d, device="cuda")
    lens = s["lens"].tolist()
    for i in range(n):
        longest = max(lens[i])
        if longest == 0:
            continue
        ids = s["pages"][i, :-(-longest // page)].to(torch.int64)
        for h in range(hkv):
            k, v = ((s[x + "_cache"][ids, h].to(d) * (s[x + "_scale"][ids, h].to(d).unsqueeze(-1) if s[x + "_scale"] is not None else 1.0))
                    .reshape(-1, dim)[:longest] for x in ("k", "v"))
            q = s["q"][i * t:(i + 1) * t, h * g:(h + 1) * g].to(d).reshape(t * g, dim)
            scores = (q @ k.t()) / math.sqrt(dim)
            hidden = torch.arange(longest, device="cuda") >= s["lens"][i].view(t, 1)
            scores.view(t, g, longest).masked_fill_(hidden.unsqueeze(1), -math.inf)
            weights = torch.softmax(scores, dim=1)
            rows = (torch.nan_to_num(weights, nan=0.0) @ v).view(t, g, dim)
            out[i * t:(i + 1) * t, h * g:(h + 1) * g] = rows
            lse[i * t:(i + 1) * t, h * g:(h + 1) * g] = torch.logsumexp(scores, dim=1).view(t, g)
    return {"out": out, "lse": lse}

"""Plain 64-bit forms of the operators of include/hoard_attn.h, on the CPU, and the bounds their results are held to.

As in opsref.py bounds count roundings: u(t) is half a step of type t, a sum of n terms in 32 bits is off by at most
n * u(f32) of the sum of their magnitudes, each factor of a term adds a u.

Cosines and sines: the fraction of a turn rounds to 32 bits (at most half of 2 pi u of an angle up to pi), the function
itself is good to 4 u of 1, and the turns are formed with three roundings in 64 bits on either side.
"""
import math

import torch

from opsref import U32, close, stored, u  # noqa: F401

D = torch.float64


def t64(t):
    return None if t is None else t.detach().cpu().to(D)


def angles(pos, freq, axis):
    """[tokens, 1, rot / 2] angles of pos [axes, tokens], and how far off a cosine may be."""
    pos, freq = t64(pos), t64(freq)
    axis = torch.zeros(len(freq), dtype=torch.int64) if axis is None else axis.cpu().to(torch.int64).clamp(max=len(pos) - 1)
    a = (pos[axis].t() * freq).unsqueeze(1)
    return a, (math.pi + 4) * U32 + 6 * 2.0 ** -53 * a.abs()


def _halves(x, rot, pairs):
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])


def rotate(x, ex, rope, back=False):
    """x [tokens, heads, dim] turned, and its bound from ex, x's own."""
    if rope is None:
        return x, ex
    pos, freq, axis, pairs = rope
    if pos.dim() == 1:
        pos = pos.unsqueeze(0)
    rot = 2 * len(freq)
    a, ec = angles(pos, freq, axis)
    c, s = torch.cos(a), torch.sin(-a if back else a)
    out, bound = x.clone(), ex.clone()
    x1, x2 = _halves(x, rot, pairs)
    e1, e2 = _halves(ex, rot, pairs)
    y1, y2 = _halves(out, rot, pairs)
    y1.copy_(x1 * c - x2 * s)
    y2.copy_(x2 * c + x1 * s)
    off = (x1.detach().abs() + x2.detach().abs()) * (ec + 3 * U32) + (e1 + e2) * (1 + ec)
    for b in _halves(bound, rot, pairs):
        b.copy_(off)
    return out, bound


def head_norm(x, w, eps, offset):
    """(y, its bound, rho) of x [tokens, heads, dim]: rho's sum of squares is off by dim + 2 roundings, halved by the
    root, which rounds twice with its reciprocal; three products and a sum follow."""
    if w is None:
        return x, torch.zeros_like(x), torch.ones(x.shape[:2], dtype=D)
    rho = 1.0 / torch.sqrt(x.square().mean(dim=-1) + eps)
    y = x * rho.unsqueeze(-1) * (offset + w)
    return y, y.abs() * ((x.shape[-1] + 2) / 2 + 8) * U32, rho


def heads(x, w, rope, eps, offset):
    """(z, bound before storing, rho)."""
    y, e, rho = head_norm(t64(x), t64(w), eps, offset)
    z, e = rotate(y, e, rope)
    return z, e, rho


def heads_grad(dz, x, w, rope, rho, offset):
    """(dx, its bound, dw, its bound) given the statistics as stored."""
    dz, x, w = t64(dz), t64(x), t64(w)
    dy, e = rotate(dz, torch.zeros_like(dz), rope, back=True)
    if w is None:
        return dy, e, None, None
    rho = t64(rho).unsqueeze(-1)
    wo = offset + w
    uu, eu = dy * wo, (e + dy.abs() * 3 * U32) * wo.abs()
    n = x.shape[-1]
    mean = (uu * x).mean(dim=-1, keepdim=True)
    em = ((uu * x).abs() * (n + 8) * U32 + eu * x.abs()).mean(dim=-1, keepdim=True)
    dx = rho * (uu - x * rho ** 2 * mean)
    ex = rho * (eu + x.abs() * rho ** 2 * (em + 8 * U32 * mean.abs()) + 4 * U32 * (uu.abs() + (x * rho ** 2 * mean).abs()))
    terms = dy * x * rho
    count = x.shape[0] * x.shape[1]
    dw = terms.sum(dim=(0, 1))
    ew = (terms.abs() * (count + 8) * U32 + e * (x * rho).abs()).sum(dim=(0, 1))
    return dx, ex, dw, ew


# -- the cache ----------------------------------------------------------------------

def quantised(x):
    """Codes and steps of rows of fp32 values, each operation rounded to 32 bits as the kernel forms it."""
    x = x.detach().cpu().to(torch.float32)
    step = x.abs().amax(dim=-1) / 127.0
    q = torch.where(step.unsqueeze(-1) > 0, torch.round(x / step.unsqueeze(-1)), 0.0).clamp(-127, 127)
    bad = ~torch.isfinite(x).all(dim=-1)
    return torch.where(bad.unsqueeze(-1), 0.0, q).to(torch.int8), torch.where(bad, math.nan, step)


def values(cache, scale):
    """float64 values of cache rows."""
    x = t64(cache)
    return x if scale is None else x * t64(scale).unsqueeze(-1)


# -- attention ------------------------------------------------------------------------

def gathered(pages, n, page, n_pages):
    """(page, place) of the first n keys, and which of them are on a page of the cache."""
    j = torch.arange(n)
    p = pages[j // page].to(torch.int64)
    ok = (p >= 0) & (p < n_pages)
    return torch.where(ok, p, 0), j % page, ok


def attention(q, k, v, ks, vs, pages, lens, scale, dtype):
    """(out, bound before storing, lse, its bound) of q [rows, heads, dim] with caches k, v [pages, kv, page, dim].

    A score is off by its sum's dim roundings and a few more (the two scales, the change of base); fp32 queries are held
    to 2^-22 of a value or 2^-38 of the row's largest.  A weight is off by the score's error in the exponent, by 4 u of
    the exponential, and held to 2^-15 for 16-bit activations and 2^-21 for fp32 ones (a scale of the value
    among its factors).  Numerator and denominator are sums of n weighted values, and of what was joined of them."""
    q64 = t64(q)
    kk, vv = values(k, ks), values(v, vs)
    n_pages, n_kv, page, dim = k.shape
    rows, heads, _ = q64.shape
    pages, lens = pages.cpu(), lens.cpu().reshape(len(pages), -1)
    n_new = lens.shape[1]
    held = 2.0 ** -21 if dtype == torch.float32 else 2.0 ** -15
    out, bound = torch.zeros_like(q64), torch.zeros_like(q64)
    lse, lse_bound = torch.full((rows, heads), -math.inf, dtype=D), torch.zeros((rows, heads), dtype=D)
    for r in range(rows):
        s, t = divmod(r, n_new)
        n = min(int(lens[s, t]), pages.shape[1] * page)
        if n <= 0:
            continue
        p, o, ok = gathered(pages[s], n, page, n_pages)
        if not bool(ok.any()):
            continue
        p, o = p[ok], o[ok]
        for h in range(heads):
            kr, vr, qr = kk[p, h * n_kv // heads, o], vv[p, h * n_kv // heads, o], q64[r, h]
            sc = scale * (kr @ qr)
            size = kr.abs() @ qr.abs()
            es = abs(scale) * ((dim + 8) * U32 * size + (2.0 ** -22 * size + 2.0 ** -38 * qr.abs().max() * kr.abs().sum(1)
                                                         if dtype == torch.float32 else 0.0)) + 4 * U32 * sc.abs()
            w = torch.softmax(sc, 0)
            e = 2 * float(es.max()) + 16 * U32 + 4 * U32 * float(sc.abs().max())
            out[r, h] = w @ vr
            bound[r, h] = (w @ vr.abs()) * (e + held + 2 * (len(sc) + 64) * U32)
            lse[r, h] = torch.logsumexp(sc, 0)
            lse_bound[r, h] = e + (len(sc) + 64) * U32 + 4 * U32 * lse[r, h].abs()
    return out, bound, lse, lse_bound

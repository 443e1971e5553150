"""Plain 64-bit forms of the operators of include/hoard_ops.h, on the CPU, and the bounds their results are held to.

Bounds count roundings.  u(t) = finfo(t).eps / 2 is half a step of type t relative to a value.  A result stored in type
t is off by u(t) of itself; a sum of n terms in 32 bits is off by at most n * u(f32) of the sum of the terms'
magnitudes in any order (each partial sum rounds once and is no larger than that), and each factor of a term adds a u.
"""
import torch

U32 = torch.finfo(torch.float32).eps / 2


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest step, for results below the normal range."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, bound, what):
    """got within bound (elementwise, float64) of want."""
    got = got.detach().cpu().to(torch.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off[bad].max()), float((off / bound.clamp(min=1e-300)).nan_to_num(0).max()))


# -- 4-bit products ---------------------------------------------------------------

def dense(codes, scales, zeros):
    """float64 weights of codes [..., rows, cols/2]."""
    c = codes.cpu().to(torch.int64)
    q = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).to(torch.float64)
    s = scales.cpu().to(torch.float64)
    group = q.shape[-1] // s.shape[-1]
    z = zeros.cpu().to(torch.float64) if zeros is not None else torch.full_like(s, 8.0)
    return (q - z.repeat_interleave(group, -1)) * s.repeat_interleave(group, -1), q, z.repeat_interleave(group, -1), \
        s.repeat_interleave(group, -1)


def product(x, m, e):
    """(value, bound before storing) of x [r, cols] times matrix e of m = (codes, scales, zeros).

    The kernels may form a group's sum of (B + q) x less (B + z) times the sum of x, B up to 16 for fp32 activations
    (split into at most three parts, so three terms a column) and f16, 128 for bf16: both sums, of magnitudes up to
    (B + q) |x| and (B + z) |x|, round once a term and a few times more, their difference is scaled, and the groups'
    sums, now of magnitudes |q - z| |s| |x|, are added."""
    if m[0].dim() == 3:
        m = tuple(t[e] if t is not None else None for t in m)
    w, q, z, s = dense(*m)
    groups = m[1].shape[-1]
    group = q.shape[-1] // groups
    bias, terms = {torch.float32: (16, 3), torch.bfloat16: (128, 1), torch.float16: (16, 1)}[x.dtype]
    x = x.cpu().to(torch.float64)
    inner = x.abs() @ ((2 * bias + q + z) * s.abs()).t()
    outer = x.abs() @ w.abs().t()
    return x @ w.t(), ((terms * group + 8) * inner + (groups + 16) * outer) * U32


def swiglu(g, bg, up, bu):
    """silu(g) * up and its bound, given those of g and up: silu' lies within [-0.1, 1.1]; e^-g, the sum, the quotient
    and the product round about 6 times, e^-g itself by 2 steps (of a quotient no larger than |g|)."""
    s = g / (1.0 + torch.exp(-g))
    return s * up, 1.1 * bg * up.abs() + s.abs() * bu + 1.1 * bg * bu + 10 * U32 * (s * up).abs() + 2 * U32 * g.abs() * up.abs()


def stored(value, bound, dtype):
    """The bound once the value is rounded to dtype."""
    return bound + u(dtype) * (value.abs() + bound) + tiny(dtype)


# -- pairs ------------------------------------------------------------------------

def sort_pairs(ids, n_expert):
    flat = ids.cpu().reshape(-1).tolist()
    rows = [[] for _ in range(n_expert)]
    for p, e in enumerate(flat):
        if 0 <= e < n_expert:
            rows[e].append(p)
    offsets, order = [0], []
    for r in rows:
        order += r
        offsets.append(len(order))
    place = [-1] * len(flat)
    for row, p in enumerate(order):
        place[p] = row
    order += [-1] * (len(flat) - len(order))
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return t(place).view(ids.shape), t(order), t(offsets)


# -- norms ------------------------------------------------------------------------

def norm(x, eps):
    return x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + eps)

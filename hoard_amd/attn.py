"""The operators of a layer's attention half (include/hoard_attn.h) on torch tensors.

As in ops.py torch allocates the outputs and workspaces and hands over its current stream on the tensors' device;
every computation is a call into libhoard_moe.so, asynchronous on that stream.  A tensor given to write to lies apart
from the inputs except where said, a tensor that wants a gradient is refused where gradients are recorded.  Heads are
[tokens, heads, head_dim] tensors whose rows of heads are dense and may be columns of wider rows, as the parts of one
projection's output are.

A layer's attention half for one new token of each of N sequences (qkv [N, (n_q + 2 n_kv) * dim] from q4_matmul):

    q, k, v = split_heads(qkv, n_q, n_kv, dim)
    st = heads_forward(q, k, v, w_q=wq, w_k=wk, rope=Rope(pos, freq), eps=eps, cache=cache, slots=slots)
    o = attn_decode(st.q_out, cache, pages, lens).out       # lens int32 [N]: keys, the new one included
    b = q4_matmul(o.view(N, n_q * dim), w_o)

A verify step takes n_new tokens a sequence: q [N * n_new, n_q, dim], lens [N, n_new].  For training heads_forward is
called without a cache and with want_stats, and heads_backward gives the gradients.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import (ROPE_HALVES, ROPE_PAIRS, TYPE_BF16, TYPE_F16, TYPE_I8, AttnArgs, HeadsArgs, HeadsGrads, KvCache, check,
               load_library)
from .ops import _TYPES, _need, _On, _p, _tensor, _type

_CACHE_TYPES = {torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16, torch.int8: TYPE_I8}


def _heads(name: str, t, shape=None, dtype=None, device=None) -> int:
    """Checks of [tokens, heads, dim] with dense rows of heads; the distance from a token's row to the next."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 3, f"{name}: not a device tensor of tokens, heads and values")
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name}: wants a gradient, which this call does not record")
    _need(shape is None or tuple(t.shape) == tuple(shape), f"{name}: shape {tuple(t.shape)}, wanted {shape}")
    _need(dtype is None or t.dtype == dtype, f"{name}: {t.dtype}, wanted {dtype}")
    _need(device is None or t.device == device, f"{name}: on {t.device}, wanted {device}")
    n, h, d = t.shape
    row = h * d
    if t.numel() == 0 or n == 1 and t.is_contiguous():
        return row
    _need((d == 1 or t.stride(2) == 1) and (h == 1 or t.stride(1) == d), f"{name}: heads of a token are not dense")
    if n == 1:
        return row
    _need(t.stride(0) >= row, f"{name}: rows overlap")
    return t.stride(0)


def _span(t):
    size = t.element_size()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + last * size


def _apart(a, b) -> bool:
    """Whether two tensors share no element: their spans are apart, or they are different columns of the same rows."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0 or not a.numel() or not b.numel():
        return True
    if a.dim() != 3 or b.dim() != 3:
        return False
    step = a.stride(0) * a.element_size()
    if step != b.stride(0) * b.element_size():
        return False
    row = lambda t: t.shape[1] * t.shape[2] * t.element_size()  # noqa: E731
    between = (b0 - a0) % step
    return between >= row(a) and between + row(b) <= step


def _written(name: str, t, inputs=(), or_same=None) -> None:
    """A tensor to write to, its own checks done: apart from the inputs, but for one of them, `or_same`, whose whole it may
    be.  Another input that is the same tensor goes on being read, by other waves.  Its version counts the write:
    autograd refuses a gradient that needs what it held."""
    for i in inputs:
        if isinstance(i, torch.Tensor):
            if i is or_same and i.data_ptr() == t.data_ptr() and i.stride() == t.stride() and i.shape == t.shape:
                or_same = None
                continue
            _need(_apart(t, i), f"{name}: overlaps an input")
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


# -- the cache ------------------------------------------------------------------------


class KVCache:
    """Keys and values [n_pages, n_kv_heads, page, head_dim] as float16, bfloat16 or, with scales float32 [n_pages,
    n_kv_heads, page], int8 codes.  Slot s is place s % page of page s // page.  To be written to, its tensors lie apart
    from each other."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _tensor("k", k)
        _need(k.dim() == 4 and k.numel() > 0 and k.dtype in _CACHE_TYPES, f"k: {k.dtype} of shape {tuple(k.shape)}")
        _tensor("v", v, k.shape, k.dtype, k.device)
        _need((k.dtype == torch.int8) == (k_scale is not None) == (v_scale is not None), "scales go with int8 codes")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t is not None:
                _tensor(name, t, k.shape[:3], torch.float32, k.device)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.page, self.head_dim = k.shape
        self.device = k.device
        self.desc = KvCache(_p(k), _p(v), _p(k_scale), _p(v_scale), _CACHE_TYPES[k.dtype], self.n_pages, self.page,
                            self.n_kv_heads, self.head_dim)

    @classmethod
    def new(cls, n_pages: int, page: int, n_kv_heads: int, head_dim: int, dtype=torch.bfloat16, device="cuda"):
        """A cache of zeros."""
        new = lambda *shape, t: torch.zeros(shape, dtype=t, device=device)  # noqa: E731
        shape = (n_pages, n_kv_heads, page)
        scales = [new(*shape, t=torch.float32) if dtype == torch.int8 else None for _ in range(2)]
        return cls(new(*shape, head_dim, t=dtype), new(*shape, head_dim, t=dtype), *scales)

    def _tensors(self):
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None]

    def _write(self, inputs) -> None:
        tensors = self._tensors()
        for n, t in enumerate(tensors):
            _written("cache", t, (*inputs, *tensors[:n]))


def _slots(slots, n, device):
    _tensor("slots", slots, (n,), torch.int32, device)


def _cache(cache):
    _need(isinstance(cache, KVCache), "cache: no KVCache")


def kv_write(cache: KVCache, slots, k=None, v=None) -> None:
    """Rows of k and v [tokens, n_kv_heads, head_dim] to their slots int32 [tokens]; a slot outside the cache drops its
    token, the others must be distinct."""
    _cache(cache)
    first = k if k is not None else v
    _need(isinstance(first, torch.Tensor) and first.dim() == 3, "neither k nor v")
    n, dtype = first.shape[0], first.dtype
    shape = (n, cache.n_kv_heads, cache.head_dim)
    strides = [_heads(name, t, shape, dtype, cache.device) if t is not None else 0 for name, t in (("k", k), ("v", v))]
    _slots(slots, n, cache.device)
    dt = _type("k" if k is not None else "v", first)
    cache._write((k, v, slots))
    with _On(cache.device) as stream:
        check(load_library().hoard_kv_write(ctypes.byref(cache.desc), dt, n, _p(slots), _p(k), strides[0], _p(v),
                                            strides[1], stream))


def kv_read(cache: KVCache, slots, dtype=None, *, k=None, v=None):
    """(k, v) [tokens, n_kv_heads, head_dim] of the slots int32 [tokens], into the tensors given or new ones of `dtype`
    (the cache's; bfloat16 for codes).  Rows of a slot outside the cache are left as they are (zero in new tensors)."""
    _cache(cache)
    _need(isinstance(slots, torch.Tensor) and slots.dim() == 1, "slots: no vector")
    n = slots.shape[0]
    _slots(slots, n, cache.device)
    given = k if k is not None else v
    _need(given is None or isinstance(given, torch.Tensor), "k or v: no tensor")
    dtype = dtype or (given.dtype if given is not None else torch.bfloat16 if cache.k.dtype == torch.int8 else cache.k.dtype)
    _need(dtype in _TYPES, f"{dtype} is no activation type")
    shape, strides, out = (n, cache.n_kv_heads, cache.head_dim), [], []
    for name, t in (("k", k), ("v", v)):
        if t is None:
            t = torch.zeros(shape, dtype=dtype, device=cache.device)
            strides.append(shape[1] * shape[2])
        else:
            strides.append(_heads(name, t, shape, dtype, cache.device))
            _written(name, t, (*cache._tensors(), slots, *out))
        out.append(t)
    with _On(cache.device) as stream:
        check(load_library().hoard_kv_read(ctypes.byref(cache.desc), _TYPES[dtype], n, _p(slots), _p(out[0]), strides[0],
                                           _p(out[1]), strides[1], stream))
    return tuple(out)


# -- heads normed and rotated -----------------------------------------------------------


class Rope(NamedTuple):
    """Positions int32 [tokens] or [axes, tokens]; freq float64 [rot_dim / 2], radians a position; axis uint8
    [rot_dim / 2], the axis of each pair (None: the first); pairs: value 2i turns with 2i + 1, not i with
    i + rot_dim / 2."""
    pos: torch.Tensor
    freq: torch.Tensor
    axis: torch.Tensor | None = None
    pairs: bool = False


def rope_freq(rot_dim: int, base: float, device="cuda"):
    """base ** (-2i / rot_dim), float64 [rot_dim / 2]."""
    return base ** (-2.0 * torch.arange(rot_dim // 2, dtype=torch.float64, device=device) / rot_dim)


def split_heads(qkv, n_q: int, n_kv: int, dim: int):
    """The q, k and v heads of a fused projection's rows [tokens, (n_q + 2 n_kv) * dim], as views."""
    _need(isinstance(qkv, torch.Tensor) and qkv.dim() == 2 and qkv.shape[1] == (n_q + 2 * n_kv) * dim,
          "qkv: no matrix of that many heads")
    return torch.split(qkv.view(qkv.shape[0], n_q + 2 * n_kv, dim), [n_q, n_kv, n_kv], dim=1)


class HeadsState(NamedTuple):
    q_out: torch.Tensor | None
    k_out: torch.Tensor | None
    stats: torch.Tensor | None  # float32 [tokens, n_q + n_kv], for heads_backward


class HeadsGradients(NamedTuple):
    dq: torch.Tensor | None
    dk: torch.Tensor | None
    dw_q: torch.Tensor | None
    dw_k: torch.Tensor | None


def _fill_heads(q, k, v, w_q, w_k, rope, eps, w_offset, cache):
    """(HeadsArgs without outputs, tokens, dim, dtype, device) after the checks that both directions share."""
    first = next((t for t in (q, k, v) if t is not None), None)
    _need(isinstance(first, torch.Tensor) and first.dim() == 3, "neither q, k nor v")
    n, _, d = first.shape
    dtype, device = first.dtype, first.device
    a = HeadsArgs(type=_type("heads", first), n_tokens=n, head_dim=d, n_axes=1, eps=eps, w_offset=w_offset)
    if q is not None:
        a.q_stride, a.n_q_heads, a.q = _heads("q", q, (n, q.shape[1], d), dtype, device), q.shape[1], _p(q)
    kv = k if k is not None else v
    _need(kv is None or isinstance(kv, torch.Tensor) and kv.dim() == 3, "k or v: no heads")
    heads = kv.shape[1] if kv is not None else cache.n_kv_heads if cache is not None else 0
    a.n_kv_heads = heads
    if k is not None:
        a.k_stride, a.k = _heads("k", k, (n, heads, d), dtype, device), _p(k)
    if v is not None:
        a.v_stride, a.v = _heads("v", v, (n, heads, d), dtype, device), _p(v)
    for name, w in (("w_q", w_q), ("w_k", w_k)):
        if w is not None:
            _tensor(name, w, (d,), torch.float32, device)
            setattr(a, name, _p(w))
    if rope is not None:
        _need(isinstance(rope, Rope), "rope: no Rope")
        _need(isinstance(rope.freq, torch.Tensor) and rope.freq.dim() == 1, "freq: no vector")
        _tensor("freq", rope.freq, None, torch.float64, device)
        _need(isinstance(rope.pos, torch.Tensor) and rope.pos.dim() in (1, 2), "pos: no vector or matrix")
        axes = rope.pos.shape[0] if rope.pos.dim() == 2 else 1
        _tensor("pos", rope.pos, (axes, n) if rope.pos.dim() == 2 else (n,), torch.int32, device)
        if rope.axis is not None:
            _tensor("axis", rope.axis, rope.freq.shape, torch.uint8, device)
        a.rot_dim, a.rope, a.n_axes = 2 * rope.freq.shape[0], ROPE_PAIRS if rope.pairs else ROPE_HALVES, axes
        a.pos, a.freq, a.axis = _p(rope.pos), _p(rope.freq), _p(rope.axis)
    return a, n, d, dtype, device


def heads_forward(q=None, k=None, v=None, *, w_q=None, w_k=None, rope: Rope | None = None, eps: float = 1e-6,
                  w_offset: float = 0.0, cache: KVCache | None = None, slots=None, q_out=None, k_out=None,
                  want_stats: bool = False) -> HeadsState:
    """Each head of q and k normed by its weight (w_offset + w_q, w_k [head_dim]; None: not normed) and rotated.  With a
    cache the rotated k and v as it is go to slots int32 [tokens], and k_out is only written if given; without one it
    is a new tensor.  q_out may be q, and k_out k."""
    if cache is not None:
        _cache(cache)
    a, n, d, dtype, device = _fill_heads(q, k, v, w_q, w_k, rope, eps, w_offset, cache)
    inputs = (q, k, v, w_q, w_k, slots) + (tuple(rope[:3]) if rope is not None else ())
    if cache is not None:
        _need(cache.device == device, "cache: on another device")
        _need(slots is not None, "slots: wanted with a cache")
        _slots(slots, n, device)
        a.cache, a.slots = ctypes.addressof(cache.desc), _p(slots)
    else:
        _need(slots is None and v is None, "slots or v without a cache")
    _need(q_out is None or q is not None, "q_out: without q")
    _need(k_out is None or k is not None, "k_out: without k")
    outs = []
    for name, x, t, same in (("q_out", q, q_out, q), ("k_out", k, k_out, k)):
        if x is not None and t is None and (name == "q_out" or cache is None):
            t = torch.empty(x.shape, dtype=dtype, device=device)
        elif t is not None:
            _heads(name, t, x.shape, dtype, device)
            _written(name, t, (*inputs, *outs), same)
        if t is not None:
            setattr(a, name + "_stride", _heads(name, t))
            setattr(a, name, _p(t))
        outs.append(t)
    if cache is not None:
        cache._write((*inputs, *outs))
    stats = torch.ones((n, a.n_q_heads + a.n_kv_heads), dtype=torch.float32, device=device) if want_stats else None
    a.stats = _p(stats)
    with _On(device) as stream:
        check(load_library().hoard_heads_forward(ctypes.byref(a), stream))
    return HeadsState(*outs, stats)


def heads_backward(dq_out=None, dk_out=None, *, q=None, k=None, w_q=None, w_k=None, rope: Rope | None = None, stats=None,
                   eps: float = 1e-6, w_offset: float = 0.0, dq=None, dk=None) -> HeadsGradients:
    """Gradients of heads_forward given those of q_out and k_out (either may be None): of q and k, and of the weights
    that are given, which need the forward call's q (k) and stats, the columns of all of its heads.  dq may be dq_out, and
    dk dk_out."""
    given = [t for t in (dq_out, dk_out) if t is not None]
    _need(len(given) > 0, "neither dq_out nor dk_out")
    for name, x, dx in (("q", q, dq_out), ("k", k, dk_out)):
        _need(dx is None or isinstance(dx, torch.Tensor) and dx.dim() == 3, f"d{name}_out: no heads")
    _need((w_q is None or dq_out is None or q is not None) and (w_k is None or dk_out is None or k is not None),
          "the heads that were normed: wanted")
    # without a norm the heads themselves are not read: their gradients stand for their shape
    use_q = q if q is not None else dq_out
    use_k = k if k is not None else dk_out
    a, n, d, dtype, device = _fill_heads(use_q, use_k, None, w_q, w_k, rope, eps, w_offset, None)
    if stats is not None:
        _need(isinstance(stats, torch.Tensor) and stats.dim() == 2, "stats: no matrix")
        if use_q is None:  # the columns of the heads that are not given
            a.n_q_heads = max(stats.shape[1] - a.n_kv_heads, 0)
        if use_k is None:
            a.n_kv_heads = max(stats.shape[1] - a.n_q_heads, 0)
        _tensor("stats", stats, (n, a.n_q_heads + a.n_kv_heads), torch.float32, device)
        a.stats = _p(stats)
    _need(stats is not None or (w_q is None and w_k is None), "stats: heads_forward was called without want_stats")
    g, outs = HeadsGrads(), []
    inputs = [dq_out, dk_out, q if w_q is not None else None, k if w_k is not None else None, w_q, w_k, stats]
    inputs += list(rope[:3]) if rope is not None else []
    for name, x, dx, to in (("q", use_q, dq_out, dq), ("k", use_k, dk_out, dk)):
        _need(to is None or dx is not None, f"d{name}: without d{name}_out")
        if dx is None:
            outs.append(None)
            continue
        setattr(a, name + "_out_stride", _heads(f"d{name}_out", dx, x.shape, dtype, device))
        want = x.shape[1] * x.shape[2]
        if to is None:
            to = torch.empty(x.shape, dtype=dtype, device=device)
        else:
            _heads(f"d{name}", to, x.shape, dtype, device)
            _written(f"d{name}", to, (*inputs, *outs), dx)
        setattr(g, f"d{name}_stride", _heads(f"d{name}", to))
        setattr(g, "d" + name + "_out", _p(dx))
        setattr(g, "d" + name, _p(to))
        outs.append(to)
    dw_q = torch.empty_like(w_q) if w_q is not None and dq_out is not None else None
    dw_k = torch.empty_like(w_k) if w_k is not None and dk_out is not None else None
    g.dw_q, g.dw_k = _p(dw_q), _p(dw_k)
    lib, need = load_library(), ctypes.c_size_t()
    check(lib.hoard_heads_workspace(ctypes.byref(a), ctypes.byref(need)))
    work = torch.empty((need.value + 3) // 4, dtype=torch.float32, device=device)
    with _On(device) as stream:
        check(lib.hoard_heads_backward(ctypes.byref(a), ctypes.byref(g), _p(work), need.value, stream))
    return HeadsGradients(*outs, dw_q, dw_k)


# -- attention ------------------------------------------------------------------------------


class Attention(NamedTuple):
    out: torch.Tensor        # [sequences * n_new, n_q_heads, head_dim]
    lse: torch.Tensor | None  # float32 [sequences * n_new, n_q_heads]


def attn_decode(q, cache: KVCache, pages, lens, *, scale: float | None = None, out=None, want_lse: bool = False) -> Attention:
    """softmax(scale <q, k>) v over the cache for each new token: q [sequences * n_new, n_q_heads, head_dim], pages int32
    [sequences, max_pages], lens int32 [sequences] or [sequences, n_new]: the keys that each sees (0: its row is 0).
    scale: head_dim ** -0.5 by default.  lse: the logarithm of the sum of exp(scale <q, k>), to join results over
    different keys by."""
    _cache(cache)
    _need(isinstance(lens, torch.Tensor) and lens.dim() in (1, 2), "lens: no vector or matrix")
    _tensor("lens", lens, None, torch.int32, cache.device)
    n_seq, n_new = lens.shape[0], lens.shape[1] if lens.dim() == 2 else 1
    _need(isinstance(pages, torch.Tensor) and pages.dim() == 2, "pages: no matrix")
    _tensor("pages", pages, (n_seq, pages.shape[1]), torch.int32, cache.device)
    _need(isinstance(q, torch.Tensor) and q.dim() == 3, "q: no heads")
    stride = _heads("q", q, (n_seq * n_new, q.shape[1], cache.head_dim), None, cache.device)
    dt = _type("q", q)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _tensor("out", out, q.shape, q.dtype, q.device)
        _written("out", out, (q, pages, lens, *cache._tensors()))
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if want_lse else None
    a = AttnArgs(dt, n_seq, n_new, q.shape[1], pages.shape[1], cache.head_dim ** -0.5 if scale is None else scale, stride,
                 _p(q), _p(pages), _p(lens), _p(out), _p(lse))
    lib, need, c = load_library(), ctypes.c_size_t(), ctypes.byref(cache.desc)
    check(lib.hoard_attn_workspace(c, ctypes.byref(a), ctypes.byref(need)))
    work = torch.empty((need.value + 3) // 4, dtype=torch.float32, device=q.device)
    with _On(q.device) as stream:
        check(lib.hoard_attn_decode(c, ctypes.byref(a), _p(work), need.value, stream))
    return Attention(out, lse)

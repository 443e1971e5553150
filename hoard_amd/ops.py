"""The operators around the expert stage (include/hoard_ops.h) on torch tensors.

torch allocates the outputs and workspaces and hands over its current stream on
the tensors' device; every computation is a call into libhoard_moe.so.  Calls are
asynchronous on that stream.  Tensors are dense device tensors of one device, and
one given to write to lies apart from the inputs except where said (anything else
raises HoardError); a tensor made on another stream is the caller's to order, as
with any torch operator.

A layer whose experts are 4-bit codes, M tokens, k of E experts each:

    st = norm_forward(r, w_pre=w, eps=eps)                  # h = norm(r)
    s = sort_pairs(ids, E)                                  # ids, w from the caller's router
    xs = sort_gather(st.h, s.place)
    hid = q4_matmul(xs, gate, up=up, offsets=s.offsets)     # silu(gate x) * (up x)
    y = q4_matmul(hid, down, offsets=s.offsets)
    b = sort_combine(y, s.place, w)
    st = norm_forward(r, b=b, w_post=w1, w_pre=w2, eps=eps) # residual, next block's h

Gradients: sort_combine(dxs, place) is sort_gather's, sort_combine_grad and
norm_backward are those of sort_combine and norm_forward.  The 4-bit products
have none (their weights are constants, and they serve inference), nor has the
stage: a chain through the experts takes the caller's own gradient there.  No call
records itself for autograd: where gradients are recorded, a tensor that wants one is
refused (detach it, or call under torch.no_grad(), and run the backward calls yourself).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import (ERR_INVALID, GATE_CHANNEL, GATE_FULL, GATE_NONE, GATE_TOKEN, TYPE_BF16, TYPE_F16, TYPE_F32, HoardError,
               NormArgs, NormGrads, Q4Matrix, check, load_library)

_TYPES = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise HoardError(ERR_INVALID, what)


def _tensor(name: str, t, shape=None, dtype=None, device=None) -> None:
    _need(isinstance(t, torch.Tensor) and t.is_cuda and t.is_contiguous(), f"{name}: not a dense device tensor")
    _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name}: wants a gradient, which this call does not record")
    _need(shape is None or tuple(t.shape) == tuple(shape), f"{name}: shape {tuple(t.shape)}, wanted {shape}")
    _need(dtype is None or t.dtype == dtype, f"{name}: {t.dtype}, wanted {dtype}")
    _need(device is None or t.device == device, f"{name}: on {t.device}, wanted {device}")


def _given(name: str, t, shape, dtype, device, inputs=(), or_same=None) -> None:
    """Checks of a tensor to write to: apart from the call's inputs, or all of `or_same`.  Its version counts the write:
    autograd refuses a gradient that needs what it held."""
    _tensor(name, t, shape, dtype, device)
    first, last = t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()
    for i in (*inputs, or_same):
        if not isinstance(i, torch.Tensor) or (i is or_same and i.data_ptr() == first):
            continue  # what is no tensor is refused by its own checks
        _need(last <= i.data_ptr() or i.data_ptr() + i.numel() * i.element_size() <= first, f"{name}: overlaps an input")
    if not t.is_inference():  # one made in inference mode has no version, and autograd keeps none
        torch.autograd.graph.increment_version(t)


def _type(name: str, t) -> int:
    _need(t.dtype in _TYPES, f"{name}: {t.dtype} is no activation type")
    return _TYPES[t.dtype]


def _p(t):
    # an empty tensor has no address: any stands for one that is there and never read
    return None if t is None else t.data_ptr() or 256


class _On:
    """The tensors' device made current, and torch's current stream on it."""

    def __init__(self, device):
        self.guard = torch.cuda.device(device)

    def __enter__(self):
        self.guard.__enter__()
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        return self.guard.__exit__(*exc)


# -- products with 4-bit weights --------------------------------------------------


class Q4Weight:
    """One matrix or a stack of them: codes uint8 [(n_mat,) rows, cols/2] (byte j: code 2j in its low half, 2j+1 in
    its high half), scales [(n_mat,) rows, cols/group] f32, f16 or bf16, zeros uint8 of the same shape or None (8):
    weight = scale * (code - zero)."""

    def __init__(self, codes, scales, zeros=None):
        _tensor("codes", codes, dtype=torch.uint8)
        _need(codes.dim() in (2, 3) and codes.numel() > 0, f"codes: shape {tuple(codes.shape)}")
        _tensor("scales", scales, device=codes.device)
        _need(scales.shape[:-1] == codes.shape[:-1] and scales.shape[-1] > 0, f"scales: shape {tuple(scales.shape)}")
        if zeros is not None:
            _tensor("zeros", zeros, scales.shape, torch.uint8, codes.device)
        self.codes, self.scales, self.zeros = codes, scales, zeros
        self.rows, self.cols = codes.shape[-2], 2 * codes.shape[-1]
        self.n_mat = codes.shape[0] if codes.dim() == 3 else 1
        _need(self.cols % scales.shape[-1] == 0, f"{self.cols} columns in {scales.shape[-1]} groups")
        self.desc = Q4Matrix(_p(codes), _p(scales), _p(zeros), self.rows, self.cols, self.cols // scales.shape[-1],
                             self.n_mat, _type("scales", scales))


def q4_matmul(x, w: Q4Weight, up: Q4Weight | None = None, *, ids=None, offsets=None, out=None):
    """Rows of x [rows, cols] times w transposed, in x's type; with up silu(w x) * (up x).

    ids int32 [tokens] or [tokens, k]: row by row the matrix to take, x [tokens, cols] being shared by a token's k
    (out [tokens * k, w.rows]).  offsets int32 [n_mat + 1]: rows sorted by matrix, as sort_pairs gives them."""
    _tensor("x", x)
    dt = _type("x", x)
    _need(x.dim() == 2 and x.shape[1] == w.cols, f"x: shape {tuple(x.shape)} for {w.cols} columns")
    _need(w.codes.device == x.device and (up is None or up.codes.device == x.device), "weights on another device")
    _need(ids is None or offsets is None, "ids and offsets are two forms")
    n_rows, share = x.shape[0], 1
    if ids is not None:
        _tensor("ids", ids, dtype=torch.int32, device=x.device)
        _need(ids.dim() in (1, 2) and ids.shape[0] == x.shape[0], f"ids: shape {tuple(ids.shape)} for {x.shape[0]} rows")
        share = ids.shape[1] if ids.dim() == 2 else 1
        _need(share > 0, "ids: no column")
        n_rows = x.shape[0] * share
    if offsets is not None:
        _tensor("offsets", offsets, (w.n_mat + 1,), torch.int32, x.device)
    if out is None:
        out = torch.empty((n_rows, w.rows), dtype=x.dtype, device=x.device)
    else:
        _given("out", out, (n_rows, w.rows), x.dtype, x.device, (x, ids, offsets))
    lib, a, b = load_library(), ctypes.byref(w.desc), ctypes.byref(up.desc) if up is not None else None
    with _On(x.device) as stream:
        if ids is not None:
            check(lib.hoard_q4_matmul_ids(a, b, dt, n_rows, _p(x), share, _p(ids), _p(out), stream))
        elif offsets is not None:
            check(lib.hoard_q4_matmul_sorted(a, b, dt, n_rows, _p(x), _p(offsets), _p(out), stream))
        else:
            check(lib.hoard_q4_matmul(a, b, dt, n_rows, _p(x), _p(out), stream))
    return out


# -- pairs sorted by expert, and back ---------------------------------------------


class SortedPairs(NamedTuple):
    place: torch.Tensor    # int32 [tokens, k]: the sorted row of each pair, -1 where its id is no expert
    order: torch.Tensor    # int32 [tokens * k]: the pair t * k + j at each sorted row, -1 behind the last
    offsets: torch.Tensor  # int32 [n_expert + 1]: the rows of expert e are offsets[e] .. offsets[e + 1] - 1


def sort_pairs(ids, n_expert: int) -> SortedPairs:
    """The pairs of ids int32 [tokens, k] sorted by expert, pairs of one expert in their order."""
    _tensor("ids", ids, dtype=torch.int32)
    _need(ids.dim() == 2, f"ids: shape {tuple(ids.shape)}")
    m, k = ids.shape
    lib, need = load_library(), ctypes.c_size_t()
    check(lib.hoard_sort_workspace(m, k, n_expert, ctypes.byref(need)))
    new = lambda *size: torch.empty(size, dtype=torch.int32, device=ids.device)  # noqa: E731
    place, order, offsets, work = new(m, k), new(m * k), new(n_expert + 1), new((need.value + 3) // 4)
    with _On(ids.device) as stream:
        check(lib.hoard_sort_pairs(m, k, n_expert, _p(ids), _p(place), _p(order), _p(offsets), _p(work), need.value,
                                   stream))
    return SortedPairs(place, order, offsets)


def _rows(name, x, place, w, rows):
    """The checks that the row operators share: (type, tokens, k, n)."""
    _tensor(name, x)
    _need(x.dim() == 2 and x.shape[1] > 0, f"{name}: shape {tuple(x.shape)}")
    _tensor("place", place, dtype=torch.int32, device=x.device)
    _need(place.dim() == 2, f"place: shape {tuple(place.shape)}")
    m, k = place.shape
    _need(x.shape[0] == rows(m, k), f"{name}: {x.shape[0]} rows for places of shape {tuple(place.shape)}")
    if w is not None:
        _tensor("w", w, (m, k), torch.float32, x.device)
    return _type(name, x), m, k, x.shape[1]


def sort_gather(x, place, w=None, *, out=None):
    """x [tokens, n] laid out by sorted row, [tokens * k, n], times w [tokens, k] if given.  Rows that no pair names
    are left as they are (not initialised in a new tensor)."""
    dt, m, k, n = _rows("x", x, place, w, lambda m, k: m)
    if out is None:
        out = torch.empty((m * k, n), dtype=x.dtype, device=x.device)
    else:
        _given("out", out, (m * k, n), x.dtype, x.device, (x, place, w))
    with _On(x.device) as stream:
        check(load_library().hoard_sort_gather(dt, m, k, n, _p(x), _p(place), _p(w), _p(out), stream))
    return out


def sort_combine(y, place, w=None, res=None, *, out=None):
    """res + sum over j of w[t, j] * y[place[t, j]] (w None: ones, the gradient of sort_gather); out may be res."""
    dt, m, k, n = _rows("y", y, place, w, lambda m, k: m * k)
    if res is not None:
        _tensor("res", res, (m, n), y.dtype, y.device)
    if out is None:
        out = torch.empty((m, n), dtype=y.dtype, device=y.device)
    else:
        _given("out", out, (m, n), y.dtype, y.device, (y, place, w), res)
    with _On(y.device) as stream:
        check(load_library().hoard_sort_combine(dt, m, k, n, _p(y), _p(place), _p(w), _p(res), _p(out), stream))
    return out


def sort_combine_grad(dout, y, place, w, *, dy=None):
    """(dy, dw) of sort_combine; rows of dy that no pair names are left as they are (zero in a new tensor); dy may be y."""
    dt, m, k, n = _rows("y", y, place, w, lambda m, k: m * k)
    _need(w is not None, "w: wanted")
    _tensor("dout", dout, (m, n), y.dtype, y.device)
    if dy is None:
        dy = torch.zeros_like(y)
    else:
        _given("dy", dy, y.shape, y.dtype, y.device, (dout, place, w), y)
    dw = torch.empty_like(w)
    with _On(y.device) as stream:
        check(load_library().hoard_sort_combine_grad(dt, m, k, n, _p(dout), _p(y), _p(place), _p(w), _p(dy), _p(dw),
                                                     stream))
    return dy, dw


# -- norms around a block -----------------------------------------------------------


class NormState(NamedTuple):
    """What norm_forward gives."""
    r_out: torch.Tensor         # the residual stream after the block (r itself without b)
    h: torch.Tensor | None      # the next block's input
    stats: torch.Tensor | None  # f32 [rows, 2], for norm_backward


class NormGradients(NamedTuple):
    dr: torch.Tensor
    db: torch.Tensor | None
    dgate: torch.Tensor | None
    dw_post: torch.Tensor | None
    dw_pre: torch.Tensor | None


def _norm_args(r, b, gate, w_post, w_pre, r_out, h, stats, dtype, eps, scale, w_offset, gate_sigmoid) -> NormArgs:
    _tensor("r", r)
    _need(r.dim() == 2, f"r: shape {tuple(r.shape)}")
    m, n = r.shape
    _need(dtype in _TYPES, f"{dtype} is no activation type")
    if b is not None:
        _tensor("b", b, (m, n), dtype, r.device)
    kind = GATE_NONE
    if gate is not None:
        _need(isinstance(gate, torch.Tensor) and gate.dim() in (1, 2), "gate: no vector or matrix")
        if gate.dim() == 1:
            kind = GATE_CHANNEL
            _tensor("gate", gate, (n,), torch.float32, r.device)
        elif gate.shape[1] == 1:
            kind = GATE_TOKEN
            _tensor("gate", gate, (m, 1), torch.float32, r.device)
        else:
            kind = GATE_FULL
            _tensor("gate", gate, (m, n), dtype, r.device)
    for name, t in (("w_post", w_post), ("w_pre", w_pre)):
        if t is not None:
            _tensor(name, t, (n,), torch.float32, r.device)
    return NormArgs(_TYPES[dtype], _type("r", r), kind, int(bool(gate_sigmoid)), m, n, eps, scale, w_offset, _p(r), _p(b),
                    _p(gate), _p(w_post), _p(w_pre), _p(r_out), _p(h), _p(stats))


def norm_forward(r, b=None, w_post=None, gate=None, w_pre=None, *, eps: float, scale: float = 1.0,
                 w_offset: float = 0.0, gate_sigmoid: bool = False, dtype=None, want_stats: bool = False,
                 r_out=None) -> NormState:
    """c = norm(b) * (w_offset + w_post) (w_post None: b), r_out = r + scale * gate * c, h = norm(r_out) * (w_offset +
    w_pre) (w_pre None: no h), row by row.  gate: f32 [n] a channel's, f32 [rows, 1] a row's, or [rows, n] of b's type,
    behind a sigmoid with gate_sigmoid.  dtype: h's type (default b's, or r's without b).  r_out may be r."""
    dtype = dtype or (b.dtype if b is not None else r.dtype)
    new = lambda shape, t: torch.empty(shape, dtype=t, device=r.device)  # noqa: E731
    if b is None:
        _need(r_out is None, "r_out: without b")
    elif r_out is None:
        r_out = new(r.shape, r.dtype)
    else:
        _given("r_out", r_out, r.shape, r.dtype, r.device, (b, gate, w_post, w_pre), r)
    h = new(r.shape, dtype) if w_pre is not None else None
    stats = new((r.shape[0], 2), torch.float32) if want_stats else None
    a = _norm_args(r, b, gate, w_post, w_pre, r_out, h, stats, dtype, eps, scale, w_offset, gate_sigmoid)
    with _On(r.device) as stream:
        check(load_library().hoard_norm_forward(ctypes.byref(a), stream))
    return NormState(r if b is None else r_out, h, stats)


def norm_backward(state: NormState, dr_out=None, dh=None, b=None, w_post=None, gate=None, w_pre=None, *, eps: float,
                  scale: float = 1.0, w_offset: float = 0.0, gate_sigmoid: bool = False) -> NormGradients:
    """Gradients of norm_forward from its result (called with want_stats) and its arguments: of r, and of b, gate,
    w_post and w_pre as far as they were given.  dr_out, dh: the gradients of r_out and h (None: zero)."""
    r = state.r_out
    _need(state.stats is not None, "stats: norm_forward was called without want_stats")
    _need(dr_out is not None or dh is not None, "neither dr_out nor dh")
    dtype = b.dtype if b is not None else dh.dtype if dh is not None else r.dtype
    a = _norm_args(r, b, gate, w_post, w_pre, r, None, state.stats, dtype, eps, scale, w_offset, gate_sigmoid)
    _tensor("stats", state.stats, (r.shape[0], 2), torch.float32, r.device)
    if dr_out is not None:
        _tensor("dr_out", dr_out, r.shape, r.dtype, r.device)
    if dh is not None:
        _tensor("dh", dh, r.shape, dtype, r.device)
    like = lambda t: torch.empty_like(t) if t is not None else None  # noqa: E731
    out = NormGradients(torch.empty_like(r), like(b), like(gate), like(w_post), like(w_pre) if dh is not None else None)
    g = NormGrads(_p(dr_out), _p(dh), _p(out.dr), _p(out.db), _p(out.dgate), _p(out.dw_post), _p(out.dw_pre))
    lib, need = load_library(), ctypes.c_size_t()
    check(lib.hoard_norm_workspace(ctypes.byref(a), ctypes.byref(need)))
    work = torch.empty((need.value + 3) // 4, dtype=torch.float32, device=r.device)
    with _On(r.device) as stream:
        check(lib.hoard_norm_backward(ctypes.byref(a), ctypes.byref(g), _p(work), need.value, stream))
    return out

"""Bounds on how often a 16-bit result of a 4-bit product may differ from the rounded 64-bit one, and on fp32 products.

A result differs from the rounded exact one where the error of its 32-bit sums carries it over a border between two
values of the type.  Borders lie a step apart, so for errors e of either sign, small beside the step, that happens to a
share E|e| / step of the results, and E|e| is at most the root of their mean square.

A group's sum of q x (and z times its sum of x, where the kernel corrects by it) is formed by instructions of 32 columns
that round their result once; its partial sums are, in the mean square over signs of x, no larger than the whole.  Each
rounding is at most u = 2^-24 of them, and they are independent: u^2 (group / 32) (sum q^2 x^2 + z^2 sum x^2) a group,
scaled by its scale and added over the groups.
"""
import torch

import opsref as R


def expected_over_border(x, m, dtype):
    """(value, the number of results that are expected to differ from the rounded value) for codes summed as they are."""
    w, q, z, s = R.dense(*m)
    group = w.shape[-1] // m[1].shape[-1]
    x = x.cpu().to(torch.float64)
    y = x @ w.t()
    square = (x * x) @ ((q * q + z * z) * s * s).t() * R.U32 ** 2 * (group / 32)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1e-30)))) * torch.finfo(dtype).eps
    return y, float((square.sqrt() / step).clamp(max=1.0).sum())


def allowed(expected):
    """Three deviations above the expected number."""
    return expected + 3.0 * expected ** 0.5


def over_border(got, value):
    got = got.detach().cpu()
    return int((got != value.to(got.dtype)).sum())

"""Bounds on how often a 16-bit result of a 4-bit product may differ from the rounded 64-bit one, and on fp32 products.

A result differs from the rounded exact one where the error of its 32-bit sums carries it over a border between two
values of the type.  Borders lie a step apart, so for errors e of either sign, small beside the step, that happens to a
share E|e| / step of the results, and E|e| is at most the root of their mean square.

A group's sum of q x (and z times its sum of x, where the kernel corrects by it) is formed by instructions of 32 columns
that round their result once; its partial sums are, in the mean square over signs of x, no larger than the whole.  Each
rounding is at most u = 2^-24 of them, and they are independent: u^2 (group / 32) (sum q^2 x^2 + z^2 sum x^2) a group,
scaled by its scale and added over the groups.  With an offset in the codes, q and z are what they are with it.
"""
import torch

import opsref as R


def expected_over_border(x, m, dtype, bias=0):
    """(value, the number of results that are expected to differ from the rounded value) for sums of code + bias."""
    w, q, z, s = R.dense(*m)
    group = w.shape[-1] // m[1].shape[-1]
    x = x.cpu().to(torch.float64)
    y = x @ w.t()
    square = (x * x) @ (((bias + q) ** 2 + (bias + z) ** 2) * s * s).t() * R.U32 ** 2 * (group / 32)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1e-30)))) * torch.finfo(dtype).eps
    return y, float((square.sqrt() / step).clamp(max=1.0).sum())


def allowed(expected):
    """Three deviations above the expected number."""
    return expected + 3.0 * expected ** 0.5


def over_border(got, value):
    got = got.detach().cpu()
    return int((got != value.to(got.dtype)).sum())


# -- fp32 ------------------------------------------------------------------------------
#
# The mean square error of fp32 products, over x of either sign.  The terms (q - z) x s of a group are added with at most
# two roundings a column, each at most u of a partial sum, which is in the mean square no larger than the whole; the
# groups' sums and the parts of a split row round a few times more.  Matrix tiles hold x to 2^-23 of itself, or to 2^-39
# of its group's largest value.  All these errors are independent of each other, so their squares add.

def fp32_product(x, m):
    """(value, the mean square error that each result may have) of x times the matrix m."""
    w, _, _, s = R.dense(*m)
    groups = m[1].shape[-1]
    group = w.shape[-1] // groups
    x = x.cpu().to(torch.float64)
    most = x.abs().view(len(x), groups, group).amax(dim=2).repeat_interleave(group, dim=1)
    held = torch.maximum(2.0 ** -23 * x.abs(), 2.0 ** -39 * most)
    ww = (w * w).t()
    return x @ w.t(), (held * held + (2 * group + groups + 24) * R.U32 ** 2 * x * x) @ ww


def fp32_swiglu(g, vg, up, vu):
    """silu(g) * up and its mean square error: silu' lies within [-0.1, 1.1], and R.swiglu's roundings."""
    s = g / (1.0 + torch.exp(-g))
    own = 10 * R.U32 * (s * up).abs() + 2 * R.U32 * g.abs() * up.abs()
    return s * up, 1.21 * up * up * vg + s * s * vu + 1.21 * vg * vu + own * own


def rms_ratio(got, value, square):
    """The root mean square error of all results, over the one they may have once rounded to fp32."""
    off = got.detach().cpu().to(torch.float64) - value
    return float((off.square().sum() / (square + (R.U32 * value) ** 2).sum()) ** 0.5)

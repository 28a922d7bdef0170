"""Layer norm of rows whose mean is far above their deviation: how far a kernel may be off
that centres the row before it squares it.

A row's sum is formed of at most 32 elements a lane one after the other, 6 steps within a
wave and 16 waves one after the other: DEPTH roundings of 2^-24 of the sum of magnitudes.
With R = mean |h| / deviation and E = (DEPTH + 2) 2^-24 R, a mean is off by at most E
deviations.  The mean square of the centred row is then off by E^2 of the variance and not
by E, since the row without its true mean adds up to zero; so 1 / deviation is off by E^2 / 2
and the (DEPTH + C) 2^-24 of the second sum, its division and its root: 1e-5 with R = 1000.

E[h^2] - mean^2 in place of it is off by roundings of 2^-24 of R^2 variances: some per cent.
"""
from __future__ import annotations

import torch

F32 = 2.0 ** -24
DEPTH = 32 + 6 + 16
C = 16


def rows(T, H, ratio, seed=0):
    """fp32 rows of deviation about 1 around +-ratio."""
    g = torch.Generator().manual_seed(seed)
    sign = torch.where(torch.arange(T) % 2 == 0, 1.0, -1.0)[:, None]
    return torch.randn(T, H, generator=g) + ratio * sign


def one_pass(x, eps=1e-5):
    """The layer norm by E[x^2] - mean^2 in fp32."""
    m = x.mean(1, keepdim=True)
    var = (x * x).mean(1, keepdim=True) - m * m
    return (x - m) / torch.sqrt(var.clamp(min=0) + eps)


def two_pass(x, eps=1e-5):
    c = x - x.mean(1, keepdim=True)
    return c / torch.sqrt((c * c).mean(1, keepdim=True) + eps)


def faults(y, h, h_err=0.0, y_unit=F32, eps=1e-5):
    """(rows whose deviation is off, rows whose mean is off) of y, the norm without weight and
    bias of h (in 64 bits), which the kernel forms with errors of at most h_err and whose
    result is rounded with y_unit."""
    h, y = h.double(), y.double()
    m = h.mean(1, keepdim=True)
    var = (h - m).square().mean(1, keepdim=True)
    ir = 1 / torch.sqrt(var + eps)
    off = (DEPTH + 2) * F32 * h.abs().mean(1, keepdim=True) * ir + h_err * ir
    rel = off ** 2 / 2 + h_err * ir + (DEPTH + C) * F32  # (|h - m| is below a deviation on average)
    spread = y.std(1, keepdim=True, correction=0)
    want = torch.sqrt(var) * ir
    # an element is off by y_unit + 2 F32 of itself where it is rounded, by F32 of |h - m|
    # where the mean is taken from it
    wrong = (spread / want - 1).abs() > (rel + y_unit + 3 * F32) * (1 + off)
    moved = y.mean(1, keepdim=True).abs() > off + (y_unit + 3 * F32) * y.abs().mean(1, keepdim=True)
    return int(wrong.sum()), int(moved.sum())


def gradient(x, up, eps=1e-5):
    """(dx in 64 bits, tolerance) of the norm without weight and bias."""
    x, d = x.double(), up.double()
    m = x.mean(1, keepdim=True)
    c = x - m
    ir = 1 / torch.sqrt(c.square().mean(1, keepdim=True) + eps)
    hn = c * ir
    off = (DEPTH + 2) * F32 * x.abs().mean(1, keepdim=True) * ir  # of hn, the same in a row
    rel = off ** 2 / 2 + (DEPTH + C) * F32
    hn_err = off + (rel + 3 * F32) * hn.abs()
    s0, s1 = d.mean(1, keepdim=True), (d * hn).mean(1, keepdim=True)
    f = (DEPTH + 2) * F32
    s0_err = f * d.abs().mean(1, keepdim=True)
    # (a shift of hn by off moves the mean of d hn by off times the mean of d)
    s1_err = off * s0.abs() + (rel + f + 3 * F32) * (d * hn).abs().mean(1, keepdim=True)
    inner = d.abs() + s0.abs() + (hn * s1).abs()
    dx = ir * (d - s0 - hn * s1)
    err = ir * (s0_err + (hn.abs() + hn_err) * s1_err + hn_err * s1.abs() + C * F32 * inner) + rel * ir * inner
    return dx, err

"""Orthogonalised updates in 64 bits, from their definition, and how far a right kernel may
be from them.

A step maps X to p(X) = X (a + b X^T X + c (X^T X)^2), odd in the singular values.  With u
the rounding of an operand (half a step of fp16, 2^-11, for bf16 matrices; 2^-21 for
fp32 ones, whose products take the rounded value and its rest, 2^-22, and leave out the
product of two rests), a step's own error is at most, in the Frobenius norm,

    u |D|2 |X|F + u |D|F |X|2 + (|b + 2 c mu| + 2 |c| |E|2) |X|2 dE,
    dE = u |E|F + 2 u |X|2 |X|F

(X, D, E and the two copies of X in A, each rounded once), and the steps after it carry it
on by at most the largest divided difference of their joint map over the singular values
and their negatives.  To that the result's own rounding is added, and for fp32 what the
fp32 sums lose: FP32_SUMS times what the same steps lose in torch's fp32 products.

That is what the worst signs of all roundings add up to, some per cent.  The error of a
matrix of many elements is the norm of a sum of as many independent roundings, so that
it lies near what the same roundings give when they are made in 64 bits (emulated): a
matrix of at least MANY elements is held to SPREAD times that as well.
"""
from __future__ import annotations

import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
FP32_SUMS = 4
MANY, SPREAD = 4096, 2


def triples(coefficients, steps):
    flat = not isinstance(coefficients[0], (tuple, list))
    return [tuple(coefficients)] * steps if flat else [tuple(x) for x in coefficients]


def iterate(x, coefficients, dtype, norm, eps):
    """The states X0 .. X_steps of one wide matrix."""
    x = x.to(dtype) * torch.as_tensor(1.0 / (norm + eps), dtype=dtype)
    states = [x]
    for a, b, c in coefficients:
        g = x @ x.T.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
        states.append(x)
    return states


def _carried(s, coefficients):
    """The largest divided difference of the steps' joint map over +-s."""
    t = torch.cat([s, -s])
    v, slope = t.clone(), torch.ones_like(t)
    for a, b, c in coefficients:
        slope = slope * (a + 3 * b * v ** 2 + 5 * c * v ** 4)
        v = v * (a + b * v ** 2 + c * v ** 4)
    gap = t[:, None] - t[None, :]
    near = gap.abs() < 1e-9
    ratio = (v[:, None] - v[None, :]) / torch.where(near, torch.ones_like(gap), gap)
    ratio = torch.where(near, slope[:, None].expand_as(ratio), ratio)
    return float(ratio.abs().max())


def _split(x, scale, planes):
    """x as fp16 numbers hold it: the rounded value and, with two planes, its rest."""
    hi = (x * scale).half().double()
    lo = (x * scale - hi).half().double() if planes == 2 else torch.zeros_like(hi)
    return hi / scale, lo / scale


def _product(x, y, planes, scale):
    """x y^T as fp16 products give it with exact sums."""
    (xh, xl), (yh, yl) = _split(x, scale, planes), _split(y, scale, planes)
    return xh @ yh.T + xh @ yl.T + xl @ yh.T


def emulated(x, coefficients, norm, eps, planes):
    """The last state of a wide matrix with the kernels' roundings to fp16."""
    x = x / (norm + eps)
    scale = 2.0 ** 13
    for a, b, c in coefficients:
        mu = float(x.square().sum()) / x.shape[0]
        e = _product(x, x, planes, scale) - mu * torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
        rounded = sum(_split(e, 2.0 ** 12, planes))
        d = (b + 2 * c * mu) * rounded + c * _product(e, e, planes, 2.0 ** 12)
        x = (a + mu * (b + c * mu)) * x + _product(d, x.T.contiguous(), planes, 2.0 ** 12)
    return x


def orthogonalize(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """(value, bound of the Frobenius norm of the error before the last rounding) of one
    matrix."""
    k = triples(coefficients, steps)
    tall = update.shape[0] > update.shape[1]
    x = update.detach().double()
    x = x.T.contiguous() if tall else x
    norm = float(x.square().sum().sqrt())
    states = iterate(x, k, torch.float64, norm, eps)
    u = 2.0 ** -21 if update.dtype == torch.float32 else 2.0 ** -11
    bound = 0.0
    r = x.shape[0]
    for i, (a, b, c) in enumerate(k):
        s = torch.linalg.svdvals(states[i].cpu())
        mu = float((s ** 2).sum()) / r
        e = torch.cat([s ** 2, torch.zeros(r - len(s), dtype=s.dtype)]) - mu
        d = (b + 2 * c * mu) * e + c * e ** 2
        top, full = float(s.max()), float(s.norm())
        de = u * float(e.norm()) + 2 * u * top * full
        own = u * float(d.abs().max()) * full + u * float(d.norm()) * top \
            + (abs(b + 2 * c * mu) + 2 * abs(c) * float(e.abs().max())) * top * de
        after = torch.linalg.svdvals(states[i + 1].cpu())
        bound += own * (_carried(after, k[i + 1:]) if k[i + 1:] else 1.0)
    sums = 0.0
    if update.dtype == torch.float32:
        single = iterate(x.float(), k, torch.float32, norm, eps)[-1]
        sums = FP32_SUMS * float((single.double() - states[-1]).norm())
    bound += sums
    if x.numel() >= MANY:
        like = emulated(x, k, norm, eps, 2 if update.dtype == torch.float32 else 1)
        bound = min(bound, sums + SPREAD * float((like - states[-1]).norm()))
    return (states[-1].T if tall else states[-1]).cpu(), bound


def assert_within(got, update, **kw):
    """One matrix's result within its bound, as a whole and each element."""
    want, bound = orthogonalize(update, **kw)
    x = got.detach().double().cpu()
    assert torch.isfinite(x).all()
    u = torch.finfo(update.dtype).eps / 2
    size = float(want.norm())
    off = x - want
    floor = 2.0 ** -126
    assert float(off.norm()) <= u * size + (1 + u) * bound + floor, (
        f"off by {float(off.norm()):.3g}, allowed {u * size:.3g} + {bound:.3g} of {size:.3g}")
    assert bool((off.abs() <= u * want.abs() + (1 + u) * bound + floor).all())
    return float(off.norm()) / max(size, floor), bound / max(size, floor)

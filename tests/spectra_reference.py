"""Orthogonalised updates of bf16 matrices whose singular values are far apart, and how
their fp16 products may be rounded.

A step maps X to a X + M X, M = b A + c A^2.  The product's operand is X rounded to fp16, X~,
and its error M (X~ - X).  Taken around mu, as D X~ + p(mu) X with D = M - p(mu) I, the
error is D (X~ - X) instead: smaller where all eigenvalues of A lie near mu, but D is -p(mu)
and not 0 along singular vectors of small singular values, and what gets in there is lifted by
the steps that follow as those are.  With p(mu) (f X + (1 - f) X~) the error is (M - f p(mu) I)
(X~ - X).  Its sum over the eigenvalues, each lifted to about 1 in the end, is least where
f mu is their harmonic mean; f = 1 - var / mu^2, at least 0, is that mean's ratio to mu for
the eigenvalues of large random matrices, and 0 where they spread further.  The last two steps
take f = 1: little is lifted after them.
"""
from __future__ import annotations

import math

import torch

from update_reference import COEFFICIENTS, _product, _split, iterate, triples


def rounded(x, coefficients, norm, eps, around=False):
    """The last state of a wide matrix with one fp16 product a term: f as above, or f = 1 in
    every step (around)."""
    x = x / (norm + eps)
    scale, mid, r = 2.0 ** 13, 2.0 ** 12, x.shape[0]
    for i, (a, b, c) in enumerate(coefficients):
        mu = float(x.square().sum()) / r
        e = _product(x, x, 1, scale) - mu * torch.eye(r, dtype=x.dtype)
        linear = _split(e, mid, 1)[0]
        square = _product(e, e, 1, mid)
        var = float(square.trace()) / r
        f = 1.0 if around or i + 2 >= len(coefficients) else max(0.0, 1.0 - var / mu ** 2)
        p = mu * (b + c * mu)
        d = (b + 2 * c * mu) * linear + c * square
        x = (a + f * p) * x + (1 - f) * p * _split(x, scale, 1)[0] + _product(d, x.T.contiguous(), 1, mid)
    return x


def matrices(r, c, seed=0):
    """{kind: a bf16 matrix r x c}."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    i, k = torch.arange(r, dtype=torch.float64) / r, max(1, r // 8)

    def spectrum(s):
        u, v = torch.linalg.qr(rand(r, r))[0], torch.linalg.qr(rand(c, r))[0]
        return (u * s) @ v.T.contiguous()

    found = {
        "random": rand(r, c),
        "momentum": (rand(r, k) * torch.exp(rand(1, k))) @ rand(k, c) / math.sqrt(k) + rand(r, c),
        "rows apart": torch.exp(3 * rand(r, 1)) * rand(r, c),
        "10^-3": spectrum(10 ** (-3 * i)),
        "10^-6": spectrum(10 ** (-6 * i)),
        "an eighth strong": rand(r, k) @ rand(k, c) + 0.01 * rand(r, c),
        "half strong": rand(r, r // 2 or 1) @ rand(r // 2 or 1, c) + 0.05 * rand(r, c),
        "most strong": rand(r, r * 7 // 8 or 1) @ rand(r * 7 // 8 or 1, c) + 0.05 * rand(r, c),
        "rank 1": rand(r, 1) @ rand(1, c),
    }
    return {n: x.to(torch.bfloat16) for n, x in found.items()}


def exact(x, coefficients=COEFFICIENTS, steps=5, eps=1e-7):
    """The last state of a wide bf16 matrix in 64 bits."""
    x = x.double()
    return iterate(x, triples(coefficients, steps), torch.float64, float(x.norm()), eps)[-1]


def ratio(got, want):
    """The error of a bf16 result over that of the exact value rounded to bf16."""
    off = (got.double() - want).norm()
    return float(off / (want.to(torch.bfloat16).double() - want).norm())

"""bf16 matrices whose singular values are far apart, and their orthogonalised updates in 64
bits."""
from __future__ import annotations

import math

import torch

from update_reference import COEFFICIENTS, iterate, triples


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

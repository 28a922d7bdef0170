"""The workspace of an orthogonalised update is what the documentation says."""
from __future__ import annotations

import ctypes

import pytest

from mini_trainer_amd import _lib

import update_reference as ref

FIVE = (ctypes.c_double * 15)(*ref.COEFFICIENTS * 5)


def little(m, n):
    """State, sums of squares (4 bytes a tile of 64 x 64), whole 256 bytes."""
    return (16 << 10) + m * n // 1024


def need(m, n, dtype, batch=1):
    a = _lib.OrthogonalizeArgs()
    for name, value in dict(coefficients=ctypes.addressof(FIVE), eps=1e-7, batch=batch, m=m, n=n, in_row=n,
                            in_batch=m * n, steps=5, dtype=dtype).items():
        setattr(a, name, value)
    return _lib.load().mt_orthogonalize_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("m,n", [(4096, 4096), (14336, 4096), (256, 1536), (128, 8192), (64, 65536), (16384, 256)])
def test_bytes_of_a_matrix(m, n):
    r, c = min(m, n), max(m, n)
    for dtype, rc, rr in ((1, 10, 6), (0, 16, 12)):
        least = rc * r * c + rr * r * r
        more = (8 << 20) if r <= 1024 else 0
        assert least <= need(m, n, dtype) <= least + more + little(m, n)
        assert need(m, n, dtype, 1000) <= max(2 << 30, need(m, n, dtype))


def test_a_short_side_counts_as_64_in_part():
    for dtype, own, padded in ((1, 6, 4), (0, 8, 8)):
        got = need(16, 16384, dtype)
        least = (own * 16 + padded * 64) * 16384
        assert least <= got <= least + (8 << 20) + little(16, 16384)

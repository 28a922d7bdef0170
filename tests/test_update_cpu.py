"""Orthogonalised updates without a GPU: what the entry points refuse, in Python and in
the C ABI, before anything is launched."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mini_trainer_amd as mt
from mini_trainer_amd import _lib, update

import update_reference as ref

P = 1 << 20
BIG = 2 ** 63 - 1
FIVE = (ctypes.c_double * 15)(*ref.COEFFICIENTS * 5)


def args(coefficients=FIVE, **kw):
    a = _lib.OrthogonalizeArgs()
    base = dict(input=P, out=P, coefficients=ctypes.addressof(coefficients) if coefficients else None, eps=1e-7,
                batch=2, m=140, n=172, in_row=172, in_batch=140 * 172, steps=5, dtype=1)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), 1), (dict(batch=-1), 1), (dict(m=-1), 1), (dict(n=-5), 1), (dict(steps=0), 1),
    (dict(steps=65), 1), (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(eps=math.inf), 1),
    (dict(coefficients=None), 1), (dict(batch=BIG), 3), (dict(m=BIG), 3), (dict(n=BIG), 3),
    (dict(m=32768, n=32768, in_row=32768), 3), (dict(m=1, n=1 << 24, in_row=1 << 24), 3),
    (dict(in_row=171), 1), (dict(in_row=BIG), 1), (dict(in_batch=-1), 1), (dict(in_batch=BIG), 1),
    (dict(input=None), 1), (dict(out=None), 1), (dict(input=P + 1), 1), (dict(out=P + 1), 1),
    (dict(coefficients=(ctypes.c_double * 15)(*[40.0, 0.0, 0.0] * 5)), 3),
    (dict(coefficients=(ctypes.c_double * 15)(*[3.0, math.nan, 0.0] * 5)), 1),
    (dict(coefficients=(ctypes.c_double * 15)(*[1e300, 1e300, 1e300] * 5)), 3),
])
def test_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_orthogonalize(ctypes.byref(args(**kw)), P, 1 << 40, None) == code
    assert lib.mt_flce_last_error()


def test_workspace():
    lib = _lib.load()
    need = lib.mt_orthogonalize_workspace_bytes(ctypes.byref(args()))
    assert need % 512 == 0 and need >= 2 * (140 * 192 * 2 + 2 * 172 * 192 * 2 + 3 * 140 * 192 * 2 + 140 * 172 * 4)
    one = lib.mt_orthogonalize_workspace_bytes(ctypes.byref(args(batch=1)))
    assert need == 2 * one
    assert lib.mt_orthogonalize(ctypes.byref(args()), P, one - 1, None) == 2
    assert lib.mt_orthogonalize(ctypes.byref(args()), P + 16, need, None) == 1
    assert lib.mt_orthogonalize(ctypes.byref(args()), None, need, None) == 1
    assert lib.mt_orthogonalize(None, P, need, None) == 1
    # a stack asks for up to 2 GiB, or for one matrix
    big = args(batch=1 << 20, m=4096, n=4096, in_row=4096)
    single = lib.mt_orthogonalize_workspace_bytes(ctypes.byref(args(batch=1, m=4096, n=4096, in_row=4096)))
    assert lib.mt_orthogonalize_workspace_bytes(ctypes.byref(big)) == (2 << 30) // single * single
    for kw in (dict(batch=0), dict(m=0), dict(m=BIG), dict(batch=BIG), dict(dtype=9), dict(batch=-BIG)):
        assert lib.mt_orthogonalize_workspace_bytes(ctypes.byref(args(**kw))) == 0
    # small matrices take none
    for m, n, dtype, none in ((128, 352, 1, True), (352, 128, 1, True), (128, 353, 1, False), (16, 4096, 1, True),
                              (16, 4097, 1, False), (17, 2048, 1, True), (64, 992, 1, True), (64, 993, 1, False), (129, 129, 1, False),
                              (64, 416, 0, True), (64, 417, 0, False), (65, 65, 0, False), (16, 2400, 0, True)):
        a = args(batch=1, m=m, n=n, in_row=n, dtype=dtype)
        assert (lib.mt_orthogonalize_workspace_bytes(ctypes.byref(a)) == 0) == none, (m, n, dtype)
        a = args(batch=1, m=m, n=n, in_row=n, dtype=dtype, steps=17)
        assert lib.mt_orthogonalize_workspace_bytes(ctypes.byref(a)) > 0
    # nothing to do: no launch
    for kw in (dict(batch=0), dict(m=0), dict(n=0)):
        assert lib.mt_orthogonalize(ctypes.byref(args(**kw, input=None, out=None)), None, 0, None) == 0


def test_python_refusals():
    x = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.orthogonalize(x)
    for bad in ((1.0, 2.0), [(1.0, 2.0, 3.0)] * 4, [(1.0, 2.0)] * 5, (1.0, math.nan, 2.0), ()):
        with pytest.raises(ValueError, match="coefficients"):
            update._coefficients(bad, 5)
    assert list(update._coefficients((1, 2, 3), 2)) == [1.0, 2.0, 3.0] * 2
    assert list(update._coefficients([(1, 2, 3), (4, 5, 6)], 2)) == [1.0, 2.0, 3.0, 4.0, 5.0, 6.0]


def test_the_reference_brings_singular_values_near_one():
    x = torch.randn(72, 140, generator=torch.Generator().manual_seed(0))
    for t, within in ((x.bfloat16(), 2.0 ** -8), (x, 2.0 ** -16)):
        value, bound = ref.orthogonalize(t)
        s = torch.linalg.svdvals(value)
        assert 0.6 < float(s.min()) and float(s.max()) < 1.3 and bound < within * float(value.norm())

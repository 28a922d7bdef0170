"""What the C ABI of packed attention refuses, beside test_step_cpu.py, and the
arguments it takes."""
from __future__ import annotations

import ctypes

import pytest

from mini_trainer_amd import _lib

from test_step_cpu import P, attn


@pytest.mark.parametrize("kw", [
    dict(softcap=3e38),                # softcap log2(e) is infinite
    dict(scale=1e-10, softcap=1e30),   # scale / softcap is no normal number
    dict(scale=1e-30, softcap=1e20),   # it is 0
])
@pytest.mark.parametrize("dtype", [0, 1])
def test_softcaps_out_of_range(kw, dtype):
    lib = _lib.load()
    a = attn(**kw, dtype=dtype)
    assert lib.mt_attn_forward(ctypes.byref(a), None) == 1
    assert b"softcap" in lib.mt_flce_last_error()
    assert lib.mt_attn_backward(ctypes.byref(a), P, 1 << 40, None) == 1

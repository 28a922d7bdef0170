"""The C ABI of a step's operators on the host: what it refuses, and how much memory it
asks for (beside test_step_cpu.py)."""
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


@pytest.mark.parametrize("T", [1, 2, 3, 5, 511, 512, 513, 2047, 2048, 65536, 2 ** 31 - 1025])
@pytest.mark.parametrize("H", [1, 64, 512, 513, 1000, 1024, 1025, 1032, 4096, 8192, 32768])
def test_norm_workspace_is_three_sums_of_the_partial_rows(T, H):
    """512 workgroups at most, each with a partial row, four up to 1024 elements: 25 MB
    for rows of 4096 and 50 for 8192, however many there are."""
    need = _lib.load().mt_norm_backward_workspace_bytes(T, H)
    rows = max(4, min(-(-T // 4), 512) * 4) if H <= 1024 else min(T, 512)
    assert need == 3 * rows * H * 4 <= 3 * 512 * 4 * max(4 * min(H, 1024), H)


@pytest.mark.parametrize("dtype,V", [(0, 4), (1, 8)])
def test_norm_workspace_holds_what_every_variant_writes(dtype, V):
    """Threads of a row and rows of a workgroup by width and alignment, as they are chosen:
    a wave for up to two vectors a lane, else one row."""
    lib = _lib.load()
    for H in list(range(1, 1100)) + [2048, 4096, 8191, 8192, 32768]:
        for aligned in (True, False):
            wave = aligned and H % V == 0 and H <= 64 * 2 * V
            per = 4 if wave else 1
            for T in (1, 3, 4, 5, 600, 2044, 2045, 5000):
                parts = min(-(-T // per), 512) * per
                assert 3 * parts * H * 4 <= lib.mt_norm_backward_workspace_bytes(T, H)


BIG = 2 ** 63 - 1


def test_queries_of_what_no_call_takes():
    """No arithmetic on sizes that the calls refuse: 0 bytes."""
    lib = _lib.load()
    for kw in (dict(heads=BIG), dict(heads=2 ** 40, kv_heads=1), dict(T=BIG), dict(S=BIG), dict(head_dim=BIG),
               dict(kv_heads=BIG), dict(kv_heads=8), dict(T=-BIG), dict(heads=-4)):
        assert lib.mt_attn_backward_workspace_bytes(ctypes.byref(attn(**kw))) == 0
        assert lib.mt_attn_backward(ctypes.byref(attn(**kw)), P, 1 << 40, None) in (1, 3)
    for stride in ("q_h", "k_h", "v_h"):  # addresses in 64 bits
        assert lib.mt_attn_forward(ctypes.byref(attn(**{stride: 2 ** 41})), None) == 3
    assert lib.mt_norm_backward_workspace_bytes(BIG, 64) == 0
    for bad in ([BIG, BIG], [8, -BIG], [2 ** 40 + 1]):
        table = (ctypes.c_int64 * len(bad))(*bad)
        assert lib.mt_grad_norm_workspace_bytes(table, len(bad)) == 0
    assert lib.mt_grad_norm_workspace_bytes((ctypes.c_int64 * 2)(2 ** 40, 2 ** 40), 2) > 0

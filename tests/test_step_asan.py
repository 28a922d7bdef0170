"""The host code of a step's operators under AddressSanitizer and
UndefinedBehaviorSanitizer: sizes, strides and tables at the ends of their types, and the
host tests."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SWEEP = """
import ctypes, sys
sys.path.insert(0, "tests")
from test_step_cpu import P, attn, norm, table
from mini_trainer_amd import _lib

lib = _lib.load()
assert "libmt_flce_san" in str(_lib.LIB_PATH)
B = 2 ** 63 - 1
ends = [B, -B - 1, B - 7, 2 ** 62, 2 ** 41, -1, 0]
for field in ("q_t", "q_h", "k_t", "k_h", "v_t", "v_h", "dout_t", "dout_h", "T", "S", "heads",
              "kv_heads", "head_dim", "window"):
    for x in ends:
        a = attn(**{field: x})
        lib.mt_attn_backward_workspace_bytes(ctypes.byref(a))
        lib.mt_attn_backward(ctypes.byref(a), P, 1, None)  # (never enough memory to launch)
for field in ("x_t", "residual_t", "gate_t", "dnormed_t", "dresidual_out_t", "T", "H"):
    for x in ends:
        a = norm(**{field: x})
        lib.mt_norm_backward_workspace_bytes(a.T, a.H)
        lib.mt_norm_backward(ctypes.byref(a), P, 1, None)
for numel in ends:
    for cols in ends:
        for pitch in ends:
            t = table([(P, numel, cols, pitch, 1)])
            lib.mt_grad_norm_workspace_bytes(t[1], 1)
            lib.mt_grad_norm(*t, 1, 0, 1.0, P, 1, P, None)
for T in ends:
    for S in ends:
        lib.mt_attn_plan_bytes(T, S)
        lib.mt_attn_plan(P, None, S, T, 5, P, 1, P, None)
print("sweep ok")
"""


def test_step_host_code_under_sanitizers():
    from mini_trainer_amd.build import asan_runtime, build_sanitized, san_is_stale

    rt = asan_runtime()
    if not rt.is_absolute() or not rt.exists():
        pytest.skip("clang ASan runtime not found next to hipcc")
    lib = build_sanitized() if san_is_stale() else \
        ROOT / "mini_trainer_amd" / "_build" / "libmt_flce_san.so"
    env = dict(os.environ, MT_FLCE_LIB=str(lib), LD_PRELOAD=str(rt), PYTHONPATH=str(ROOT),
               ASAN_OPTIONS="detect_leaks=0:halt_on_error=1:abort_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", HIP_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", SWEEP], env=env, cwd=ROOT, capture_output=True, text=True,
                       timeout=600)
    assert r.returncode == 0 and "sweep ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider",
                        "tests/test_step_cpu.py", "tests/test_step_host_cpu.py"], env=env, cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-4000:]

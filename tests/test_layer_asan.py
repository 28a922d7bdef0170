"""The host code of token embedding, layer norm and orthogonalised updates under
AddressSanitizer and UndefinedBehaviorSanitizer: sizes and strides at the ends of their
types, and the host tests."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SWEEP = """
import ctypes, itertools, sys
sys.path.insert(0, "tests")
from test_layer_cpu import P, embed, norm
from test_update_cpu import args
from mini_trainer_amd import _lib

lib = _lib.load()
assert "libmt_flce_san" in str(_lib.LIB_PATH)
B = 2 ** 63 - 1
ends = [B, -B - 1, B - 7, 2 ** 62, 2 ** 41, 2 ** 31 - 1, 2 ** 24, -1, 0]
for field in ("T", "V", "H", "weight_t", "dout_t", "dweight_t", "padding_idx"):
    for x in ends:
        a = embed(**{"T": 300, field: x})
        lib.mt_embed_backward(ctypes.byref(a), P, 1, None)  # (never enough memory to launch)
        a.out = None
        lib.mt_embed_forward(ctypes.byref(a), None)
for sizes in itertools.product(ends, repeat=3):
    lib.mt_embed_backward_workspace_bytes(*sizes)
for field in ("T", "H", "x_t", "residual_t", "dnormed_t", "dresidual_out_t"):
    for x in ends:
        a = norm(**{field: x})
        lib.mt_layer_norm_backward(ctypes.byref(a), P, 1, None)
        a.normed = None
        lib.mt_layer_norm_forward(ctypes.byref(a), None)
for sizes in itertools.product(ends, repeat=2):
    lib.mt_layer_norm_backward_workspace_bytes(*sizes)
every = (ctypes.c_double * 51)(*[3.4445, -4.775, 2.0315] * 17)
for batch, m, n in itertools.product(ends + [1, 2 ** 30], repeat=3):
    for dtype in (0, 1):
        a = args(every, batch=batch, m=m, n=n, in_row=max(n, 0), in_batch=2 ** 40, dtype=dtype, steps=17)
        lib.mt_orthogonalize_workspace_bytes(ctypes.byref(a))
        lib.mt_orthogonalize(ctypes.byref(a), 256, 1, None)
print("sweep ok")
"""


def test_layer_host_code_under_sanitizers():
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
                        "tests/test_layer_cpu.py", "tests/test_update_cpu.py"], env=env, cwd=ROOT,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-4000:]

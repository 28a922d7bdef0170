"""Autograd nodes without a GPU: what they hand to the C ABI, whose entries are replaced by
functions of this file that look at it."""
from __future__ import annotations

import ctypes
import os
import sys
import types
from ctypes import POINTER, c_int, c_int64, c_size_t, c_void_p

import pytest
import torch

from mini_trainer_amd import _lib, build, norms
from mini_trainer_amd._lib import EmbedArgs, LayerNormArgs, NormArgs

OK = ctypes.CFUNCTYPE(c_int, c_void_p, c_void_p)
BYTES = ctypes.CFUNCTYPE(c_size_t, c_int64, c_int64)


@pytest.fixture
def nodes():
    """bind(name=function, ...): the nodes call these in place of the library's."""
    ops, lib, kept = _lib.torch_ops(), _lib.load(), []

    def bind(**own):
        kept.extend(own.values())
        ops.bind([ctypes.cast(own.get(name) or getattr(lib, name), c_void_p).value for name in _lib._BOUND],
                 _lib.FlceError)
        return ops

    yield bind
    bind()


def matrix(address, pitch, T, H, dtype=ctypes.c_float):
    """[T, H] numbers whose rows begin `pitch` apart at an address."""
    flat = (dtype * ((T - 1) * pitch + H)).from_address(address)
    return torch.tensor([[flat[t * pitch + c] for c in range(H)] for t in range(T)])


def shuffled(t):
    """Equal values that lie in memory in another order."""
    if t.dim() == 2:
        return t.T.contiguous().T
    return torch.stack([t, t], -1)[..., 0] if t.dim() == 1 else t


@pytest.mark.parametrize("residual", [False, True])
def test_saved_tensors_may_come_back_in_another_layout(nodes, residual):
    """A hook on saved tensors answers for their values alone."""
    T, H = 5, 8
    seen = []

    def backward(a, ws, bytes_, stream):
        a = a.contents
        h = matrix(a.new_residual, H, T, H) if residual else matrix(a.x, a.x_t, T, H)
        stat = matrix(ctypes.cast(a.stat, c_void_p).value, 2 * T, 1, 2 * T)
        seen.append((h, matrix(a.weight, H, 1, H), stat))
        return 0

    def forward(a, stream):
        a = ctypes.cast(a, POINTER(LayerNormArgs)).contents
        if residual:
            ctypes.memmove(a.new_residual, a.x, 4 * T * H)
        for i in range(2 * T):
            (ctypes.c_float * (2 * T)).from_address(a.stat)[i] = i
        return 0

    ops = nodes(mt_layer_norm_forward=OK(forward),
                mt_layer_norm_backward=ctypes.CFUNCTYPE(c_int, POINTER(LayerNormArgs), c_void_p, c_size_t,
                                                        c_void_p)(backward))
    x = torch.arange(T * H, dtype=torch.float32).view(T, H).requires_grad_(True)
    r = torch.zeros(T, H, requires_grad=True) if residual else None
    w = torch.arange(H, dtype=torch.float32).requires_grad_(True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), shuffled):
        outs = ops.layer_norm(x, r, w, None, 1e-5, 1.0, 1.0, True, 0)
        torch.autograd.grad(outs[0], w, torch.zeros(T, H))
    h, weight, stat = seen[0]
    assert torch.equal(h, x) and torch.equal(weight[0], w)
    assert torch.equal(stat[0], torch.arange(2.0 * T))


def test_saved_ids_may_come_back_in_another_layout(nodes):
    seen = []

    def backward(a, ws, bytes_, stream):
        seen.append(matrix(a.contents.ids, 7, 1, 7, ctypes.c_int64))
        return 0

    ops = nodes(mt_embed_forward=OK(lambda a, stream: 0),
                mt_embed_backward=ctypes.CFUNCTYPE(c_int, POINTER(EmbedArgs), c_void_p, c_size_t,
                                                   c_void_p)(backward))
    ids, w = torch.arange(7), torch.zeros(9, 4, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), shuffled):
        out = ops.embedding(ids, w, 1.0, -1, None, None, 0)
        torch.autograd.grad(out, w, torch.zeros(7, 4))
    assert torch.equal(seen[0][0], ids)


@pytest.mark.parametrize("back", [shuffled, torch.Tensor.contiguous])
@pytest.mark.parametrize("gated", [norms.GATE_CHANNEL, norms.GATE_TOKEN, norms.GATE_ELEMENT])
def test_residual_rms_norm_reads_what_a_hook_hands_back(monkeypatch, back, gated):
    """contiguous: as torch.autograd.graph.save_on_cpu does it with rows of a wider tensor."""
    T, H = 6, 8
    shape = {norms.GATE_CHANNEL: (H,), norms.GATE_TOKEN: (T, 1), norms.GATE_ELEMENT: (T, H)}[gated]
    wide = torch.arange(T * 24, dtype=torch.float32).view(T, 24)
    x, w = wide[:, 3:3 + H].requires_grad_(True), torch.arange(H, dtype=torch.float32)
    gate = wide[:, 12:12 + shape[-1]] if len(shape) == 2 else torch.arange(H) + 0.5
    r, seen = torch.ones(T, H), []

    def launch(dev, what, entry, args, *rest):
        a = NormArgs.from_buffer_copy(args)
        if what == "mt_norm_forward":
            ctypes.memmove(a.new_residual, r.data_ptr(), 4 * T * H)
            for i in range(2 * T):
                (ctypes.c_float * (2 * T)).from_address(a.rstd)[i] = i
            return
        seen.append((a.x_t, a.gate_t))
        assert a.x_t <= H and a.gate_t <= H  # (what came back has no more)
        pitch, rows_ = (a.gate_t, T) if gated != norms.GATE_CHANNEL else (H, 1)
        seen.append((matrix(a.x, a.x_t, T, H), matrix(a.gate, pitch, rows_, shape[-1]),
                     matrix(a.weight, H, 1, H)[0], matrix(a.new_residual, H, T, H),
                     matrix(a.rstd, 2 * T, 1, 2 * T)[0]))

    monkeypatch.setattr(norms, "_launch", launch)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), back):
        y, _ = norms._ResidualRmsNorm.apply(x, r, w, None, gate, gated, 1e-6, 1.0, 1.0, 0.0)
        torch.autograd.grad(y, x, torch.zeros(T, H))
    got_x, got_gate, got_w, got_r, got_rstd = seen[1]
    assert torch.equal(got_x, x) and torch.equal(got_gate.reshape(shape), gate) and torch.equal(got_w, w)
    assert torch.equal(got_r, r) and torch.equal(got_rstd, torch.arange(2.0 * T))


def test_errors_of_a_backward_are_the_packages(nodes):
    """They come to Python out of the engine, not through a call of the module."""
    refuse = lambda *a: 3  # noqa: E731
    ops = nodes(mt_layer_norm_forward=OK(lambda a, stream: 0), mt_embed_forward=OK(lambda a, stream: 0),
                mt_layer_norm_backward=ctypes.CFUNCTYPE(c_int, c_void_p, c_void_p, c_size_t, c_void_p)(refuse),
                mt_embed_backward=ctypes.CFUNCTYPE(c_int, c_void_p, c_void_p, c_size_t, c_void_p)(refuse))
    x, w = torch.zeros(3, 8, requires_grad=True), torch.zeros(9, 4, requires_grad=True)
    for out, leaf in ((ops.layer_norm(x, None, None, None, 1e-5, 1.0, 1.0, True, 0)[0], x),
                      (ops.embedding(torch.arange(7), w, 1.0, -1, None, None, 0), w)):
        with pytest.raises(_lib.FlceError, match="_backward: MT_ERR_UNSUPPORTED"):
            torch.autograd.grad(out, leaf, torch.zeros_like(out))


@pytest.mark.parametrize("change,what", [(dict(abi_version=_lib.ABI_VERSION - 1), "ABI version"),
                                         (dict(abi_version=None), "ABI version"),
                                         (dict(torch_version="1.13.0"), "torch 1.13.0")])
def test_nodes_of_another_build_are_refused(monkeypatch, change, what):
    """Before they are handed the library's functions: a struct of theirs may differ."""
    have = dict(abi_version=_lib.ABI_VERSION, torch_version=torch.__version__,
                bind=lambda *a: pytest.fail("bound"))
    have = {k: v for k, v in {**have, **change}.items() if v is not None}
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setitem(sys.modules, "mini_trainer_amd._mt_torch", types.SimpleNamespace(**have))
    with pytest.raises(_lib.FlceError, match=what):
        _lib.torch_ops()
    assert _lib._torch_ops is None


def test_nodes_are_stale_with_their_source(tmp_path, monkeypatch):
    """The module counts as the library does: missing, or older than what it is built from."""
    lib, module, source, header = (tmp_path / n for n in ("lib.so", "module.so", "ops.cpp", "abi.h"))
    for p in (source, header, lib, module):
        p.write_text("")
    for name, value in (("LIB_PATH", lib), ("TORCH_PATH", module), ("DEPENDS", [header]),
                        ("TORCH_DEPENDS", [source, header])):
        monkeypatch.setattr(build, name, value, raising=False)

    def at(**times):
        for p in (source, header, lib, module):
            os.utime(p, (times.get(p.stem, 100),) * 2)
        return build.is_stale()

    assert not at(lib=200, module=200)
    assert at(lib=200, module=50) and at(lib=50, module=200)
    assert at(lib=200, module=200, ops=300) and at(lib=400, module=200, abi=300)
    assert not at(lib=200, module=400, ops=300)
    module.unlink()
    assert build.is_stale()

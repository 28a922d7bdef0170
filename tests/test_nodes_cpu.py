"""The C++ autograd nodes without a GPU: what they hand to the C ABI, whose backward entries
are replaced by functions of this file that look at it."""
from __future__ import annotations

import ctypes
from ctypes import POINTER, c_int, c_int64, c_size_t, c_void_p

import pytest
import torch

from mini_trainer_amd import _lib
from mini_trainer_amd._lib import EmbedArgs, LayerNormArgs

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

"""Token embedding and layer norm without a GPU: what the entry points refuse, in Python
and in the C ABI, before anything is launched; the references that the GPU tests use,
against torch's own functions and autograd."""
from __future__ import annotations

import ctypes
import math
import sys

import pytest
import torch

import mini_trainer_amd as mt
from mini_trainer_amd import _lib
from mini_trainer_amd._lib import EmbedArgs, LayerNormArgs

import layer_reference as ref

P = 1 << 20  # an aligned address that no checked call reads
BIG = 2 ** 63 - 1


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.token_embedding(torch.zeros(3, dtype=torch.int64), t)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.layer_norm(t)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.residual_layer_norm(t, t)
    with pytest.raises(ValueError, match="residual"):
        mt.residual_layer_norm(t, None)


def embed(**kw):
    a = EmbedArgs()
    base = dict(ids=P, weight=P, out=P, dout=P, dweight=P, weight_t=64, dout_t=64, dweight_t=64, T=10,
                V=100, H=64, padding_idx=-1, scale=1.0, dtype=1, ids_bytes=8, accumulate=0)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return a


EMBED_BOTH = [
    (dict(dtype=5), 1), (dict(ids_bytes=2), 1), (dict(T=-1), 1), (dict(T=2 ** 31), 1), (dict(V=0), 1),
    (dict(V=BIG), 1), (dict(H=0), 1), (dict(H=(1 << 24) + 1, weight_t=BIG, dout_t=BIG, dweight_t=BIG), 3),
    (dict(scale=math.nan), 1), (dict(scale=math.inf), 1), (dict(padding_idx=-2), 1),
    (dict(padding_idx=100), 1), (dict(ids=None), 1), (dict(ids=P + 4), 1),
]


@pytest.mark.parametrize("kw,code", EMBED_BOTH + [
    (dict(weight_t=63), 1), (dict(weight_t=2 ** 32 + 1), 3), (dict(weight=None), 1), (dict(out=None), 1),
    (dict(weight=P + 1), 1), (dict(out=P + 1), 1), (dict(status=P + 2), 1),
    (dict(T=2 ** 31 - 1025, H=1 << 24, weight_t=1 << 24), 3),  # 2^32 threads and more
])
def test_embedding_forward_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_embed_forward(ctypes.byref(embed(**kw)), None) == code
    assert lib.mt_flce_last_error()


@pytest.mark.parametrize("kw,code", EMBED_BOTH + [
    (dict(dout_t=63), 1), (dict(dweight_t=63), 1), (dict(dout_t=BIG), 3), (dict(dweight_t=BIG), 3),
    (dict(dout=None), 1), (dict(dweight=None), 1), (dict(dout=P + 1), 1),
    (dict(accumulate=1, dweight=P + 2), 1),
])
def test_embedding_backward_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_embed_backward(ctypes.byref(embed(**kw)), P, 1 << 40, None) == code


def test_embedding_workspace():
    lib = _lib.load()
    need = lib.mt_embed_backward_workspace_bytes
    # 256 buckets of whole ids and one end, the tokens' order, two rows for each 32 tokens
    assert need(65536, 128256, 4096) == -(-4 * (256 * 501 + 1) // 64) * 64 + 4 * 65536 + 2 * 2048 * 4096 * 4
    assert need(257, 1000, 64) == -(-4 * (256 * 4 + 1) // 64) * 64 + -(-4 * 257 // 64) * 64 + 2 * 9 * 64 * 4
    assert need(300, 262145, 1) == -(-4 * (512 * 513 + 1) // 64) * 64 + -(-4 * 300 // 64) * 64 + 2 * 10 * 4 * 4
    # few tokens are not sorted
    assert need(256, 1000, 64) == need(0, 1, 1) == 0
    for bad in ((-1, 5, 5), (5, 0, 5), (5, 5, 0), (BIG, 5, 5), (5, BIG, 5), (5, 5, BIG)):
        assert need(*bad) == 0
    a = embed(T=300)
    n = need(300, 100, 64)
    assert lib.mt_embed_backward(ctypes.byref(a), P, n - 1, None) == 2
    assert lib.mt_embed_backward(ctypes.byref(a), None, n, None) == 1
    assert lib.mt_embed_backward(ctypes.byref(a), P + 8, n, None) == 1
    assert lib.mt_embed_backward(None, P, n, None) == lib.mt_embed_forward(None, None) == 1
    # nothing to do: no launch
    assert lib.mt_embed_forward(ctypes.byref(embed(T=0, ids=None, out=None)), None) == 0


def norm(**kw):
    a = LayerNormArgs()
    base = dict(x=P, residual=P, weight=P, bias=P, normed=P, new_residual=P, residual_lo=P, stat=P,
                dnormed=P, dresidual_out=P, dx=P, dresidual=P, dweight=P, dbias=P, x_t=64, residual_t=64,
                dnormed_t=64, dresidual_out_t=64, T=10, H=64, eps=1e-5, block_scale=1.0,
                residual_scale=1.0, has_residual=1, dtype=1)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return a


NORM_BOTH = [
    (dict(dtype=5), 1), (dict(T=-1), 1), (dict(T=2 ** 31), 1), (dict(H=0), 1), (dict(H=32769), 3),
    (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(eps=math.inf), 1), (dict(block_scale=math.inf), 1),
    (dict(residual_scale=math.nan), 1), (dict(new_residual=None), 1), (dict(weight=P + 1), 1),
    (dict(has_residual=0), 1), (dict(stat=P + 2), 1),
]


@pytest.mark.parametrize("kw,code", NORM_BOTH + [
    (dict(x_t=63), 1), (dict(residual_t=63), 1), (dict(x=None), 1), (dict(residual=None), 1),
    (dict(normed=None), 1), (dict(x=P + 1), 1),
    (dict(T=2 ** 31 - 1025, H=32768, x_t=32768, residual_t=32768), 3),  # 2^32 threads and more
])
def test_layer_norm_forward_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_layer_norm_forward(ctypes.byref(norm(**kw)), None) == code
    assert lib.mt_flce_last_error()


@pytest.mark.parametrize("kw,code", NORM_BOTH + [
    (dict(dnormed_t=63), 1), (dict(dresidual_out_t=63), 1), (dict(dnormed=None), 1), (dict(stat=None), 1),
    (dict(residual_lo=None), 1), (dict(dx=P + 1), 1),
])
def test_layer_norm_backward_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_layer_norm_backward(ctypes.byref(norm(**kw)), P, 1 << 40, None) == code


def test_layer_norm_workspace():
    lib = _lib.load()
    need = lib.mt_layer_norm_backward_workspace_bytes
    for T in (1, 3, 511, 513, 65536):
        for H in (1, 64, 1024, 1025, 4096, 32768):
            rows = max(4, min(-(-T // 4), 512) * 4) if H <= 1024 else min(T, 512)
            assert need(T, H) == 2 * rows * H * 4
    assert need(0, 64) == need(BIG, 64) == need(4, BIG) == need(-1, 4) == 0
    n = need(10, 64)
    assert lib.mt_layer_norm_backward(ctypes.byref(norm()), P, n - 1, None) == 2
    assert lib.mt_layer_norm_backward(ctypes.byref(norm()), None, n, None) == 1
    assert lib.mt_layer_norm_backward(None, P, n, None) == lib.mt_layer_norm_forward(None, None) == 1
    assert lib.mt_layer_norm_forward(ctypes.byref(norm(T=0, x=None)), None) == 0
    assert lib.mt_layer_norm_backward(ctypes.byref(norm(T=0, dnormed=None)), None, 0, None) == 0


def test_the_nodes_are_there_and_fail_loudly(monkeypatch):
    ops = _lib.torch_ops()
    assert ops is _lib.torch_ops()
    with pytest.raises(_lib.FlceError, match="null coefficients"):
        ops.orthogonalize(torch.zeros(4, 4), 0, 5, 1e-7, 0)
    monkeypatch.setattr(_lib, "_torch_ops", None)
    monkeypatch.setitem(sys.modules, "mini_trainer_amd._mt_torch", None)  # (as if it were not there)
    with pytest.raises(_lib.FlceError, match="not built"):
        _lib.torch_ops()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True), (True, True)])
def test_gradients_go_to_the_tensors_that_are_there(residual, weight, bias):
    """No rows: nothing is launched, so that the nodes' edges can be looked at here."""
    leaf = lambda there, *shape: torch.zeros(*shape, requires_grad=True) if there else None  # noqa: E731
    given = leaf(True, 0, 8), leaf(residual, 0, 8), leaf(weight, 8), leaf(bias, 8)
    outs = _lib.torch_ops().layer_norm(*given, 1e-5, 1.0, 0.5, True, 0)
    assert len(outs) == 1 + residual
    leaves = [t for t in given if t is not None]
    both = torch.autograd.grad(outs, leaves, [torch.zeros_like(t) for t in outs], retain_graph=True)
    alone = [torch.autograd.grad(outs[0], t, outs[0], retain_graph=True)[0] for t in leaves]
    for t, a, b in zip(leaves, both, alone):
        assert a.shape == b.shape == t.shape and not a.any() and not b.any()


def test_the_references_agree_with_torch():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(30, 8, generator=g, dtype=torch.float32)
    ids = torch.randint(0, 30, (50,), generator=g)
    d = torch.randn(50, 8, generator=g)
    leaf = w.double().requires_grad_(True)
    out = 0.7 * torch.nn.functional.embedding(ids, leaf, padding_idx=4)
    (grad,) = torch.autograd.grad(out, leaf, d.double())
    got = ref.embedding(ids, w, d, 0.7, 4)
    assert torch.allclose(got["out"][0], out) and torch.allclose(got["dweight"][0], grad)
    x, r, u0, u1 = (torch.randn(6, 16, generator=g) for _ in range(4))
    wt, b = torch.randn(16, generator=g), torch.randn(16, generator=g)
    at = [t.double().requires_grad_(True) for t in (x, r, wt, b)]
    h = 0.9 * at[1] + 0.3 * at[0]
    y = torch.nn.functional.layer_norm(h, (16,), at[2], at[3], 1e-5)
    grads = torch.autograd.grad([y, h], at, [u0.double(), u1.double()])
    got = ref.layer_norm(x, r, wt, b, u0, u1, 1e-5, 0.3, 0.9)
    for name, value in zip(("normed", "residual", "dx", "dresidual", "dweight", "dbias"), (y, h, *grads)):
        assert torch.allclose(got[name][0], value), name

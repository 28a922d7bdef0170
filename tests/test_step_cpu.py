"""Attention, norms and clipping without a GPU: what the entry points refuse, in
Python and in the C ABI, before anything is launched; the references that the GPU
tests use, against torch's own functions and autograd."""
from __future__ import annotations

import ctypes
import inspect
import math

import pytest
import torch

import mini_trainer_amd as mt
from mini_trainer_amd import _lib, grad_clip
from mini_trainer_amd._lib import AttnArgs, NormArgs

import step_reference as ref

P = 1 << 20  # an aligned address that no checked call reads


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 2, 64)
    w = torch.zeros(64)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.packed_attention(t, t, t, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.residual_rms_norm(t[:, 0], t[:, 0], w)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.clip_gradients_([w], 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        mt.packed_attention_plan(torch.tensor([0, 4], dtype=torch.int32), 4, device="cpu")


def test_plan_arguments_are_checked_before_the_device():
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for kw, err in ((dict(window=0), ValueError), (dict(window=-3), ValueError),
                    (dict(prefix_lens=torch.zeros(2, dtype=torch.int32)), ValueError),
                    (dict(prefix_lens=torch.zeros(1)), TypeError)):
        with pytest.raises(err):
            mt.packed_attention_plan(cu, 4, **kw)
    with pytest.raises(TypeError):
        mt.packed_attention_plan(cu.float(), 4)
    with pytest.raises(ValueError):
        mt.packed_attention_plan(cu[:0], 4)
    with pytest.raises(ValueError):
        mt.packed_attention_plan(cu, -1)


def test_clip_arguments():
    with pytest.raises(ValueError, match="norm_type"):
        mt.clip_gradients_([torch.zeros(3)], 1.0, norm_type=1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            mt.clip_gradients_([torch.zeros(3)], bad)
    # no gradients: torch's own answer, without a device
    assert mt.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0).item() == 0.0
    names = list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters)
    assert list(inspect.signature(mt.clip_grad_norm_).parameters) == names


def test_gradient_layouts():
    x = torch.zeros(6, 8)
    assert grad_clip._layout(x) == (0, 0)
    assert grad_clip._layout(x.T) == (0, 0)
    assert grad_clip._layout(x.view(2, 3, 8).permute(2, 0, 1)) == (0, 0)
    assert grad_clip._layout(x[:, :5]) == (5, 8)
    assert grad_clip._layout(x[:, :5].T) == (5, 8)
    assert grad_clip._layout(x.view(2, 3, 8)[:, :, :4]) == (4, 8)
    assert grad_clip._layout(x[::2]) == (8, 16)
    assert grad_clip._layout(x[:, ::2]) == (1, 2)
    assert grad_clip._layout(x.view(2, 3, 8)[:, :2]) == (16, 24)
    for bad in (x.view(2, 3, 8)[:, :2, :4], x[:1].expand(6, 8), torch.zeros(9).as_strided((3, 3), (2, 1))):
        with pytest.raises(ValueError):
            grad_clip._layout(bad)


def attn(**kw):
    a = AttnArgs()
    base = dict(q=P, k=P, v=P, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, plan=P, q_t=256, q_h=64,
                k_t=128, k_h=64, v_t=128, v_h=64, dout_t=256, dout_h=64, T=10, S=2, heads=4,
                kv_heads=2, head_dim=64, window=2 ** 31 - 1, scale=0.125, softcap=0.0, dtype=1)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), 1), (dict(T=-1), 1), (dict(T=2 ** 31), 1), (dict(S=-1), 1), (dict(heads=3), 1),
    (dict(heads=0), 1), (dict(kv_heads=0), 1), (dict(head_dim=4), 3), (dict(head_dim=136), 3),
    (dict(head_dim=0), 3), (dict(window=0), 1), (dict(window=2 ** 31), 1), (dict(scale=0.0), 1),
    (dict(scale=-1.0), 1), (dict(scale=math.inf), 1), (dict(scale=math.nan), 1),
    (dict(softcap=-1.0), 1), (dict(softcap=math.nan), 1), (dict(q_t=4), 1), (dict(k_h=-8), 1),
    (dict(v_t=(1 << 24) + 8), 3), (dict(q=None), 1), (dict(k=P + 8), 1), (dict(lse=None), 1),
    (dict(plan=None), 1), (dict(T=1 << 28, heads=4096, kv_heads=2), 3),
    (dict(out_lo=P + 8), 1),
    (dict(scale=10.0, softcap=1e-38), 1),                     # their quotient is infinite
    (dict(T=1 << 24, S=1 << 19, heads=32, kv_heads=8), 3),    # 2^32 threads and more
    (dict(T=1 << 24, S=1 << 22, heads=4, kv_heads=4), 3),
])
def test_attention_host_checks(kw, code):
    lib = _lib.load()
    a = attn(**kw)
    assert lib.mt_attn_forward(ctypes.byref(a), None) == code
    assert lib.mt_flce_last_error()
    assert lib.mt_attn_backward(ctypes.byref(a), P, 1 << 40, None) == code


def test_attention_backward_and_plan_host_checks():
    lib = _lib.load()
    for kw in (dict(dout=None), dict(dq=None), dict(dk=P + 4), dict(dout_t=12)):
        assert lib.mt_attn_backward(ctypes.byref(attn(**kw)), P, 1 << 40, None) == 1
    a = attn()
    need = lib.mt_attn_backward_workspace_bytes(ctypes.byref(a))
    assert need >= 4 * 10 * 4
    assert lib.mt_attn_backward(ctypes.byref(a), P, need - 1, None) == 2
    assert lib.mt_attn_backward(ctypes.byref(a), None, need, None) == 1
    assert lib.mt_attn_forward(None, None) == 1
    # nothing to do: no launch
    assert lib.mt_attn_forward(ctypes.byref(attn(T=0, q=None, out=None, plan=None)), None) == 0
    nbytes = lib.mt_attn_plan_bytes(1000, 3)
    tiles = -(-1000 // 128) + 3 + 1
    assert nbytes == 4 * (16 + 2 * 8 * tiles + 3 + 2)
    assert lib.mt_attn_plan(P, None, 3, 1000, 1, P, nbytes - 1, P, None) == 2
    assert lib.mt_attn_plan(P, None, 3, 1000, 0, P, nbytes, P, None) == 1
    assert lib.mt_attn_plan(None, None, 3, 1000, 1, P, nbytes, P, None) == 1
    assert lib.mt_attn_plan(P, None, -1, 1000, 1, P, nbytes, P, None) == 1
    assert lib.mt_attn_plan_bytes(-1, 0) == 0


def norm(**kw):
    a = NormArgs()
    base = dict(x=P, residual=P, weight=P, normed=P, new_residual=P, rstd=P, dnormed=P,
                dresidual_out=P, dx=P, dresidual=P, dweight=P, x_t=64, residual_t=64, gate_t=0,
                dnormed_t=64, dresidual_out_t=64, T=10, H=64, eps=1e-6, block_scale=1.0,
                residual_scale=1.0, weight_offset=0.0, gate_mode=0, dtype=1)
    for name, value in {**base, **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=7), 1), (dict(T=-1), 1), (dict(H=0), 1), (dict(H=40000, x_t=40000), 3),
    (dict(gate_mode=1), 1), (dict(gate=P), 1), (dict(gate=P, gate_mode=4), 1),
    (dict(gate=P, gate_mode=3, gate_t=60), 1), (dict(gate=P, gate_mode=2, gate_t=0), 1),
    (dict(eps=-1.0), 1), (dict(eps=math.nan), 1), (dict(block_scale=math.inf), 1),
    (dict(x_t=63), 1), (dict(residual_t=8), 1), (dict(weight=None), 1), (dict(rstd=None), 1),
    (dict(new_residual=P + 1), 1),
])
def test_norm_host_checks(kw, code):
    lib = _lib.load()
    assert lib.mt_norm_forward(ctypes.byref(norm(**kw)), None) == code
    assert lib.mt_norm_backward(ctypes.byref(norm(**kw)), P, 1 << 40, None) == code


def test_rows_beyond_one_launch():
    lib = _lib.load()
    assert lib.mt_norm_forward(ctypes.byref(norm(T=1 << 26)), None) == 3


def test_plans_of_several_rows():
    """Rows are documents of their own, and so are the parts of a row whose
    position_ids restart."""
    from mini_trainer_amd.decoder import minibatch_plans

    tokens = torch.zeros(2, 6, dtype=torch.int64)
    for pos, want in ((None, [0, 6, 12]), (torch.arange(6)[None], [0, 6, 12]),
                      (torch.tensor([[0, 1, 2, 0, 1, 2], [3, 4, 0, 1, 2, 3]]), [0, 3, 6, 8, 12])):
        assert minibatch_plans(tokens, pos, None)._args[0].tolist() == want
    assert minibatch_plans(tokens[:1], torch.tensor([[0, 1, 0, 1, 2, 3]]), None)._args[0].tolist() == [0, 2, 6]
    assert minibatch_plans(tokens[:1], None, None)._args[0].tolist() == [0, 6]


def test_norm_backward_workspace():
    lib = _lib.load()
    need = lib.mt_norm_backward_workspace_bytes(10, 64)
    assert need > 0
    assert lib.mt_norm_backward(ctypes.byref(norm()), P, need - 1, None) == 2
    assert lib.mt_norm_backward(ctypes.byref(norm(dnormed=None)), P, need, None) == 1
    assert lib.mt_norm_backward(ctypes.byref(norm(x=None, post_weight=P)), P, need, None) == 1
    assert lib.mt_norm_forward(ctypes.byref(norm(normed=None)), None) == 1
    assert lib.mt_norm_forward(ctypes.byref(norm(T=0, x=None)), None) == 0


def table(entries):
    n = len(entries)
    ptr, numel, cols, pitch, code = zip(*entries) if n else ((),) * 5
    return ((ctypes.c_void_p * n)(*ptr), (ctypes.c_int64 * n)(*numel), (ctypes.c_int64 * n)(*cols),
            (ctypes.c_int64 * n)(*pitch), (ctypes.c_int32 * n)(*code))


@pytest.mark.parametrize("entry", [
    (P, 8, 0, 0, 9), (None, 8, 0, 0, 1), (P, -1, 0, 0, 1), (P + 1, 8, 0, 0, 1), (P + 2, 8, 0, 0, 0),
    (P, 8, 3, 4, 1), (P, 8, 4, 3, 1), (P, 8, -1, 0, 1),
])
def test_clip_host_checks(entry):
    lib = _lib.load()
    t = table([(P, 8, 0, 0, 0), entry])
    assert lib.mt_grad_norm(*t, 2, 0, 1.0, P, 1 << 30, P, None) == 1
    assert lib.mt_grad_scale(*t, 2, P, None) == 1


def test_clip_workspace():
    lib = _lib.load()
    t = table([(P, 1 << 20, 0, 0, 1), (P, 100, 10, 20, 0)])
    need = lib.mt_grad_norm_workspace_bytes(t[1], 2)
    assert need >= 16 and need % 8 == 0
    assert lib.mt_grad_norm(*t, 2, 0, 1.0, P, need - 1, P, None) == 2
    assert lib.mt_grad_norm(*t, 2, 0, -1.0, P, need, P, None) == 1
    assert lib.mt_grad_norm(*t, 2, 0, math.nan, P, need, P, None) == 1
    assert lib.mt_grad_norm(*t, 2, 0, 1.0, None, need, P, None) == 1
    # sums of a large set stay few
    big = (ctypes.c_int64 * 400)(*[10 ** 8] * 400)
    assert lib.mt_grad_norm_workspace_bytes(big, 400) <= 8 * (16384 + 400)


@pytest.mark.parametrize("softcap", [None, 2.0])
def test_attention_reference_is_torchs(softcap):
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(9, h, 8, generator=g, dtype=torch.float64) for h in (4, 2, 2, 4))
    mask = ref.seen_mask([4, 3], 9, window=3, prefix=[2, 0])
    assert mask[0].tolist() == [True, True] + [False] * 7  # the prefix is seen from before it
    assert mask[3].tolist() == [False, True, True, True] + [False] * 5
    assert not mask[7:].any() and not mask[:, 7:].any()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    z = torch.einsum("ihd,jhd->hij", leaves[0], leaves[1].repeat_interleave(2, 1)) * 8 ** -0.5
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    z = z.masked_fill(~mask, -math.inf)[:, :7, :7]
    out = torch.einsum("hij,jhd->ihd", torch.softmax(z, -1), leaves[2].repeat_interleave(2, 1)[:7])
    want = torch.autograd.grad(out, leaves, do[:7])
    got = ref.attention(q, k, v, do, mask, softcap=softcap)
    assert torch.allclose(got["out"][0][:7], out, atol=1e-12) and not got["out"][0][7:].any()
    for name, w in zip(("dq", "dk", "dv"), want):
        assert torch.allclose(got[name][0], w, atol=1e-12), name


@pytest.mark.parametrize("gate", ["none", "channel", "token", "element"])
@pytest.mark.parametrize("post", [False, True])
def test_norm_reference_is_torchs(gate, post):
    g = torch.Generator().manual_seed(2)
    shapes = {"none": None, "channel": (6,), "token": (5, 1), "element": (5, 6)}
    t = {n: torch.randn(s, generator=g, dtype=torch.float64) for n, s in
         (("x", (5, 6)), ("residual", (5, 6)), ("weight", (6,)))}
    if post:
        t["post_weight"] = torch.randn(6, generator=g, dtype=torch.float64)
    if shapes[gate]:
        t["gate"] = torch.randn(shapes[gate], generator=g, dtype=torch.float64)
    dy, dh = torch.randn(2, 5, 6, generator=g, dtype=torch.float64)
    leaf = {n: v.clone().requires_grad_(True) for n, v in t.items()}
    rms = torch.nn.functional.rms_norm
    u = rms(leaf["x"], (6,), leaf["post_weight"] + 1.0, 1e-3) if post else leaf["x"]
    h = 0.7 * leaf["residual"] + 0.3 * leaf.get("gate", 1.0) * u
    y = rms(h, (6,), leaf["weight"] + 1.0, 1e-3)
    want = torch.autograd.grad([y, h], list(leaf.values()), [dy, dh])
    got = ref.residual_norm(t["x"], t["residual"], t["weight"], dy, dh, 1e-3, t.get("post_weight"),
                            t.get("gate"), 0.3, 0.7, 1.0)
    assert torch.allclose(got["normed"][0], y) and torch.allclose(got["residual"][0], h)
    for name, w in zip(leaf, want):
        assert torch.allclose(got["d" + name][0], w), name

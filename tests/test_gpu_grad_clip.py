"""Gradient norm and clipping on the GPU.  The norm is the fp32 rounding of a
64-bit sum (2^-24, and 2^-40 for the sum's own order); a clipped element is its
value times a coefficient that is right to two fp32 roundings, rounded once more
to its type."""
from __future__ import annotations

import math

import pytest
import torch

from mini_trainer_amd import clip_grad_norm_, clip_gradients_, patch_target_module

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def make(shapes, seed=0, std=1e-2):
    """Alternating bf16 and fp32 gradients."""
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to((torch.bfloat16, torch.float32)[i % 2]).cuda()
            for i, s in enumerate(shapes)]


def norm_of(gs, kind=2.0):
    flat = torch.cat([g.double().cpu().flatten() for g in gs])
    return float(flat.norm() if kind == 2.0 else flat.abs().max())


def check(gs, max_norm, kind=2.0, **kw):
    before = [g.clone() for g in gs]
    want = norm_of(gs, kind)
    norm = clip_gradients_(gs, max_norm, kind, **kw)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.is_cuda
    assert abs(norm.item() - want) <= (F32 + 2.0 ** -40) * want
    c = max_norm / (want + 1e-6)
    for g, b in zip(gs, before):
        if c >= 1.0:
            assert torch.equal(g, b)
            continue
        v = b.double() * c
        u = torch.finfo(g.dtype).eps / 2
        # (below the type's normal numbers a rounding is half the smallest step)
        tiny = torch.finfo(g.dtype).tiny * u
        assert ((g.double() - v).abs() <= (u + 3 * F32) * v.abs() + tiny).all()
    return norm


SHAPES = [(1,), (7,), (8,), (513, 3), (128, 64), (1, 1, 5), (16384,), (16385,), (40000,), (2, 3, 4, 5)]


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.0, 1e-3, 0.5, 1e6])
def test_matches_the_definition(gpu, kind, max_norm):
    check(make(SHAPES), max_norm, kind)


def test_many_tensors_and_a_large_one(gpu):
    check(make([(1 + 37 * i % 300, 3) for i in range(400)], seed=1), 0.1)
    check(make([(9_000_001,), (3,), (5_000_000,)], seed=2), 1.0)
    check(make([(3,)] * 80, seed=3), 1e-3)
    check(make([(3,)] * 81, seed=4), 1e-3)


def test_layouts(gpu):
    base = make([(64, 96), (64, 96)], seed=5)
    odd = torch.randn(1001, device=gpu).to(torch.bfloat16)
    gs = [base[0][:, :40], base[0][:, 40:81], base[1].T, odd[1:1000], base[1].new_zeros(0),
          torch.randn(6, 5, 4, device=gpu).permute(2, 0, 1), torch.randn((), device=gpu)]
    untouched = base[0][:, 81:].clone(), odd[[0, 1000]].clone()
    check(gs, 0.01)
    assert torch.equal(base[0][:, 81:], untouched[0]) and torch.equal(odd[[0, 1000]], untouched[1])


def test_the_same_gradient_twice_counts_once(gpu):
    g = make([(100,), (50,)], seed=6)
    again = [g[0], g[1], g[0], g[1].view(5, 10), g[0][:]]
    want = norm_of(g)
    before = [t.clone() for t in g]
    norm = clip_gradients_(again, want / 2)
    assert abs(norm.item() - want) <= 2 * F32 * want
    c = (want / 2) / (want + 1e-6)
    for t, b in zip(g, before):
        u = torch.finfo(t.dtype).eps / 2
        assert ((t.double() - b.double() * c).abs() <= (u + 3 * F32) * b.double().abs() * c).all()


def test_refusals(gpu):
    x = torch.randn(64, 32, device=gpu)
    for bad in ([x[:40], x[30:]], [x, x[:, :4]], [x[:, :20], x[:, 16:]], [x.flatten()[:9], x.flatten()[8:]],
                [x[:, :8], x[:, 8:16], x[:, 12:20]], [x[:1].expand(4, 32)], [x, x.T[:3]]):
        before = x.clone()
        with pytest.raises(ValueError):
            clip_gradients_(bad, 1e-3)
        assert torch.equal(x, before)
    with pytest.raises(TypeError):
        clip_gradients_([x.half()], 1.0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        clip_gradients_([x, x.cpu()], 1.0)
    with pytest.raises(TypeError):
        clip_gradients_([x.to_sparse()], 1.0)


@pytest.mark.parametrize("kind", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_nonfinite(gpu, kind, bad):
    gs = make([(40000,), (70,)], seed=7)
    gs[0][12345] = bad
    held = [g.clone() for g in gs]
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_gradients_(gs, 1.0, kind, error_if_nonfinite=True)
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(gs, held))
    norm = clip_gradients_(gs, 1.0, kind)
    if math.isnan(bad):
        assert norm.isnan() and all(g.isnan().all() for g in gs)
    else:  # the coefficient is 0: what is finite becomes 0, the infinity NaN
        assert norm.item() == math.inf
        assert gs[0][12345].isnan() and not gs[1].any()
        assert not torch.cat([gs[0][:12345], gs[0][12346:]]).any()


def test_range_of_the_squares(gpu):
    """Elements whose squares leave fp32's range at either end."""
    for size in (1e30, 1e-30):
        gs = make([(1000,), (999,)], seed=8, std=size)
        norm = check(gs, size)
        assert 0.0 < norm.item() < math.inf


def test_repeats_and_streams(gpu):
    shapes = [(5000, 7), (123456,), (64,)]
    want = None
    for stream in (None, torch.cuda.Stream(), torch.cuda.Stream()):
        gs = make(shapes, seed=9)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            norm = clip_gradients_(gs, 0.01)
        torch.cuda.synchronize()
        want = want or (norm, gs)
        assert torch.equal(norm, want[0]) and all(torch.equal(a, b) for a, b in zip(gs, want[1]))


def test_clip_grad_norm_is_torchs(gpu, monkeypatch):
    """Installed in place of torch's function, as train.py:24 calls it: fp32
    gradients get torch's norm and values to fp32 rounding."""
    monkeypatch.setattr(torch.nn.utils, "clip_grad_norm_", torch.nn.utils.clip_grad_norm_)
    original = torch.nn.utils.clip_grad_norm_
    params = [torch.nn.Parameter(torch.randn(n, device=gpu)) for n in (3000, 17, 1)]
    other = [torch.nn.Parameter(p.detach().clone()) for p in params]
    params.append(torch.nn.Parameter(torch.zeros(2, device=gpu)))  # without a gradient
    for p, q in zip(params, other):
        p.grad = torch.randn_like(p)
        q.grad = p.grad.clone()
    want = original(other, 0.7)
    patch_target_module("torch.nn.utils.clip_grad_norm_", clip_grad_norm_)
    got = torch.nn.utils.clip_grad_norm_(iter(params), 0.7, foreach=True)
    assert abs(got.item() - want.item()) <= 64 * F32 * want.item()
    for p, q in zip(params, other):
        assert torch.allclose(p.grad, q.grad, rtol=64 * F32, atol=0)
    assert params[-1].grad is None
    one = torch.nn.Parameter(torch.ones(4, device=gpu))
    one.grad = torch.full((4,), 2.0, device=gpu)
    assert clip_grad_norm_(one, 100.0).item() == 4.0 and one.grad.tolist() == [2.0] * 4


def test_version_counter_and_empty(gpu):
    g = make([(10,)], seed=10)[0]
    v = g._version
    clip_gradients_([g], 1e-3)
    assert g._version > v
    assert clip_gradients_([], 1.0).item() == 0.0
    assert clip_gradients_([torch.zeros(0, device=gpu)], 1.0).item() == 0.0
    z = torch.zeros(5, device=gpu)
    assert clip_gradients_([z], 1.0).item() == 0.0 and not z.any()


def test_captured_and_replayed(gpu):
    gs = make([(3000,), (77, 5), (40000,)], seed=11)
    clip_gradients_(gs, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_gradients_(gs, 0.1)
    for n in range(4):
        new = make([(3000,), (77, 5), (40000,)], seed=40 + n, std=10.0 ** -(n + 1))
        for g, x in zip(gs, new):
            g.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = clip_gradients_(new, 0.1)
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(gs, new))

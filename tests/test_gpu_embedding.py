"""Token embedding on the GPU against its definition in 64 bits (layer_reference.py,
which also derives the tolerances)."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import token_embedding

import layer_reference as ref
from step_reference import assert_within

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


def make(T, V, H, dtype, seed=0, spread=None):
    """ids of Zipf's law (spread: how many ids occur), weight and upstream gradient."""
    g = torch.Generator().manual_seed(seed)
    p = 1.0 / (torch.arange(spread or V, dtype=torch.float64) + 2.7)
    ids = torch.multinomial(p, T, True, generator=g) if T else torch.zeros(0, dtype=torch.int64)
    w, d = (torch.randn(n, H, generator=g).to(dtype).cuda() for n in (V, T))
    return ids.cuda(), w, d


def run(ids, w, d, accumulator=None, **kw):
    leaf = w.detach().requires_grad_(True)
    out = token_embedding(ids, leaf, dw_accumulator=accumulator, **kw)
    (grad,) = torch.autograd.grad(out, leaf, d, allow_unused=accumulator is not None)
    if accumulator is None:
        return {"out": out, "dweight": grad}
    assert grad is None
    return {"out": out, "accumulator": accumulator}


def check(ids, w, d, scale=1.0, padding_idx=None, accumulate=False):
    for acc in [None] + [torch.randn(w.shape, device=w.device)] * accumulate:
        want = ref.embedding(ids, w, d, scale, padding_idx, acc)
        got = run(ids, w, d, acc, scale=scale, padding_idx=padding_idx)
        assert got["out"].shape == ids.shape + (w.shape[1],) and got["out"].dtype == w.dtype
        for name in want:
            assert_within(got[name], want[name], name)


@BOTH
@pytest.mark.parametrize("T,V,H", [(1, 1, 1), (1, 1000, 64), (63, 7, 8), (64, 100, 24), (65, 300, 520),
                                   (300, 50, 1030), (1000, 1000, 128), (2000, 30, 512), (777, 5000, 2056),
                                   (33, 3, 8192)])
def test_matches_the_definition(gpu, T, V, H, dtype):
    ids, w, d = make(T, V, H, dtype, seed=T)
    check(ids, w, d, accumulate=True)
    check(ids.to(torch.int32), w, d, scale=0.37, padding_idx=-1, accumulate=True)


@BOTH
@pytest.mark.parametrize("H", [2, 3, 4, 5, 7, 9, 15, 17, 31, 33, 511, 513, 1023, 1025, 2047, 4095])
def test_widths_of_no_whole_vectors(gpu, H, dtype):
    """The last vector of a row begins within the one before: twice summed, once added."""
    for T, V in ((200, 30), (700, 90)):
        ids, w, d = make(T, V, H, dtype, seed=H)
        check(ids, w, d, scale=1.7, accumulate=True)


@BOTH
@pytest.mark.parametrize("T", [31, 32, 33, 64, 65, 256, 257, 1024, 1025, 5000])
def test_one_id_takes_all_tokens(gpu, T, dtype):
    """A row of many pieces, from the first sorted token on and behind another row's."""
    ids, w, d = make(T, 40, 136, dtype, seed=T)
    check(torch.full_like(ids, 17), w, d, accumulate=True)
    ids = torch.full_like(ids, 256 + 3)  # (its bucket follows that of 3, whose tokens come first)
    ids[::5] = 3
    _, w, d = make(T, 600, 136, dtype, seed=T)
    check(ids, w, d, accumulate=True)


def test_ids_beyond_a_bucket_and_int32_offsets(gpu):
    """More ids than 256 buckets hold, and a weight of more than 2^31 elements."""
    for V, H in ((300_000, 40), (263_001, 9)):
        ids, w, d = make(700, V, H, torch.bfloat16, seed=V)
        ids[:50] += V - 1 - int(ids[:50].max())
        check(ids, w, d, accumulate=True)
    V, H = 2_200_000, 1024
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=gpu)
    ids = torch.tensor([V - 1, 3, V - 1, V - 2], device=gpu)
    w[ids] = torch.randn(4, H, device=gpu).to(w.dtype)
    d = torch.randn(4, H, device=gpu).to(w.dtype)
    got = run(ids, w, d)
    assert torch.equal(got["out"], w[ids])
    rows = torch.stack([d[1], d[3], (d[0].float() + d[2].float()).to(d.dtype)])
    assert torch.equal(got["dweight"][[3, V - 2, V - 1]], rows)
    assert int(got["dweight"].count_nonzero()) == int(rows.count_nonzero())


def test_ids_out_of_range(gpu):
    ids, w, d = make(200, 50, 64, torch.bfloat16)
    bad = ids.clone()
    bad[[0, 63, 64, 199]] = torch.tensor([-1, 50, 2 ** 31 - 1, 2 ** 40], device=gpu)
    with pytest.raises(IndexError, match=r"\[0, 50\)"):
        token_embedding(bad, w)
    token_embedding(ids, w)
    got, want = run(bad, w, d, validate=False), ref.embedding(bad, w, d)
    nan = torch.isnan(want["out"][0])
    assert torch.equal(torch.isnan(got["out"]).cpu(), nan) and int(nan.sum()) == 4 * 64
    assert torch.equal(got["out"].double().cpu()[~nan], want["out"][0][~nan])
    assert_within(got["dweight"], want["dweight"], "dweight")


def test_no_tokens(gpu):
    w = torch.randn(9, 16, device=gpu)
    got = run(torch.zeros(0, dtype=torch.int64, device=gpu), w, w[:0])
    assert got["out"].shape == (0, 16) and not got["dweight"].any()
    acc = torch.ones(9, 16, device=gpu)
    run(torch.zeros((2, 0), dtype=torch.int32, device=gpu), w, w[:0].view(2, 0, 16), acc)
    assert bool((acc == 1).all())


def test_padding_alone_and_none_of_it(gpu):
    ids, w, d = make(100, 30, 32, torch.bfloat16)
    assert not run(torch.full_like(ids, 29), w, d, padding_idx=29)["dweight"].any()
    got = run(ids, w, d, padding_idx=0)
    assert not got["dweight"][0].any() and torch.equal(got["out"], w[ids])
    acc = torch.randn(30, 32, device=gpu)
    first = acc[0].clone()
    run(ids, w, d, acc, padding_idx=0)
    assert torch.equal(acc[0], first)


@BOTH
def test_strides(gpu, dtype):
    ids, w, d = make(300, 90, 40, dtype)
    want = run(ids, w, d)
    wide = torch.randn(90, 57, device=gpu).to(dtype)
    wide[:, 3:43] = w
    dwide = torch.randn(300, 3, 48, device=gpu).to(dtype)
    dwide[:, 1, 1:41] = d
    for weight in (wide[:, 3:43], w.T.contiguous().T):
        for up in (dwide[:, 1, 1:41], d.T.contiguous().T):
            got = run(torch.stack([ids, ids], 1)[:, 1], weight, up)
            assert torch.equal(got["out"], want["out"]) and torch.equal(got["dweight"], want["dweight"])
    acc, strided = torch.zeros(90, 40, device=gpu), torch.zeros(90, 43, device=gpu)
    run(ids, w, d, acc)
    run(ids, w, d, strided[:, 1:41])
    assert torch.equal(acc, strided[:, 1:41]) and not strided[:, 41:].any() and not strided[:, 0].any()
    # a gradient that is one number for all: the row sums of its ids' counts
    leaf = w.detach().requires_grad_(True)
    token_embedding(ids.view(3, 100), leaf).sum().backward()
    counts = torch.bincount(ids, minlength=90).to(dtype)
    assert torch.equal(leaf.grad, counts[:, None].expand(90, 40))


def test_results_repeat(gpu):
    ids, w, d = make(20000, 5000, 256, torch.bfloat16)
    first = run(ids, w, d)
    for _ in range(3):
        again = run(ids, w, d)
        assert torch.equal(again["dweight"], first["dweight"])


def test_frozen_weight_and_no_grad(gpu):
    ids, w, _ = make(10, 20, 16, torch.float32)
    assert not token_embedding(ids, w).requires_grad
    with torch.no_grad():
        assert not token_embedding(ids, w.requires_grad_(True)).requires_grad


def test_another_stream(gpu):
    ids, w, d = make(3000, 700, 512, torch.bfloat16)
    want = run(ids, w, d)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(ids, w, d)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got["out"], want["out"]) and torch.equal(got["dweight"], want["dweight"])


def test_captured(gpu):
    ids, w, d = make(3000, 700, 264, torch.bfloat16)
    acc = torch.zeros(700, 264, device=gpu)
    static = ids.clone()

    def both():
        return run(static, w, d, validate=False)["dweight"], run(static, w, d, acc, validate=False)["out"]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dweight, out = both()
    for seed in range(3):
        ids, _, _ = make(3000, 700, 8, torch.bfloat16, seed=seed, spread=700 if seed else 3)
        static.copy_(ids)
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want, sums = run(ids, w, d), torch.zeros_like(acc)
        run(ids, w, d, sums)
        assert torch.equal(dweight, want["dweight"]) and torch.equal(out, want["out"])
        assert torch.equal(acc, sums)


def test_gradient_against_differences(gpu):
    ids, w, d = make(50, 12, 16, torch.float32)
    grad = run(ids, w, d, scale=1.7)["dweight"]
    step = torch.randn_like(w) * 0.125
    ends = [(token_embedding(ids, w + s * step, scale=1.7).double() * d.double()).sum() for s in (1, -1)]
    # linear in the weight: the difference is exact but for roundings, 2^-23 of each term
    size = (1.7 * (w.abs() + step.abs())[ids] * d.abs()).sum()
    assert abs(float(ends[0] - ends[1]) - 2 * float((grad.double() * step.double()).sum())) <= \
        8 * 2.0 ** -23 * float(size)


def test_captured_beside_an_eager_graph_of_the_leaf(gpu):
    """Refused where the leaf's gradient node belongs to the eager graph's stream; without
    that graph the same capture runs."""
    ids, w, d = make(400, 50, 64, torch.bfloat16)
    leaf = w.detach().requires_grad_(True)
    want, = torch.autograd.grad(token_embedding(ids, leaf), leaf, d)

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            (grad,) = torch.autograd.grad(token_embedding(ids, leaf, validate=False), leaf, d)
        return graph, grad

    alive = token_embedding(ids, leaf, validate=False)
    with pytest.raises(RuntimeError, match="another stream"):
        capture()
    del alive
    graph, grad = capture()
    for _ in range(3):
        grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want)


def test_not_differentiable_twice(gpu):
    ids, w, d = make(40, 50, 64, torch.float32)
    leaf = w.detach().requires_grad_(True)
    d.requires_grad_(True)
    (grad,) = torch.autograd.grad(token_embedding(ids, leaf), leaf, d, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.sum().backward()

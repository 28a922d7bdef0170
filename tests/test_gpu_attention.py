"""Attention over a packed row on the GPU against its definition in 64 bits
(step_reference.py, which also derives the tolerances)."""
from __future__ import annotations

import math

import pytest
import torch

from mini_trainer_amd import packed_attention, packed_attention_plan

import step_reference as ref

pytestmark = pytest.mark.gpu


def cu_of(lengths, device=None):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist() if lengths else [0],
                        dtype=torch.int32, device=device)


def inputs(T, heads, kv_heads, D, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(T, h, D, generator=g) for h in (heads, kv_heads, kv_heads, heads))
    return [t.to(dtype).cuda() for t in (q * spread, k, v, do)]


def run(q, k, v, do, plan, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, plan, **kw)
    grads = torch.autograd.grad(out, leaves, do)
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def check(got, want):
    for name, w in want.items():
        ref.assert_within(got[name], w, name)


CASES = [
    # lengths, T, heads, kv_heads, D, window, prefix, softcap
    ([1], 1, 1, 1, 64, None, None, None),
    ([1, 1, 1], 3, 2, 1, 128, None, None, None),
    ([2, 1, 3], 6, 4, 2, 32, None, None, None),
    ([31, 33], 64, 4, 4, 64, None, None, None),
    ([63, 64, 65], 192, 2, 1, 128, None, None, None),
    ([127, 128, 129], 384, 2, 2, 64, None, None, None),
    ([300], 300, 8, 1, 128, None, None, None),
    ([300], 300, 7, 1, 64, None, [300], None),               # all of it a prefix
    ([130, 200], 340, 6, 2, 128, None, [130, 63], None),
    ([257, 5], 270, 4, 2, 64, 1, None, None),                # a token sees itself
    ([257, 5], 270, 4, 2, 64, 1, [100, 5], None),
    ([257, 70], 330, 4, 2, 128, 64, None, None),
    ([257, 70], 330, 4, 2, 128, 37, [150, 70], 5.0),
    ([0, 200, 0, 0, 9, 0], 215, 2, 1, 64, None, None, 30.0),  # empty documents, rows behind
    ([], 20, 2, 2, 64, None, None, None),                    # no document at all
    ([200], 200, 2, 1, 8, None, None, None),
    ([200], 200, 2, 1, 40, 50, None, 30.0),
    ([200], 200, 3, 3, 120, None, [7], None),
    ([150, 50], 200, 2, 1, 65, None, None, None),            # padded to whole chunks
    ([150, 50], 201, 2, 1, 1, None, None, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"T{c[1]}D{c[4]}w{c[5]}c{c[7]}")
def test_matches_the_definition(gpu, case, dtype):
    lengths, T, heads, kv, D, window, prefix, cap = case
    q, k, v, do = inputs(T, heads, kv, D, dtype)
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=gpu)
    plan = packed_attention_plan(cu_of(lengths, gpu), T, window=window, prefix_lens=pre)
    got = run(q, k, v, do, plan, softcap=cap)
    mask = ref.seen_mask(lengths, T, window, prefix)
    check(got, ref.attention(q, k, v, do, mask, softcap=cap))
    behind = sum(lengths)
    for t in got.values():  # rows behind the last document: exactly zero
        assert not t[behind:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_document_and_many_short_ones(gpu, dtype):
    lengths = [1500] + [1 + (7 * i) % 19 for i in range(150)]
    T = sum(lengths) + 11
    q, k, v, do = inputs(T, 2, 1, 64, dtype, seed=3)
    plan = packed_attention_plan(cu_of(lengths, gpu), T)
    check(run(q, k, v, do, plan), ref.attention(q, k, v, do, ref.seen_mask(lengths, T)))


def test_scores_far_apart(gpu):
    """A running maximum that grows by hundreds from block to block, and rows
    whose first blocks are almost all of the sum."""
    T = 400
    q, k, v, do = inputs(T, 2, 1, 64, torch.bfloat16, seed=4, spread=1.0)
    ramp = torch.linspace(0.5, 40.0, T, device=gpu)[:, None, None]
    for keys in (k * ramp, k * ramp.flip(0)):
        keys = keys.to(torch.bfloat16)
        plan = packed_attention_plan(cu_of([T], gpu), T)
        got = run(q, keys, v, do, plan, scale=0.7)
        check(got, ref.attention(q, keys, v, do, ref.seen_mask([T], T), scale=0.7))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_is_the_difference_quotient(gpu, dtype):
    """(L(x + e d) - L(x - e d)) / 2e against <grad, d>, L in 64 bits from the
    kernel's own definition: the truncation of a smooth L at e = 1e-4 is some
    1e-8, far below the gradients' own tolerances, summed over |d|."""
    lengths, T = [90, 45], 140
    q, k, v, do = inputs(T, 4, 2, 64, dtype, seed=5)
    mask = ref.seen_mask(lengths, T, window=60)
    plan = packed_attention_plan(cu_of(lengths, gpu), T, window=60)
    got = run(q, k, v, do, plan, softcap=20.0)
    want = ref.attention(q, k, v, do, mask, softcap=20.0)
    g = torch.Generator().manual_seed(6)
    base = [t.double().cpu() for t in (q, k, v)]

    def loss(x):
        z = torch.einsum("ihd,jhd->hij", x[0], x[1].repeat_interleave(2, 1)) / 8.0
        z = (20.0 * torch.tanh(z / 20.0)).masked_fill(~mask, -math.inf)[:, :135, :135]
        out = torch.einsum("hij,jhd->ihd", torch.softmax(z, -1), x[2].repeat_interleave(2, 1)[:135])
        return (out * do.double().cpu()[:135]).sum()

    for n, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        e = 1e-4
        moved = [[b + s * e * d if i == n else b for i, b in enumerate(base)] for s in (1, -1)]
        quotient = (loss(moved[0]) - loss(moved[1])) / (2 * e)
        tol = (want[name][1] * d.abs()).sum() + 1e-6 * quotient.abs() + 1e-6
        assert abs(quotient - (got[name].double().cpu() * d).sum()) <= tol, name


def peaked_gradients(q, k, v, do, mask, rounded_out=False):
    """((dq, tolerance), (dk, tolerance)) of one head in 64 bits where all keys of a row
    lie in one block.  There its largest probability is 2^0 to fp32's rounding and
    enters the product with V unrounded, so delta is off by at most
        e = 2^-8 sum over the other keys of p_j |dP_j| + 2^-16 |dO| . |O|
    (the second: O kept to 16 bits; its halves' rounding and the fp32 sums), and
        |error of dS_j| <= 2^-8 |dS_j| + p_j (e + fp32's (D + C) 2^-24 terms).
    rounded_out: the gradients themselves with delta from bf16(O)."""
    D = q.shape[-1]
    scale, F = D ** -0.5, (D + ref.C) * ref.F32
    q, k, v, do = (t.double().cpu() for t in (q, k, v, do))
    p = torch.softmax((scale * q @ k.T).masked_fill(~mask, -math.inf), -1)
    o, dp = p @ v, do @ v.T
    delta = (do * (o.to(torch.bfloat16).double() if rounded_out else o)).sum(1, keepdim=True)
    alone = (mask.sum(1, keepdim=True) > 1).double()  # (one key: dS is exactly 0)
    ds = alone * p * (dp - delta)
    others = torch.where(p == p.amax(1, keepdim=True), torch.zeros(()).double(), p)
    size = do.abs() @ v.abs().T                       # of dP's sum, and of delta's
    e = 2.0 ** -8 * (others * dp.abs()).sum(1, keepdim=True) \
        + 2.0 ** -16 * (do.abs() * o.abs()).sum(1, keepdim=True) + F * (p * size).sum(1, keepdim=True)
    worst = (F * scale * (q.abs() @ k.abs().T)).masked_fill(~mask, 0.0).amax(1, keepdim=True)
    tol = 2.0 ** -8 * ds.abs() + alone * p * (e + F * size + (2 * worst + F) * (dp.abs() + delta.abs()))
    tol = 1.01 * tol + ref.FLOOR * mask  # (products of two errors)
    made = ((scale * ds @ k, scale * tol @ k.abs()), (scale * ds.T @ q, scale * tol.T @ q.abs()))
    return tuple((g, t + 2.0 ** -8 * (g.abs() + t) + ref.F32 * 64 * t) for g, t in made)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_with_one_large_probability(gpu, D):
    lengths = [2] * 20 + [5] * 8 + [40, 64, 1, 33]
    # queries so wide that most rows put nearly all of their probability on one key
    q, k, v, do = inputs(sum(lengths), 4, 4, D, torch.bfloat16, seed=22, spread=6.0)
    mask = ref.seen_mask(lengths, sum(lengths))
    noticed = 0
    got = run(q, k, v, do, packed_attention_plan(cu_of(lengths, gpu), sum(lengths)))
    for h in range(4):
        (dq, dq_tol), (dk, dk_tol) = peaked_gradients(*(t[:, h] for t in (q, k, v, do)), mask)
        ref.assert_within(got["dq"][:, h], (dq, dq_tol), "dq")
        ref.assert_within(got["dk"][:, h], (dk, dk_tol), "dk")
        rounded = peaked_gradients(*(t[:, h] for t in (q, k, v, do)), mask, rounded_out=True)
        noticed += int(((rounded[0][0] - dq).abs() > dq_tol).sum())
    assert noticed > 100  # delta from bf16(O) is beyond the tolerance


def test_strides(gpu):
    """Views of a fused projection, heads first, expanded key heads, odd addresses."""
    T, H, Hk, D = 150, 4, 2, 64
    lengths = [100, 50]
    q, k, v, do = inputs(T, H, Hk, D, torch.bfloat16, seed=7)
    plan = packed_attention_plan(cu_of(lengths, gpu), T)
    want = run(q, k, v, do, plan)
    fused = torch.cat([q.view(T, -1), k.view(T, -1), v.view(T, -1)], 1)
    a, b, c = fused.split([H * D, Hk * D, Hk * D], 1)
    views = (a.view(T, H, D), b.view(T, Hk, D), c.view(T, Hk, D))
    first = tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    odd = []
    for t in (q, k, v):  # two bytes off every boundary
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)
        odd.append(flat[1:].view(t.shape).copy_(t))
    last = tuple(t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in (q, k, v))  # stride(D) != 1
    for other in (views, first, tuple(odd), last):
        got = run(*other, do.transpose(0, 1).contiguous().transpose(0, 1), plan)
        for name in want:
            assert torch.equal(got[name], want[name]), name
    # one key head expanded over the query heads: its gradient is the sum
    one_k, one_v = k[:, :1].detach().requires_grad_(True), v[:, :1].detach().requires_grad_(True)
    ex = packed_attention(q, one_k.expand(T, H, D), one_v.expand(T, H, D), plan)
    gk, gv = torch.autograd.grad(ex, [one_k, one_v], do)
    mqa = run(q, k[:, :1], v[:, :1], do, plan)
    assert torch.equal(ex, mqa["out"])
    w = ref.attention(q, k[:, :1], v[:, :1], do, ref.seen_mask(lengths, T))
    for got_, name in ((gk, "dk"), (gv, "dv")):
        value, tol = w[name]
        # each head's part is rounded before autograd adds four of them
        parts = ref.attention(q, k[:, :1].expand(T, H, D), v[:, :1].expand(T, H, D), do,
                              ref.seen_mask(lengths, T))[name]
        tol = parts[1].sum(1, keepdim=True) + 4 * 2.0 ** -8 * parts[0].abs().sum(1, keepdim=True)
        ref.assert_within(got_, (value, tol), name)
    # an upstream gradient that is one number expanded
    ones = torch.ones((), dtype=torch.bfloat16, device=gpu).expand(T, H, D)
    got = run(q, k, v, ones, plan)
    full = run(q, k, v, ones.contiguous(), plan)
    assert all(torch.equal(got[n], full[n]) for n in got)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_other_documents_stay_apart(gpu, bad):
    """NaN and infinite values of one document, and of the rows behind the last
    one, reach no other document, in either direction."""
    lengths, T = [70, 40, 90], 230
    q, k, v, do = inputs(T, 4, 2, 64, torch.bfloat16, seed=8)
    plan = packed_attention_plan(cu_of(lengths, gpu), T)
    clean = run(q, k, v, do, plan)
    for t in (q, k, v, do):
        t[75:100] = bad
        t[200:] = bad
    got = run(q, k, v, do, plan)
    for name in clean:
        assert torch.equal(got[name][:70], clean[name][:70]), name
        assert torch.equal(got[name][110:200], clean[name][110:200]), name
        assert not got[name][200:].any(), name
    assert got["out"][75:100].isnan().any()


def test_masked_scores_do_not_count(gpu):
    """Keys that a mask hides may score as high as they like."""
    T = 200
    q, k, v, do = inputs(T, 2, 1, 64, torch.bfloat16, seed=9)
    q = q.abs()
    k[150:] = 1e4  # scores of 1e6 for the rows that see them
    plan = packed_attention_plan(cu_of([T], gpu), T)
    got = run(q, k, v, do, plan)
    short = packed_attention_plan(cu_of([150], gpu), T)
    want = run(q, k, v, do, short)
    assert torch.equal(got["out"][:150], want["out"][:150])
    assert torch.equal(got["dq"][:150], want["dq"][:150])


def test_results_repeat(gpu):
    lengths = [900, 13, 400, 1, 77]
    T = sum(lengths)
    q, k, v, do = inputs(T, 8, 2, 128, torch.bfloat16, seed=10)
    first = None
    for _ in range(4):
        plan = packed_attention_plan(cu_of(lengths, gpu), T)
        got = run(q, k, v, do, plan, softcap=30.0)
        first = first or got
        assert all(torch.equal(got[n], first[n]) for n in got)


def test_malformed_boundaries(gpu):
    T = 300
    q, k, v, do = inputs(T, 2, 1, 64, torch.bfloat16, seed=11)
    for bad in ([1, 300], [0, 200, 100, 300], [0, 301], [0, -5], [0, 2 ** 31 - 1], [-2 ** 31, 5],
                [0, 100, -2 ** 31, 300]):
        cu = torch.tensor(bad, dtype=torch.int32)
        for where in (cu, cu.to(gpu)):
            with pytest.raises(ValueError, match="cu_seqlens"):
                packed_attention_plan(where, T)
        plan = packed_attention_plan(cu.to(gpu), T, validate=False)
        got = run(q, k, v, do, plan)
        assert not any(t.any() for t in got.values()), bad
        with pytest.raises(ValueError, match="cu_seqlens"):
            plan.validate()
    cu = cu_of([100, 200], gpu)
    for bad in ([101, 0], [0, -1]):
        pre = torch.tensor(bad, dtype=torch.int32, device=gpu)
        with pytest.raises(ValueError, match="prefix"):
            packed_attention_plan(cu, T, prefix_lens=pre)
        plan = packed_attention_plan(cu, T, prefix_lens=pre, validate=False)
        held = torch.tensor([min(max(bad[0], 0), 100), max(bad[1], 0)], dtype=torch.int32, device=gpu)
        want = run(q, k, v, do, packed_attention_plan(cu, T, prefix_lens=held))
        got = run(q, k, v, do, plan)
        assert all(torch.equal(got[n], want[n]) for n in got)


def test_boundaries_that_no_int32_holds(gpu):
    wrapped = torch.tensor([0, 2 ** 32 + 300])
    for where in (wrapped, wrapped.to(gpu)):
        with pytest.raises(ValueError, match="cu_seqlens"):
            packed_attention_plan(where, 300)
    with pytest.raises(ValueError, match="prefix"):
        packed_attention_plan(cu_of([300], gpu), 300, prefix_lens=torch.tensor([2 ** 32 + 5]))


def test_plans(gpu):
    """Boundaries as int64, on the CPU, as the call's own argument; one plan for
    several layers with their own heads."""
    T, lengths = 260, [100, 160]
    q, k, v, do = inputs(T, 4, 2, 64, torch.bfloat16, seed=12)
    plan = packed_attention_plan(cu_of(lengths, gpu), T)
    want = run(q, k, v, do, plan)
    for other in (packed_attention_plan(cu_of(lengths), T),
                  packed_attention_plan(cu_of(lengths).long(), T),
                  packed_attention_plan(cu_of(lengths, gpu).long(), T, window=10 ** 12),
                  packed_attention_plan(cu_of(lengths, gpu), T, window=T),
                  cu_of(lengths, gpu), cu_of(lengths)):
        got = run(q, k, v, do, other)
        assert all(torch.equal(got[n], want[n]) for n in got)
    q2, k2, v2, do2 = inputs(T, 6, 6, 128, torch.float32, seed=13)
    check(run(q2, k2, v2, do2, plan), ref.attention(q2, k2, v2, do2, ref.seen_mask(lengths, T)))


def test_refusals(gpu):
    T = 32
    q, k, v, _ = inputs(T, 4, 2, 64, torch.bfloat16)
    plan = packed_attention_plan(cu_of([T], gpu), T)
    other = packed_attention_plan(cu_of([T], gpu), T + 1, validate=False)
    wide = torch.zeros(T, 2, 136, device=gpu, dtype=torch.bfloat16)
    for args, kw, err in (
            ((q.half(), k.half(), v.half(), plan), {}, TypeError),
            ((q, k.float(), v, plan), {}, TypeError),
            ((q[:, :3], k, v, plan), {}, ValueError),
            ((q, k[:-1], v[:-1], plan), {}, ValueError),
            ((q, k, v[:, :1], plan), {}, ValueError),
            ((q[0], k, v, plan), {}, ValueError),
            ((q, k, v, other), {}, ValueError),
            ((wide, wide, wide, plan), {}, ValueError),
            ((q, k, v, plan), dict(scale=0.0), ValueError),
            ((q, k, v, plan), dict(scale=-1.0), ValueError),
            ((q, k, v, plan), dict(scale=math.inf), ValueError),
            ((q, k, v, plan), dict(softcap=-2.0), ValueError),
            ((q, k, v, plan), dict(softcap=math.nan), ValueError),
            ((q, k, v.cpu(), plan), {}, RuntimeError)):
        with pytest.raises(err):
            packed_attention(*args, **kw)
    empty = torch.zeros(0, 4, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    e_plan = packed_attention_plan(cu_of([], gpu), 0)
    out = packed_attention(empty, empty, empty, e_plan)
    out.sum().backward()
    assert out.shape == (0, 4, 64) and empty.grad.shape == (0, 4, 64)


def test_partial_gradients_and_no_grad(gpu):
    T = 100
    q, k, v, do = inputs(T, 4, 2, 64, torch.bfloat16, seed=14)
    plan = packed_attention_plan(cu_of([60, 40], gpu), T)
    want = run(q, k, v, do, plan)
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v, plan), want["out"])
    for n, name in enumerate(("dq", "dk", "dv")):
        leaves = [t.detach().requires_grad_(i == n) for i, t in enumerate((q, k, v))]
        out = packed_attention(*leaves, plan)
        out.backward(do)
        assert torch.equal(leaves[n].grad, want[name])
        assert all(t.grad is None for i, t in enumerate(leaves) if i != n)


def test_another_stream_and_two_calls_at_once(gpu):
    T = 700
    a = inputs(T, 8, 2, 128, torch.bfloat16, seed=15)
    b = inputs(T, 4, 4, 64, torch.bfloat16, seed=16)
    plan = packed_attention_plan(cu_of([500, 200], gpu), T)
    want = [run(*a, plan), run(*b, plan, softcap=10.0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, x, kw in zip(streams, (a, b), ({}, {"softcap": 10.0})):
        with torch.cuda.stream(s):
            got.append(run(*x, plan, **kw))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(g[n], w[n]) for n in g)


def test_captured_and_replayed(gpu):
    """Plan, forward and backward in a graph, replayed over new inputs and new
    boundaries with eager work between the replays."""
    T = 500
    q, k, v, do = inputs(T, 4, 2, 64, torch.bfloat16, seed=17)
    cu = cu_of([300, 150], gpu)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def step():
        plan = packed_attention_plan(cu, T, validate=False)
        out = packed_attention(*leaves, plan, softcap=20.0)
        return (out,) + torch.autograd.grad(out, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        new = inputs(T, 4, 2, 64, torch.bfloat16, seed=20 + n)
        bounds = [100 + 90 * n, 60]
        with torch.no_grad():
            for t, x in zip((*leaves, do), new):
                t.copy_(x)
        cu.copy_(cu_of(bounds, gpu))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = run(*new, packed_attention_plan(cu_of(bounds, gpu), T), softcap=20.0)
        for g, w in zip(got, want.values()):
            assert torch.equal(g, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_as_far_apart_as_they_may_be(gpu, dtype):
    """2^24 elements: the last row of a tile lies just below 4 GiB from its first."""
    T, pitch = 140, 1 << 24
    big = torch.empty(T * pitch, dtype=dtype, device=gpu)
    q, k, v, do = inputs(T, 1, 1, 128, dtype, seed=19)
    plan = packed_attention_plan(cu_of([T], gpu), T)
    want = run(q, k, v, do, plan)
    views = [big.as_strided((T, 1, 128), (pitch, 128, 1), 128 * i) for i in range(4)]
    for view, t in zip(views, (q, k, v, do)):
        view.copy_(t)
    got = run(*views, plan)
    assert all(torch.equal(got[n], want[n]) for n in got)


@pytest.mark.parametrize("lengths,heads", [
    ([2000], 32),                              # divided by cost, 256 tiles x key heads
    ([3] * 20 + [2000] + [128] * 120, 32),     # by cost, the heavy document's tiles of 2500 only
    ([2000] * 4, 128)], ids=["one", "heavy", "number"])  # by the number of tiles
def test_parts_of_divided_heads_find_their_places(gpu, lengths, heads):
    """Every document's results against those it has alone, in two of 16 key heads."""
    kv, G, T = 16, heads // 16, sum(lengths)
    q, k, v, do = inputs(T, heads, kv, 32, torch.float32, seed=21)
    got = run(q, k, v, do, packed_attention_plan(cu_of(lengths, gpu), T))
    at = 0
    for n in lengths:
        rows = slice(at, at + n)
        at += n
        if n < 2000 and at < T:
            continue  # (the heavy ones and the last)
        mask = ref.seen_mask([n], n)
        for h in (0, 15):
            kh, qh = slice(h, h + 1), slice(G * h, G * h + G)
            want = ref.attention(q[rows, qh], k[rows, kh], v[rows, kh], do[rows, qh], mask)
            check({name: t[rows, qh if name in ("out", "dq") else kh] for name, t in got.items()}, want)


def test_rows_beyond_32_bit_offsets(gpu):
    """A cache of rows whose addresses pass 4 GiB: only the tile's own rows are
    reached with 32-bit offsets."""
    T, pitch = 700, (1 << 24) // 4
    big = torch.zeros(T * pitch, dtype=torch.bfloat16, device=gpu)
    q, k, v, do = inputs(T, 2, 1, 64, torch.bfloat16, seed=18)
    plan = packed_attention_plan(cu_of([T], gpu), T)
    want = run(q, k, v, do, plan)
    kk = big.as_strided((T, 1, 64), (pitch, 64, 1))
    vv = big.as_strided((T, 1, 64), (pitch, 64, 1), 64)
    qq = big.as_strided((T, 2, 64), (pitch, 64, 1), 128)
    kk.copy_(k), vv.copy_(v), qq.copy_(q)
    got = run(qq, kk, vv, do, plan)
    assert all(torch.equal(got[n], want[n]) for n in got)

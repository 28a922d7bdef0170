"""Packed attention with the many workgroups of ordinary sizes, whose rows are whole
tiles (more than 512 of them; calls with fewer are cut in halves), in bf16 against the
definition in 64 bits, in some key heads and all their query heads.  Tolerances:
step_reference.py."""
from __future__ import annotations

import math

import pytest
import torch

from mini_trainer_amd import packed_attention, packed_attention_plan

import step_reference as ref

pytestmark = pytest.mark.gpu

HEADS, KV = 64, 16
G = HEADS // KV
LENGTHS = [700, 1, 333, 129]
T = sum(LENGTHS) + 37  # rows behind the last document; no document ends with a tile


def cu_of(lengths, device):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)


def inputs(D, seed, tokens=T, heads=HEADS, kv=KV, spread=2.0):
    assert -(-tokens // 128) * heads > 512
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(tokens, h, D, generator=g) for h in (heads, kv, kv, heads))
    return [t.to(torch.bfloat16).cuda() for t in (q * spread, k, v, do)]


def run(q, k, v, do, plan, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, plan, **kw)
    grads = torch.autograd.grad(out, leaves, do)
    return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]}


def check_heads(got, q, k, v, do, mask, heads=(0, 13), **kw):
    group = q.shape[1] // k.shape[1]
    for h in heads:
        kh, qh = slice(h, h + 1), slice(group * h, group * h + group)
        want = ref.attention(q[:, qh], k[:, kh], v[:, kh], do[:, qh], mask, **kw)
        for name, t in got.items():
            ref.assert_within(t[:, qh if name in ("out", "dq") else kh], want[name], f"{name} of head {h}")


@pytest.mark.parametrize("softcap", [None, 5.0])
@pytest.mark.parametrize("window,prefix", [(None, None), (200, None), (None, [333, 1, 0, 129]),
                                           (150, [400, 0, 333, 60]), (1, None)])
@pytest.mark.parametrize("D", [64, 128])
def test_matches_the_definition(gpu, D, window, prefix, softcap):
    q, k, v, do = inputs(D, seed=1)
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device=gpu)
    plan = packed_attention_plan(cu_of(LENGTHS, gpu), T, window=window, prefix_lens=pre)
    got = run(q, k, v, do, plan, softcap=softcap)
    check_heads(got, q, k, v, do, ref.seen_mask(LENGTHS, T, window, prefix), softcap=softcap)
    for t in got.values():
        assert not t[sum(LENGTHS):].any()


@pytest.mark.parametrize("D", [40, 80, 96])
def test_other_widths(gpu, D):
    q, k, v, do = inputs(D, seed=2)
    plan = packed_attention_plan(cu_of(LENGTHS, gpu), T)
    check_heads(run(q, k, v, do, plan), q, k, v, do, ref.seen_mask(LENGTHS, T), heads=(7,))


def test_one_long_document(gpu):
    """Many key blocks and running maxima, 32 tiles of one head after another."""
    n, heads = 4090, 32
    q, k, v, do = inputs(128, seed=3, tokens=n + 6, heads=heads, kv=heads)
    plan = packed_attention_plan(cu_of([n], gpu), n + 6)
    check_heads(run(q, k, v, do, plan), q, k, v, do, ref.seen_mask([n], n + 6), heads=(5, 30))


def test_scores_far_apart(gpu):
    """A running maximum that grows by hundreds from block to block, or not at all."""
    q, k, v, do = inputs(64, seed=4, spread=1.0)
    ramp = torch.linspace(0.5, 40.0, T, device=gpu)[:, None, None]
    plan = packed_attention_plan(cu_of([T], gpu), T)
    for keys in ((k * ramp).to(k.dtype), (k * ramp.flip(0)).to(k.dtype)):
        check_heads(run(q, keys, v, do, plan, scale=0.7), q, keys, v, do, ref.seen_mask([T], T),
                    heads=(9,), scale=0.7)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_other_documents_stay_apart(gpu, bad):
    q, k, v, do = inputs(64, seed=5)
    plan = packed_attention_plan(cu_of(LENGTHS, gpu), T)
    clean = run(q, k, v, do, plan)
    for t in (q, k, v, do):
        t[710:900] = bad          # within the third document
        t[sum(LENGTHS):] = bad    # behind the last one
    got = run(q, k, v, do, plan)
    for name in clean:
        assert torch.equal(got[name][:701], clean[name][:701]), name
        assert torch.equal(got[name][1034:sum(LENGTHS)], clean[name][1034:sum(LENGTHS)]), name
        assert not got[name][sum(LENGTHS):].any(), name
    assert got["out"][710:900].isnan().any()


def test_strides_and_repeats(gpu):
    D = 128
    q, k, v, do = inputs(D, seed=6)
    plan = packed_attention_plan(cu_of(LENGTHS, gpu), T, window=300)
    want = run(q, k, v, do, plan, softcap=30.0)
    fused = torch.cat([q.view(T, -1), k.view(T, -1), v.view(T, -1)], 1)
    a, b, c = fused.split([HEADS * D, KV * D, KV * D], 1)
    views = (a.view(T, HEADS, D), b.view(T, KV, D), c.view(T, KV, D))
    first = tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    for other in (views, first, (q, k, v)):
        got = run(*other, do, packed_attention_plan(cu_of(LENGTHS, gpu), T, window=300), softcap=30.0)
        assert all(torch.equal(got[n], want[n]) for n in want)
    with torch.no_grad():
        assert torch.equal(packed_attention(q, k, v, plan, softcap=30.0), want["out"])


def test_captured_and_replayed(gpu):
    q, k, v, do = inputs(64, seed=7)
    cu = cu_of(LENGTHS, gpu)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]

    def step():
        plan = packed_attention_plan(cu, T, validate=False)
        out = packed_attention(*leaves, plan)
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
    for n in range(3):
        new = inputs(64, seed=20 + n)
        bounds = [200 + 150 * n, 60, 300, 8]
        with torch.no_grad():
            for t, x in zip((*leaves, do), new):
                t.copy_(x)
        cu.copy_(cu_of(bounds, gpu))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = run(*new, packed_attention_plan(cu_of(bounds, gpu), T))
        assert all(torch.equal(g, w) for g, w in zip(got, want.values()))


def test_nothing_is_kept_for_no_backward(gpu):
    """Memory at the highest point, beyond what was there: the output and one fp32 number
    for each row and head, without gradients being recorded; more where they are."""
    q, k, v, _ = inputs(128, seed=8)
    plan = packed_attention_plan(cu_of(LENGTHS, gpu), T)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    packed_attention(*leaves, plan)
    least = 2 * q.numel() + 4 * HEADS * T

    def highest():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        at = torch.cuda.memory_allocated()
        out = packed_attention(*leaves, plan)
        return torch.cuda.max_memory_allocated() - at, out

    with torch.no_grad():
        quiet, out = highest()
    recorded, other = highest()
    assert torch.equal(out, other)
    assert least <= quiet <= least + 4096  # (blocks of 512 bytes)
    assert recorded >= least + q.numel() + 4 * HEADS * T

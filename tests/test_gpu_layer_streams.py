"""Calls of the embedding, the layer norms and the updates at once: from several streams and
host threads, and graphs of theirs replayed beside each other."""
from __future__ import annotations

import threading

import pytest
import torch

from mini_trainer_amd import layer_norm, orthogonalize, residual_layer_norm, token_embedding

pytestmark = pytest.mark.gpu


def inputs(seed):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()  # noqa: E731
    t = {"ids": torch.randint(0, 900, (3000,), generator=g).cuda(), "w": rand(900, 520), "d": rand(3000, 520),
         "r": rand(3000, 520), "nw": rand(520), "nb": rand(520), "square": rand(3, 300, 410), "small": rand(70, 16, 90)}
    for name in ("w", "r", "nw", "nb"):
        t[name].requires_grad_(True)
    return t


def everything(t):
    x = token_embedding(t["ids"], t["w"], scale=3.0, validate=False)
    y, h = residual_layer_norm(x, t["r"], t["nw"], t["nb"])
    z = layer_norm(h, t["nw"])
    grads = torch.autograd.grad([y, z], [t["w"], t["r"], t["nw"], t["nb"]], [t["d"], t["d"]])
    return [y, z, *grads, orthogonalize(t["square"]), orthogonalize(t["small"]),
            orthogonalize(t["square"].float())]


def test_streams(gpu):
    sets = [inputs(seed) for seed in range(3)]
    want = [[o.detach().clone() for o in everything(t)] for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [None] * 3
    for _ in range(4):
        for i, (t, s) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(s):
                got[i] = everything(t)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_host_threads(gpu):
    sets = [inputs(seed) for seed in range(4)]
    want = [everything(t) for t in sets]
    torch.cuda.synchronize()
    got, failed = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = everything(sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # (shown by the assertion below)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not failed, failed
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_graphs_beside_each_other(gpu):
    """Each graph holds its own workspaces.  (What keeps no eager graph of the leaves: detached.)"""
    sets = [inputs(seed) for seed in range(2)]
    want = [[o.detach().clone() for o in everything(t)] for t in sets]
    graphs, outs = [], []
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(everything(t))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for out in outs:
            for o in out:
                o.detach().zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))

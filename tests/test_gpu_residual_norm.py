"""Residual and RMS norms in one pass on the GPU against their definition in 64
bits (step_reference.py, which also derives the tolerances)."""
from __future__ import annotations

import math

import pytest
import torch

from mini_trainer_amd import residual_rms_norm

import step_reference as ref

pytestmark = pytest.mark.gpu


def make(T, H, dtype, post, gate, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(T, H, generator=g) * 1.5, "residual": torch.randn(T, H, generator=g) * 3,
         "weight": torch.randn(H, generator=g) * 0.2 + 1.0}
    if post:
        t["post_weight"] = torch.randn(H, generator=g) * 0.2 + 1.0
    shape = {"none": None, "channel": (H,), "token": (T, 1), "element": (T, H)}[gate]
    if shape:
        t["gate"] = torch.randn(shape, generator=g) * 0.5 + 1.0
    ups = [torch.randn(T, H, generator=g) for _ in range(2)]
    return {n: v.to(dtype).cuda() for n, v in t.items()}, [u.to(dtype).cuda() for u in ups]


def run(t, ups, **kw):
    leaf = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    normed, residual = residual_rms_norm(**leaf, **kw)
    grads = torch.autograd.grad([normed, residual], list(leaf.values()), ups)
    return {"normed": normed, "residual": residual, **{"d" + n: g for n, g in zip(leaf, grads)}}


def check(got, t, ups, eps=1e-6, **kw):
    kw = {"offset" if n == "weight_offset" else n: v for n, v in kw.items()}
    want = ref.residual_norm(t["x"], t["residual"], t["weight"], *ups, eps, t.get("post_weight"),
                             t.get("gate"), **kw)
    assert set(got) == set(want)
    for name in want:
        assert got[name].dtype == t["x"].dtype
        ref.assert_within(got[name], want[name], name)


SCALES = dict(block_scale=0.22, residual_scale=0.9, weight_offset=0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("post,gate", [(False, "none"), (True, "none"), (False, "channel"),
                                       (True, "channel"), (True, "token"), (False, "element"),
                                       (True, "element")])
@pytest.mark.parametrize("T,H", [(1, 64), (70, 128), (5, 1001)])
def test_matches_the_definition(gpu, T, H, post, gate, dtype):
    t, ups = make(T, H, dtype, post, gate)
    check(run(t, ups, **SCALES), t, ups, **SCALES)
    check(run(t, ups), t, ups)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [1, 8, 1000, 1024, 1032, 2048, 2056, 2049, 4096, 5000, 8192, 8200,
                               8191, 16384, 32768, 32767])
def test_widths(gpu, H, dtype):
    """Every width class of the kernels, its edges, and rows that are not whole vectors."""
    t, ups = make(7, H, dtype, True, "channel", seed=H)
    check(run(t, ups, **SCALES), t, ups, **SCALES)


def test_more_rows_than_workgroups(gpu):
    for T, H, post in ((5000, 64, False), (3000, 520, True), (1100, 2056, False)):
        t, ups = make(T, H, torch.bfloat16, post, "none", seed=T)
        check(run(t, ups), t, ups)


def test_strides_and_shapes(gpu):
    t, ups = make(24, 72, torch.bfloat16, True, "element", seed=1)
    want = run(t, ups, **SCALES)
    wide = torch.zeros(24, 4, 80, dtype=torch.bfloat16, device=gpu)
    odd = torch.zeros(24, 3, 73, dtype=torch.bfloat16, device=gpu)
    views = dict(t)
    views["x"] = wide[:, 1, :72].copy_(t["x"])
    views["residual"] = odd[:, 1, 1:].copy_(t["residual"])
    views["gate"] = t["gate"].T.contiguous().T
    got = run(views, [ups[0].T.contiguous().T, wide[:, 2, 8:].copy_(ups[1])], **SCALES)
    for n in want:  # (another access width may add a row's squares in another order)
        tol = 2 * 2.0 ** -8 * want[n].double().abs() + 1e-3 * want[n].double().abs().mean()
        assert ((got[n].double() - want[n].double()).abs() <= tol).all(), n
    three = {n: (v.view(2, 12, -1) if v.dim() == 2 else v) for n, v in t.items()}
    got = run(three, [u.view(2, 12, 72) for u in ups], **SCALES)
    for n in want:
        assert torch.equal(got[n].reshape(want[n].shape), want[n]), n
    # one row of x for all rows: its gradient is the sum of theirs
    row = t["x"][:1].detach().requires_grad_(True)
    y, h = residual_rms_norm(row.expand(24, 72), t["residual"], t["weight"])
    g, = torch.autograd.grad([y, h], [row], ups)
    full = ref.residual_norm(t["x"][:1].expand(24, 72), t["residual"], t["weight"], *ups, 1e-6)["dx"]
    err = full[1].sum(0, keepdim=True) + 24 * 2.0 ** -8 * full[0].abs().sum(0, keepdim=True)
    ref.assert_within(g, (full[0].sum(0, keepdim=True), err), "dx")


def test_one_output_used(gpu):
    t, ups = make(40, 256, torch.bfloat16, True, "channel", seed=2)
    zero = torch.zeros_like(ups[0])
    for n in range(2):
        leaf = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        outs = residual_rms_norm(**leaf)
        grads = torch.autograd.grad(outs[n], list(leaf.values()), ups[n], allow_unused=True)
        want = run(t, [ups[0], zero] if n == 0 else [zero, ups[1]])
        for name, g in zip(leaf, grads):
            assert torch.equal(g, want["d" + name]), name


def test_shared_gradient_and_leaves(gpu):
    """x and residual get equal gradients where their scales are equal; writing
    into one leaf's .grad leaves the other's."""
    t, ups = make(33, 128, torch.bfloat16, False, "none", seed=3)
    x, r = (t[n].detach().requires_grad_(True) for n in ("x", "residual"))
    y, h = residual_rms_norm(x, r, t["weight"])
    torch.autograd.backward([y, h], ups)
    assert torch.equal(x.grad, r.grad)
    kept = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, kept)
    same = t["x"].detach().requires_grad_(True)  # the same tensor twice
    y, h = residual_rms_norm(same, same, t["weight"])
    g, = torch.autograd.grad([y, h], [same], ups)
    w = ref.residual_norm(t["x"], t["x"], t["weight"], *ups, 1e-6)["dx"]
    ref.assert_within(g, (2 * w[0], 2 * w[1] + 2 * 2.0 ** -8 * w[0].abs()), "dx")


def test_zero_and_extreme_rows(gpu):
    t, ups = make(6, 64, torch.float32, True, "none", seed=4)
    for n in ("x", "residual"):
        t[n][1] = 0.0     # rms = sqrt(eps)
        t[n][2] *= 1e-12
        t[n][3] *= 1e12
    check(run(t, ups, eps=1e-5), t, ups, eps=1e-5)
    for n in ("x", "residual"):
        t[n][4] = math.nan
    got = run(t, ups, eps=1e-5)
    assert got["normed"][4].isnan().all()
    ok = torch.tensor([0, 1, 2, 3, 5])
    for n in ("normed", "residual", "dx", "dresidual"):  # a row's values stay in its row
        assert torch.isfinite(got[n][ok.to(gpu)]).all()


def test_gradient_is_the_difference_quotient(gpu):
    """In 64 bits, L = <normed, a> + <residual, b>: (L(x + e d) - L(x - e d)) / 2e
    against the kernel's gradient, whose tolerance is summed over |d|."""
    t, ups = make(9, 48, torch.float32, True, "token", seed=5)
    got = run(t, ups, **SCALES)
    want = ref.residual_norm(t["x"], t["residual"], t["weight"], *ups, 1e-6, t["post_weight"],
                             t["gate"], block_scale=0.22, residual_scale=0.9, offset=0.5)
    base = {n: v.double().cpu() for n, v in t.items()}
    a, b = (u.double().cpu() for u in ups)
    rms = torch.nn.functional.rms_norm

    def loss(v):
        u = rms(v["x"], (48,), v["post_weight"] + 0.5, 1e-6)
        h = 0.9 * v["residual"] + 0.22 * v["gate"] * u
        return (rms(h, (48,), v["weight"] + 0.5, 1e-6) * a).sum() + (h * b).sum()

    g = torch.Generator().manual_seed(7)
    for n in base:
        d = torch.randn(base[n].shape, generator=g, dtype=torch.float64)
        q = (loss({**base, n: base[n] + 1e-5 * d}) - loss({**base, n: base[n] - 1e-5 * d})) / 2e-5
        tol = (want["d" + n][1].reshape(d.shape) * d.abs()).sum() + 1e-7 * q.abs() + 1e-7
        assert abs(q - (got["d" + n].double().cpu() * d).sum()) <= tol, n


def test_repeats_streams_and_empty(gpu):
    t, ups = make(3000, 512, torch.bfloat16, True, "channel", seed=6)
    want = run(t, ups)
    torch.cuda.synchronize()
    for stream in (None, torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            got = run(t, ups)
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], want[n]) for n in want)
    e, eu = make(0, 64, torch.bfloat16, True, "channel")
    got = run(e, eu)
    assert got["normed"].shape == (0, 64)
    assert all(not got[n].any() and got[n].shape == (64,) for n in ("dweight", "dpost_weight", "dgate"))


def test_captured_and_replayed(gpu):
    t, ups = make(600, 264, torch.bfloat16, True, "channel", seed=8)
    leaf = {n: v.detach().requires_grad_(True) for n, v in t.items()}

    def step():
        outs = residual_rms_norm(**leaf, **SCALES)
        return outs + torch.autograd.grad(list(outs), list(leaf.values()), ups)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for n in range(4):
        new, new_ups = make(600, 264, torch.bfloat16, True, "channel", seed=30 + n)
        with torch.no_grad():
            for name in leaf:
                leaf[name].copy_(new[name])
            for a, b in zip(ups, new_ups):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        want = run(new, new_ups, **SCALES)
        assert all(torch.equal(g, w) for g, w in zip(got, want.values()))


def test_refusals(gpu):
    t, _ = make(8, 64, torch.bfloat16, False, "none")
    x, r, w = t["x"], t["residual"], t["weight"]
    big = torch.zeros(1, 32776, dtype=torch.bfloat16, device=gpu)
    for args, kw, err in (
            ((x.half(), r.half(), w.half()), {}, TypeError),
            ((x, r.float(), w), {}, TypeError),
            ((x, r, w.float()), {}, TypeError),
            ((x, r[:4], w), {}, ValueError),
            ((x, r, w[:32]), {}, ValueError),
            ((x, r, w), dict(post_weight=w[:1]), ValueError),
            ((x, r, w), dict(gate=w[:5]), ValueError),
            ((x, r, w), dict(gate=x[:4, :1]), ValueError),
            ((x, r, w), dict(eps=-1e-6), ValueError),
            ((x, r, w), dict(eps=math.nan), ValueError),
            ((x, r, w), dict(block_scale=math.inf), ValueError),
            ((x, r, w.cpu()), {}, RuntimeError),
            ((big, big, big[0]), {}, ValueError)):
        with pytest.raises(err):
            residual_rms_norm(*args, **kw)

"""Layer norm on the GPU, with a residual and without, against its definition in 64 bits
(layer_reference.py, which also derives the tolerances)."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import layer_norm, residual_layer_norm

import layer_reference as ref
from step_reference import assert_within

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
SCALES = dict(block_scale=0.22, residual_scale=0.9)


def make(T, H, dtype, residual=True, weight=True, bias=True, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(T, H, generator=g) * 1.5}
    if residual:
        t["residual"] = torch.randn(T, H, generator=g) * 2 + mean
    else:
        t["x"] += mean
    if weight:
        t["weight"] = torch.randn(H, generator=g) * 0.2 + 1.0
    if bias:
        t["bias"] = torch.randn(H, generator=g) * 0.3
    ups = [torch.randn(T, H, generator=g) for _ in range(1 + residual)]
    return {n: v.to(dtype).cuda() for n, v in t.items()}, [u.to(dtype).cuda() for u in ups]


def run(t, ups, **kw):
    leaf = {n: v.detach().requires_grad_(True) for n, v in t.items()}
    if "residual" in t:
        outs = residual_layer_norm(**leaf, **kw)
    else:
        outs = (layer_norm(**leaf, **kw),)
    grads = torch.autograd.grad(outs, list(leaf.values()), ups)
    return {**dict(zip(("normed", "residual"), outs)), **{"d" + n: g for n, g in zip(leaf, grads)}}


def check(t, ups, eps=1e-5, **kw):
    got = run(t, ups, eps=eps, **kw)
    want = ref.layer_norm(t["x"], t.get("residual"), t.get("weight"), t.get("bias"),
                          ups[0], ups[1] if len(ups) > 1 else None, eps, **kw)
    assert set(got) == set(want)
    for name in want:
        assert got[name].dtype == t["x"].dtype
        assert_within(got[name], want[name], name)


@BOTH
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T,H", [(1, 64), (70, 128), (5, 1001)])
def test_matches_the_definition(gpu, T, H, weight, bias, dtype):
    t, ups = make(T, H, dtype, True, weight, bias)
    check(t, ups, **SCALES)
    check(t, ups)
    check(*make(T, H, dtype, False, weight, bias))


@BOTH
@pytest.mark.parametrize("H", [1, 2, 8, 1000, 1024, 1032, 2048, 2056, 2049, 4096, 5000, 8192, 8200,
                               8191, 16384, 32768, 32767])
def test_widths(gpu, H, dtype):
    """Every width class of the kernels, its edges, and rows that are not whole vectors."""
    t, ups = make(7, H, dtype, seed=H)
    check(t, ups, **SCALES)
    check(*make(6, H, dtype, False, seed=H))


@BOTH
@pytest.mark.parametrize("T,H", [(2100, 3), (2100, 5), (9, 7), (2100, 9), (9, 15), (2100, 17), (9, 511), (2100, 513),
                                 (600, 1025), (9, 2047), (600, 2051), (9, 4095), (9, 4097), (520, 8193),
                                 (9, 12289), (9, 16385), (9, 20001), (9, 24577)])
def test_the_last_vector_begins_within_the_one_before(gpu, T, H, dtype):
    t, ups = make(T, H, dtype, seed=H)
    check(t, ups, **SCALES)
    check(*make(T, H, dtype, False, seed=H))


def test_more_rows_than_workgroups(gpu):
    for T, H, residual in ((5000, 64, False), (3000, 520, True), (1100, 2056, True), (1100, 2056, False)):
        check(*make(T, H, torch.bfloat16, residual, seed=T))


def test_offsets_beyond_32_bits(gpu):
    """The last rows of tensors of more than 2^31 elements as those rows alone."""
    T, H = 270000, 8193
    x = torch.empty(T, H, dtype=torch.bfloat16, device=gpu).normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = torch.linspace(-2, 2, H, device=gpu).bfloat16()
    x.requires_grad_(True)
    normed, h = residual_layer_norm(x, x.detach(), w, w)
    (dx,) = torch.autograd.grad([normed, h], x, [x.detach(), x.detach()])
    last = x.detach()[-5:].clone().requires_grad_(True)
    n5, h5 = residual_layer_norm(last, last.detach(), w, w)
    (d5,) = torch.autograd.grad([n5, h5], last, [last.detach(), last.detach()])
    for got, want in ((normed, n5), (h, h5), (dx, d5)):
        assert torch.equal(got[-5:], want)


@BOTH
def test_large_means(gpu, dtype):
    """Rows whose mean is 50 times their deviation."""
    check(*make(40, 256, dtype, mean=100.0))
    check(*make(40, 256, dtype, False, mean=75.0))


def test_constant_rows(gpu):
    """No deviation: the normed row is the bias, the gradient finite with eps."""
    x = torch.full((3, 128), 2.0, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    b = torch.randn(128, device=gpu, dtype=torch.bfloat16)
    y = layer_norm(x, None, b)
    assert torch.equal(y, b.expand(3, 128))
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert not g.any()  # (d - mean(d) is 0)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_row_that_is_not_finite_stays_alone(gpu, bad):
    t, ups = make(9, 136, torch.bfloat16)
    want = run(t, ups)
    t["x"][4, 7] = bad
    got = run(t, ups)
    rows = [i for i in range(9) if i != 4]
    for n in ("normed", "residual", "dx", "dresidual"):
        assert torch.equal(got[n][rows], want[n][rows]), n
    assert got["normed"][4].isnan().all()


def test_strides_and_shapes(gpu):
    t, ups = make(24, 72, torch.bfloat16, seed=1)
    want = run(t, ups, **SCALES)
    wide = torch.zeros(24, 4, 80, dtype=torch.bfloat16, device=gpu)
    odd = torch.zeros(24, 3, 73, dtype=torch.bfloat16, device=gpu)
    views = dict(t)
    views["x"] = wide[:, 1, :72].copy_(t["x"])
    got = run(views, [ups[0].T.contiguous().T, wide[:, 2, 8:].copy_(ups[1])], **SCALES)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    views["residual"] = odd[:, 1, 1:].copy_(t["residual"])  # (single elements)
    check(views, ups, **SCALES)
    three = {n: (v.view(2, 12, -1) if v.dim() == 2 else v) for n, v in t.items()}
    got = run(three, [u.view(2, 12, 72) for u in ups], **SCALES)
    for n in want:
        assert torch.equal(got[n].reshape(want[n].shape), want[n]), n
    # one row of x for all rows: its gradient is the sum of theirs
    row = t["x"][:1].detach().requires_grad_(True)
    y, h = residual_layer_norm(row.expand(24, 72), t["residual"], t["weight"])
    g, = torch.autograd.grad([y, h], [row], ups)
    full = ref.layer_norm(t["x"][:1].expand(24, 72), t["residual"], t["weight"], None, *ups, 1e-5)["dx"]
    err = full[1].sum(0, keepdim=True) + 24 * 2.0 ** -8 * full[0].abs().sum(0, keepdim=True)
    assert_within(g, (full[0].sum(0, keepdim=True), err), "dx")


def test_one_output_used(gpu):
    t, ups = make(40, 256, torch.bfloat16, seed=2)
    zero = torch.zeros_like(ups[0])
    for n in range(2):
        leaf = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        outs = residual_layer_norm(**leaf)
        grads = torch.autograd.grad(outs[n], list(leaf.values()), ups[n], allow_unused=True)
        want = run(t, [ups[0], zero] if n == 0 else [zero, ups[1]])
        for name, g in zip(leaf, grads):
            assert torch.equal(g, want["d" + name]), name


def test_shared_gradient_and_leaves(gpu):
    """x and residual get equal gradients where their scales are equal; writing into one
    leaf's .grad leaves the other's."""
    t, ups = make(33, 128, torch.bfloat16, seed=3)
    x, r = (t[n].detach().requires_grad_(True) for n in ("x", "residual"))
    y, h = residual_layer_norm(x, r, t["weight"], t["bias"])
    torch.autograd.backward([y, h], ups)
    assert torch.equal(x.grad, r.grad)
    want = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, want)


def test_only_some_gradients_wanted(gpu):
    t, ups = make(50, 264, torch.bfloat16, seed=4)
    want = run(t, ups)
    for name in t:
        leaf = {n: v.detach().requires_grad_(n == name) for n, v in t.items()}
        outs = residual_layer_norm(**leaf)
        kept = [o for o in outs if o.requires_grad]
        g, = torch.autograd.grad(kept, [leaf[name]], ups[:len(kept)], allow_unused=True)
        assert torch.equal(g, want["d" + name]), name


def test_no_rows(gpu):
    t, ups = make(0, 64, torch.bfloat16)
    got = run(t, ups)
    assert got["normed"].shape == (0, 64) and not got["dweight"].any() and not got["dbias"].any()


def test_without_gradients(gpu):
    """The same values where nothing is kept for a backward."""
    t, ups = make(20, 200, torch.bfloat16)
    want = run(t, ups)
    with torch.no_grad():
        y, h = residual_layer_norm(**t)
    assert torch.equal(y, want["normed"]) and torch.equal(h, want["residual"])


def test_captured_and_another_stream(gpu):
    t, ups = make(300, 512, torch.bfloat16, seed=5)
    want = run(t, ups)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(t, ups)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(t, ups)
    for seed in range(3):
        new, _ = make(300, 512, torch.bfloat16, seed=seed)
        t["x"].copy_(new["x"])
        graph.replay()
        torch.cuda.synchronize()
        want = run(t, ups)
        for n in want:
            assert torch.equal(got[n], want[n]), n


def test_gradient_against_differences(gpu):
    t, ups = make(6, 96, torch.float32, seed=6)
    got = run(t, ups)
    g = torch.Generator().manual_seed(7)
    step = {n: (torch.randn(v.shape, generator=g) * 2.0 ** -10).cuda() for n, v in t.items()}

    def value(sign):
        outs = residual_layer_norm(**{n: v + sign * step[n] for n, v in t.items()})
        return sum(float((o.double() * u.double()).sum()) for o, u in zip(outs, ups))

    slope = sum(float((got["d" + n].double() * step[n].double()).sum()) for n in t)
    # third order of the step (2^-30 a term, some ten terms an element, whose derivatives
    # are of the order of 1), and roundings of 2^-23 of each of 2 x 576 outputs of
    # magnitude up to 10
    assert abs((value(1) - value(-1)) / 2 - slope) <= 576 * 10 * 2.0 ** -30 + 1152 * 10 * 2.0 ** -23


def test_captured_beside_an_eager_graph_of_the_leaf(gpu):
    x, w = (torch.randn(*s, device=gpu, requires_grad=True) for s in ((9, 64), (64,)))
    alive = layer_norm(x, w)
    with pytest.raises(RuntimeError, match="another stream"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.autograd.grad(layer_norm(x, w).sum(), w)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dw,) = torch.autograd.grad(layer_norm(x, w), w, x.detach())
    (want,) = torch.autograd.grad(layer_norm(x, w), w, x.detach())
    for _ in range(3):
        dw.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, want)


def test_not_differentiable_twice(gpu):
    x, r = (torch.randn(5, 64, device=gpu, requires_grad=True) for _ in range(2))
    normed, _ = residual_layer_norm(x, r)
    dx, dr = torch.autograd.grad((normed * normed).sum(), (x, r), create_graph=True)
    assert torch.equal(dx, dr)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.sum().backward()

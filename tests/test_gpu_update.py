"""Orthogonalised updates on the GPU against their definition in 64 bits
(update_reference.py, which also derives the tolerances)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from mini_trainer_amd import _lib, orthogonalize

import update_reference as ref

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


def make(*shape, dtype=torch.bfloat16, seed=0, rank=0, scale=1.0):
    """Sums of a few outer products of lognormal strength over noise, as momenta are."""
    g = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    k = rank or max(1, min(m, n) // 8)
    rows = torch.randn(*shape[:-1], k, generator=g) * torch.randn(k, generator=g).exp()
    x = rows @ torch.randn(*shape[:-2], k, n, generator=g) / k ** 0.5
    if not rank:
        x = x + torch.randn(*shape, generator=g)
    return (x * scale).to(dtype).cuda()


@BOTH
@pytest.mark.parametrize("m,n", [(1, 1), (1, 100), (100, 1), (2, 3), (8, 24), (63, 65), (64, 64), (65, 200),
                                 (128, 352), (352, 128), (128, 353), (130, 127), (257, 300), (300, 257),
                                 (96, 1000), (16, 4096), (17, 2048), (2049, 32), (33, 1000), (1000, 64), (64, 460),
                                 (4100, 16), (100, 5000), (3000, 200), (1000, 1030)])
def test_matches_the_definition(gpu, m, n, dtype):
    x = make(m, n, dtype=dtype, seed=m + n)
    out = orthogonalize(x)
    assert out.shape == x.shape and out.dtype == dtype and out.is_contiguous()
    ref.assert_within(out, x)


@BOTH
@pytest.mark.parametrize("shape", [(1, 40, 72), (5, 72, 40), (2, 3, 33, 129), (28, 64, 200), (70, 9, 9), (3, 130, 2500)])
def test_stacks(gpu, shape, dtype):
    x = make(*shape, dtype=dtype, seed=3)
    out = orthogonalize(x)
    assert out.shape == x.shape
    for a, b in zip(out.view(-1, *shape[-2:])[::7], x.view(-1, *shape[-2:])[::7]):
        ref.assert_within(a, b)
        assert torch.equal(a, orthogonalize(b))


@BOTH
@pytest.mark.parametrize("batch,m,n", [(1, 962, 2144), (15, 327, 338), (3, 1106, 1515), (43, 351, 336),
                                       (11, 716, 1483), (7, 849, 721), (53, 197, 459), (40, 814, 515),
                                       (31, 519, 560), (30, 705, 870), (1, 4100, 1990), (2, 2300, 2300)])
def test_every_tile(gpu, batch, m, n, dtype):
    """Sizes that take each tile of the symmetric products and of the last one."""
    x = make(batch, m, n, dtype=dtype, seed=m)
    out = orthogonalize(x)
    y = x[-1].double() if m <= n else x[-1].double().T.contiguous()
    k, norm = ref.triples(ref.COEFFICIENTS, 5), float(y.square().sum().sqrt())
    want = ref.iterate(y, k, torch.float64, norm, 1e-7)[-1]
    got = (out[-1] if m <= n else out[-1].T).double()
    # (ref.orthogonalize's bound, whose first part would take minutes here)
    u, planes = torch.finfo(dtype).eps / 2, 2 if dtype == torch.float32 else 1
    limit = ref.SPREAD * (ref.emulated(y, k, norm, 1e-7, planes) - want).norm() + u * want.norm()
    if dtype == torch.float32:
        single = ref.iterate(y.float(), k, torch.float32, norm, 1e-7)[-1]
        limit += ref.FP32_SUMS * (single.double() - want).norm()
    assert float((got - want).norm()) <= float(limit)


@BOTH
def test_strides(gpu, dtype):
    x = make(3, 40, 72, dtype=dtype)
    want = orthogonalize(x)
    wide = torch.randn(3, 45, 91, device=gpu).to(dtype)
    wide[:, 2:42, 3:75] = x
    for view in (wide[:, 2:42, 3:75], x.transpose(1, 2).contiguous().transpose(1, 2),
                 x.permute(1, 0, 2).contiguous().permute(1, 0, 2)):
        assert torch.equal(orthogonalize(view), want)
    assert torch.equal(orthogonalize(x[:1].expand(3, 40, 72)), want[:1].expand(3, 40, 72))
    assert torch.equal(orthogonalize(x[::2]), want[::2])
    assert torch.equal(orthogonalize(x[:, :1, ::3]),
                       torch.stack([orthogonalize(t[:1, ::3].contiguous()) for t in x]))
    leaf = x.clone().requires_grad_(True)
    assert not orthogonalize(leaf).requires_grad


@BOTH
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e-6, 1e6, 1e30])
def test_scales(gpu, scale, dtype):
    """The norm far from 1, below eps too."""
    x = make(30, 50, dtype=dtype, scale=scale, seed=5)
    ref.assert_within(orthogonalize(x), x)
    ref.assert_within(orthogonalize(x, eps=0.0), x, eps=0.0)


@BOTH
@pytest.mark.parametrize("m,n", [(12, 20), (40, 12), (200, 300), (300, 200)])
def test_scales_at_the_ends_of_the_range(gpu, m, n, dtype):
    """A power of two changes nothing without eps, also where 1 / norm is beyond fp32 or one
    of its subnormal numbers."""
    few = torch.zeros(m, n, dtype=dtype, device=gpu)
    for i in range(8):
        few[i, i + 2] = 1 - 2 * (i % 3 == 0)
    g = torch.Generator().manual_seed(m)
    many = torch.randint(-100, 101, (m, n), generator=g).to(dtype).cuda()
    for x, exponent in ((few, -133), (many, 120)):
        scaled = x * 2.0 ** (exponent / 2 // 1) * 2.0 ** (exponent - exponent / 2 // 1)
        norm = scaled.double().norm()
        assert 0 < norm < 2.0 ** -128 or norm > 2.0 ** 128
        got = orthogonalize(scaled, eps=0.0)
        assert got.isfinite().all() and torch.equal(got, orthogonalize(x, eps=0.0))
    for eps in (1e-300, 1e-45, 1.0):
        assert not orthogonalize(torch.zeros_like(few), eps=eps).any()


@BOTH
def test_special_spectra(gpu, dtype):
    for rank in (1, 4):
        x = make(48, 80, dtype=dtype, rank=rank, seed=rank)
        ref.assert_within(orthogonalize(x), x)
    q = torch.linalg.qr(torch.randn(64, 64, generator=torch.Generator().manual_seed(1)))[0]
    for x in (q, torch.eye(64), torch.ones(40, 56), torch.diag(torch.arange(1.0, 41.0))):
        x = x.to(dtype).cuda()
        ref.assert_within(orthogonalize(x), x)


@BOTH
def test_steps_and_coefficients(gpu, dtype):
    x = make(40, 60, dtype=dtype, seed=9)
    for steps in (1, 2, 6, 10, 16, 17):
        ref.assert_within(orthogonalize(x, steps=steps), x, steps=steps)
    each = [(4.0, -7.0, 3.5), (3.0, -3.5, 1.4), (1.5, -0.5, 0.0)]
    ref.assert_within(orthogonalize(x, steps=3, coefficients=each), x, steps=3, coefficients=each)
    ref.assert_within(orthogonalize(x, steps=2, coefficients=(1.875, -1.25, 0.375)), x, steps=2,
                      coefficients=(1.875, -1.25, 0.375))
    same = orthogonalize(x, steps=1, coefficients=(1.0, 0.0, 0.0)).double()
    want = x.double() / (x.double().norm() + 1e-7)
    assert bool(((same - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -22) * want.abs()).all())


@BOTH
def test_zeros_and_values_that_are_not_finite(gpu, dtype):
    x = make(6, 33, 70, dtype=dtype, seed=11)
    want = orthogonalize(x)
    bad = x.clone()
    bad[1] = 0
    bad[2, 5, 6] = float("nan")
    bad[4, 0, 0] = float("inf")
    got = orthogonalize(bad)
    assert not got[1].any() and got[2].isnan().all() and got[4].isnan().all()
    for i in (0, 3, 5):
        assert torch.equal(got[i], want[i])
    assert orthogonalize(bad[1], eps=0.0).isnan().all()  # (0 / 0)


def test_nothing_to_do(gpu):
    for shape in ((0, 5, 6), (4, 0, 6), (4, 5, 0), (0, 0)):
        assert orthogonalize(torch.empty(shape, device=gpu)).shape == shape


def test_a_workspace_of_one_matrix(gpu):
    """The stack in parts, each through the same memory."""
    x = make(5, 170, 130, seed=13)
    want = orthogonalize(x)
    out = torch.empty_like(x)
    k = (ctypes.c_double * 15)(*ref.COEFFICIENTS * 5)
    a = _lib.OrthogonalizeArgs(input=x.data_ptr(), out=out.data_ptr(), coefficients=ctypes.addressof(k), eps=1e-7,
                               batch=1, m=170, n=130, in_row=130, in_batch=170 * 130, steps=5, dtype=1)
    lib = _lib.load()
    nbytes = lib.mt_orthogonalize_workspace_bytes(ctypes.byref(a))
    a.batch = 5
    assert lib.mt_orthogonalize_workspace_bytes(ctypes.byref(a)) == 5 * nbytes
    for some in (1, 2):
        out.zero_()
        ws = torch.full((some * nbytes,), 255, dtype=torch.uint8, device=gpu)  # (NaN in every type)
        _lib.check(lib.mt_orthogonalize(ctypes.byref(a), ws.data_ptr(), some * nbytes,
                                        torch.cuda.current_stream().cuda_stream), "mt_orthogonalize")
        assert torch.equal(out, want)


def test_results_repeat_and_another_stream(gpu):
    x = make(2, 700, 900, seed=15)
    want = orthogonalize(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want) and torch.equal(orthogonalize(x), want)


def test_captured(gpu):
    x = make(2, 200, 328, seed=17)
    small = make(30, 48, dtype=torch.float32, seed=18)
    orthogonalize(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, little = orthogonalize(x), orthogonalize(small)
    for seed in range(3):
        x.copy_(make(2, 200, 328, seed=seed))
        small.copy_(make(30, 48, dtype=torch.float32, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, orthogonalize(x)) and torch.equal(little, orthogonalize(small))


def test_stacks_of_more_than_32_bits(gpu):
    """The ends of a stack of more than 2^31 elements: small matrices of one launch, and larger
    ones that the workspace takes in groups."""
    for batch, m, n in ((70000, 128, 256), (4300, 500, 1001)):
        x = torch.empty(batch, m, n, dtype=torch.bfloat16, device=gpu)
        for i, part in enumerate(x.split(1 << 12)):
            part.normal_(generator=torch.Generator("cuda").manual_seed(i))
        got = orthogonalize(x)
        for at in (0, batch // 2, batch - 1):
            ref.assert_within(got[at], x[at])

"""Orthogonalised updates of bf16 matrices whose singular values are far apart, on the GPU:
the error before the last rounding stays below that rounding's, so that the whole is less than
1.45 times what the rounded exact value is off by (spectra_reference.py)."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import orthogonalize

import spectra_reference as ref

pytestmark = pytest.mark.gpu


def ratios(r, c, gpu, tall=False, seed=0, **kw):
    found = {}
    for name, x in ref.matrices(r, c, seed).items():
        want = ref.exact(x, **kw)
        got = orthogonalize((x.T.contiguous() if tall else x).to(gpu), **kw).cpu()
        found[name] = ref.ratio(got.T if tall else got, want)
    return found


@pytest.mark.parametrize("r,c", [(1, 7), (2, 2), (2, 6), (3, 9), (4, 4), (4, 16), (5, 900), (8, 8), (8, 32), (16, 16),
                                 (16, 64), (13, 2432), (17, 17), (32, 32), (30, 1152)])
def test_small_matrices_are_as_exact_as_their_rounding(gpu, r, c):
    """Few rows: a single rounding reaches the whole result, so that their products are split."""
    for seed in range(10 if r * c < 4096 else 2):
        for tall in (False, True):
            got = ratios(r, c, gpu, tall, seed)
            assert max(got.values()) < 1.01, got


@pytest.mark.parametrize("r,c", [(16, 2900), (24, 1600), (33, 300), (48, 200), (64, 256), (64, 992), (100, 101), (128, 128),
                                 (128, 352), (128, 353), (256, 1024), (300, 301), (500, 900)])
@pytest.mark.parametrize("tall", [False, True])
def test_five_steps(gpu, r, c, tall):
    got = ratios(r, c, gpu, tall)
    assert max(got.values()) < 1.45, got


@pytest.mark.parametrize("r,c", [(96, 256), (200, 600)])
def test_more_steps_of_coefficients_that_settle(gpu, r, c):
    got = ratios(r, c, gpu, steps=12, coefficients=(1.875, -1.25, 0.375))
    assert max(got.values()) < 1.45, got


def test_stacks_take_each_matrix_spectrum(gpu):
    """What one matrix's eigenvalues say is not another's."""
    for r, c in ((64, 256), (256, 1024)):
        stack = torch.stack(list(ref.matrices(r, c).values())).to(gpu)
        got = orthogonalize(stack)
        for one, x in zip(got, stack):
            assert torch.equal(one, orthogonalize(x))


@pytest.mark.parametrize("r,c", [(4, 20), (16, 300), (32, 64)])
def test_split_small_matrices_that_are_zero_or_not_finite(gpu, r, c):
    x = torch.stack(list(ref.matrices(r, c).values())[:5]).to(gpu)
    want = orthogonalize(x)
    bad = x.clone()
    bad[0] = 0
    bad[2, r - 1, c - 1] = float("nan")
    bad[4, 0, 0] = float("-inf")
    got = orthogonalize(bad)
    assert not got[0].any() and got[2].isnan().all() and got[4].isnan().all()
    assert torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])
    assert torch.equal(orthogonalize(x.transpose(1, 2).contiguous()), want.transpose(1, 2))

"""Orthogonalised updates of bf16 matrices whose singular values are far apart, on the GPU,
against the rounded exact value's error (spectra_reference.py)."""
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


def test_stacks_take_each_matrix_spectrum(gpu):
    """What one matrix's eigenvalues say is not another's."""
    for r, c in ((64, 256), (256, 1024)):
        stack = torch.stack(list(ref.matrices(r, c).values())).to(gpu)
        got = orthogonalize(stack)
        for one, x in zip(got, stack):
            assert torch.equal(one, orthogonalize(x))

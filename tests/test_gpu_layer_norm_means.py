"""Layer norm of rows whose mean is 1000 times their deviation and more, against bounds that
E[h^2] - mean^2 does not meet (test_layer_norm_means_cpu.py shows that it does not)."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import layer_norm, residual_layer_norm

import means_reference as ref
from test_layer_norm_means_cpu import SIZES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("ratio", [1000.0, 4000.0])
def test_rows_are_centred_first(gpu, T, H, ratio):
    x, up = ref.rows(T, H, ratio), ref.rows(T, H, 0.5, 1)
    leaf = x.to(gpu).requires_grad_(True)
    y = layer_norm(leaf)
    assert ref.faults(y.detach().cpu(), x) == (0, 0)
    (got,) = torch.autograd.grad(y, leaf, up.to(gpu))
    dx, err = ref.gradient(x, up)
    assert bool(((got.double().cpu() - dx).abs() <= err).all())
    # the same rows as a sum: half and half, exactly
    half = (x / 2).to(gpu)
    y, h = residual_layer_norm(half, half)
    assert torch.equal(h.cpu(), x) and ref.faults(y.cpu(), x) == (0, 0)


def test_behind_a_residual_in_bf16(gpu):
    """The sum is rounded to 8 bits where it is returned, not where it is normalised."""
    x = ref.rows(40, 256, 0.0).bfloat16()
    y, _ = residual_layer_norm(x.to(gpu), torch.full_like(x, 1024.0, device=gpu))
    assert ref.faults(y.cpu(), x.float() + 1024.0, y_unit=2.0 ** -8) == (0, 0)

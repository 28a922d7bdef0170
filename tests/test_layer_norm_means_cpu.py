"""The bounds of means_reference.py tell a norm that centres its rows first from one that
does not."""
from __future__ import annotations

import pytest
import torch

import means_reference as ref

SIZES = [(40, 256), (9, 1601), (6, 4096), (3, 20001)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("ratio", [1000.0, 4000.0])
def test_one_pass_is_found_out(T, H, ratio):
    x = ref.rows(T, H, ratio)
    assert ref.faults(ref.two_pass(x), x) == (0, 0)
    wrong, _ = ref.faults(ref.one_pass(x), x)
    assert wrong >= T // 2


def test_one_pass_is_found_out_behind_a_residual_in_bf16():
    x = ref.rows(40, 256, 0.0).bfloat16()
    h = x.float() + 1024.0  # (exact)
    u = 2.0 ** -8
    assert ref.faults(ref.two_pass(h).bfloat16(), h, y_unit=u) == (0, 0)
    assert ref.faults(ref.one_pass(h).bfloat16(), h, y_unit=u)[0] >= 20


@pytest.mark.parametrize("T,H", SIZES)
def test_gradient_against_autograd(T, H):
    x, up = ref.rows(T, H, 1000.0).double().requires_grad_(True), ref.rows(T, H, 0.5, 1)
    y = torch.nn.functional.layer_norm(x, (H,), eps=1e-5)
    (want,) = torch.autograd.grad(y, x, up.double())
    dx, err = ref.gradient(x.detach(), up)
    assert torch.allclose(dx, want, rtol=1e-9, atol=1e-12) and float((err / dx.abs().mean()).max()) < 0.05

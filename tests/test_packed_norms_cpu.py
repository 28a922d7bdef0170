"""Which layer norms a patched decoder gives to the package, on the CPU with the operator
replaced by its definition."""
from __future__ import annotations

import types

import pytest
import torch
import torch.nn.functional as F

from mini_trainer_amd import decoder


@pytest.fixture
def run(monkeypatch):
    """Runs a patched norm as within a labelled forward: (its output, the package's calls)."""
    calls = []

    def norm(x, weight=None, bias=None, eps=1e-5):
        if not 1 <= x.shape[-1] <= 32768:  # (layer_norm's refusal)
            raise ValueError(f"hidden size {x.shape[-1]}: 1 to 32768 are supported")
        calls.append(x.shape)
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)

    monkeypatch.setattr(decoder, "layer_norm", norm)

    def patched(module, x):
        module.forward = types.MethodType(decoder._norm_forward, module)
        with decoder._set(decoder._own_ops):
            return module(x), len(calls)

    return patched


@torch.no_grad()
def test_norms_wider_than_the_operator_takes_stay_torchs(run):
    for H, own in ((32768, 1), (32769, 1)):
        x = torch.randn(2, H)
        got, calls = run(torch.nn.LayerNorm(H), x)
        assert torch.equal(got, F.layer_norm(x, (H,))) and calls == own


@torch.no_grad()
@pytest.mark.parametrize("affine", [False, True])
def test_a_wrong_width_is_refused_as_torch_does(run, affine):
    """Without a weight nothing else tells layer_norm the width."""
    with pytest.raises(RuntimeError, match="normalized_shape"):
        run(torch.nn.LayerNorm(8, elementwise_affine=affine), torch.randn(2, 16))

"""The autograd nodes on the GPU: the errors of their backward."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import layer_norm, token_embedding
from mini_trainer_amd._lib import FlceError

pytestmark = pytest.mark.gpu


def test_a_refused_capture_raises_the_packages_error(gpu):
    """From the engine's thread of the device."""
    x, w = (torch.randn(*s, device=gpu, requires_grad=True) for s in ((9, 64), (50, 64)))
    ids = torch.arange(9, device=gpu)
    alive = layer_norm(x), token_embedding(ids, w)
    for run in (lambda: torch.autograd.grad(layer_norm(x).sum(), x),
                lambda: torch.autograd.grad(token_embedding(ids, w, validate=False).sum(), w)):
        with pytest.raises(FlceError, match="another stream"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            run()
    del alive

"""The autograd nodes on the GPU: the errors of their backward, and tensors that hooks keep
for them."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import layer_norm, residual_layer_norm, residual_rms_norm, token_embedding
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


def strided(*shape, dtype, gpu, seed):
    """Rows of a wider tensor."""
    g = torch.Generator().manual_seed(seed)
    wide = torch.randn(*shape[:-1], shape[-1] + 24, generator=g).to(dtype).to(gpu)
    return wide[..., 8:8 + shape[-1]].requires_grad_(True)


def calls(dtype, gpu):
    """{name: (a call, the leaves that it takes)}."""
    t = lambda *s, seed: strided(*s, dtype=dtype, gpu=gpu, seed=seed)  # noqa: E731
    x, r, w, b = t(40, 136, seed=0), t(40, 136, seed=1), t(136, seed=2), t(136, seed=3)
    table, ids = t(50, 64, seed=4), torch.arange(300, device=gpu).view(100, 3)[:, 1] % 50
    gates = t(136, seed=5), t(40, 1, seed=6), t(40, 136, seed=7)
    found = {"layer": (lambda: layer_norm(x, w, b), [x, w, b]),
             "residual": (lambda: residual_layer_norm(x, r, w, b)[0], [x, r, w, b]),
             "embedding": (lambda: token_embedding(ids, table), [table])}
    for i, g in enumerate(gates):
        found[f"rms {i}"] = (lambda g=g: residual_rms_norm(x, r, w, post_weight=b, gate=g)[0], [x, r, w, b, g])
    return found


def turned(t):
    if t.dim() == 2:
        return t.T.contiguous().T
    return torch.stack([t, t], -1)[..., 0] if t.dim() == 1 else t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_with_saved_tensors_kept_elsewhere(gpu, dtype):
    for name, (call, leaves) in calls(dtype, gpu).items():
        out = call()
        up = torch.randn(out.shape, generator=torch.Generator().manual_seed(9)).to(dtype).to(gpu)
        want = torch.autograd.grad(out, leaves, up)
        for hooks in (torch.autograd.graph.save_on_cpu(),
                      torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), turned),
                      torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), torch.Tensor.contiguous)):
            with hooks:
                got = torch.autograd.grad(call(), leaves, up)
            for a, b in zip(got, want):
                assert torch.equal(a, b), name

"""The token embedding of a packed row and the gradient of its weight.

A decoder begins with it (the reference leaves it to the model library); its weight is
often the output head's too, so that its gradient can join the head's in the fp32
accumulator of the fused loss (flce.fused_linear_cross_entropy, dw_accumulator).  There
is no CPU or eager-PyTorch fallback: non-device tensors or a missing library raise.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ._lib import torch_ops
from .flce import _dtype_code, _require_device

__all__ = ["token_embedding"]


def token_embedding(input_ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                    padding_idx: Optional[int] = None,
                    dw_accumulator: Optional[torch.Tensor] = None,
                    validate: bool = True) -> torch.Tensor:
    """scale * weight[input_ids], [..., H] for input_ids [...] (int32 or int64) and weight
    [V, H] (bf16 or fp32), differentiable in weight.

    The product is rounded once.  The weight's gradient sums the tokens of each id in
    fp32, in their order, so that it repeats, and is rounded once; rows of ids that do not
    occur are zero, and so is padding_idx's (negative: from the end), whose output is as
    any other's.  With dw_accumulator (fp32 [V, H], rows of unit stride) these sums are
    added to it in fp32 by the backward instead of being returned to autograd, and only
    the rows of ids that occur are touched; the same tensor can be the fused loss's
    accumulator of a head that shares the weight.

    With validate an id outside [0, V) raises IndexError (one sync).  Without it nothing
    synchronises: such a token's row is NaN and gives no gradient.
    """
    _require_device("weight", weight)
    _require_device("input_ids", input_ids)
    if input_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"input_ids must be int32 or int64, got {input_ids.dtype}")
    _dtype_code(weight.dtype)
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be [V, H], got {tuple(weight.shape)}")
    if input_ids.device != weight.device:
        raise ValueError(f"input_ids lie on {input_ids.device}, weight on {weight.device}")
    V, H = weight.shape
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    padding = -1
    if padding_idx is not None:
        padding = int(padding_idx)
        if not -V <= padding < V:
            raise ValueError(f"padding_idx {padding_idx} lies outside [-{V}, {V})")
        padding %= V
    acc = dw_accumulator
    if acc is not None:
        if acc.dtype != torch.float32 or tuple(acc.shape) != (V, H) or not acc.is_cuda or \
                (H > 1 and acc.stride(1) != 1) or (V > 1 and acc.stride(0) < H):
            raise ValueError("dw_accumulator must be a float32 device tensor of shape [V, H] with rows "
                             "of unit stride")
        if acc.device != weight.device:
            raise ValueError(f"dw_accumulator lies on {acc.device}, weight on {weight.device}")
        if acc.requires_grad:
            raise ValueError("dw_accumulator must not require a gradient")
    status = torch.zeros(1, dtype=torch.int32, device=weight.device) if validate else None
    out = torch_ops().embedding(input_ids, weight, scale, padding, acc, status,
                                torch._C._cuda_getCurrentRawStream(weight.device.index))
    if validate and int(status.item()):
        raise IndexError(f"input_ids must lie in [0, {V})")
    return out

"""The token embedding of a packed row and the gradient of its weight.

A decoder begins with it (the reference leaves it to the model library); its weight is
often the output head's too, so that its gradient can join the head's in the fp32
accumulator of the fused loss (flce.fused_linear_cross_entropy, dw_accumulator).  There
is no CPU or eager-PyTorch fallback: non-device tensors or a missing library raise.
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from ._lib import load, pack_embed_args
from .flce import _backward_once, _dtype_code, _launch, _require_device
from .norms import _pitch, _rows

__all__ = ["token_embedding"]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(T: int, V: int, H: int) -> int:
    return load().mt_embed_backward_workspace_bytes(T, V, H)


class _TokenEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding, accumulator, status):
        w, flat = _rows(weight), ids.reshape(-1).contiguous()
        V, H = w.shape
        T = flat.numel()
        out = weight.new_empty(ids.shape + (H,))
        tail = (T, V, H, padding, scale, _dtype_code(weight.dtype), flat.element_size())
        args = pack_embed_args(flat.data_ptr(), w.data_ptr(), out.data_ptr(), 0, 0,
                               0 if status is None else status.data_ptr(), _pitch(w), 0, 0, *tail, 0)
        _launch(w.device, "mt_embed_forward", load().mt_embed_forward, args)
        ctx.save_for_backward(flat)
        ctx.tail, ctx.accumulator = tail, accumulator
        return out

    @_backward_once
    def backward(ctx, dout):
        if not ctx.needs_input_grad[1]:
            return (None,) * 6
        (ids,) = ctx.saved_tensors
        T, V, H = ctx.tail[:3]
        d, acc = _rows(dout), ctx.accumulator
        dw = dout.new_empty((V, H)) if acc is None else acc
        args = pack_embed_args(ids.data_ptr(), 0, 0, d.data_ptr(), dw.data_ptr(), 0, 0, _pitch(d),
                               _pitch(dw), *ctx.tail, int(acc is not None))
        nbytes = _workspace_bytes(T, V, H)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dout.device) if nbytes else None
        _launch(dout.device, "mt_embed_backward", load().mt_embed_backward, args,
                0 if ws is None else ws.data_ptr(), nbytes)
        if acc is None:
            return None, dw, None, None, None, None
        torch.autograd.graph.increment_version([acc])
        return (None,) * 6


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
    out = _TokenEmbedding.apply(input_ids, weight, scale, padding, acc, status)
    if validate and int(status.item()):
        raise IndexError(f"input_ids must lie in [0, {V})")
    return out

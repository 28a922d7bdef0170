"""The global norm of a step's gradients and their clipping.

The reference clips once per optimizer step (train.py:24).  clip_grad_norm_
keeps that call's signature, so that it can be installed with
utils.patch_target_module("torch.nn.utils.clip_grad_norm_", ...); it and
clip_gradients_ also take the fp32 accumulators the loss adds its weight
gradient into (dw_accumulator).  Nothing here synchronises unless asked to.
"""
from __future__ import annotations

import ctypes
import math
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from ._lib import MT_DTYPE_BF16, MT_DTYPE_F32, load
from .flce import _launch, _require_device

__all__ = ["clip_grad_norm_", "clip_gradients_"]


def _layout(t: torch.Tensor) -> Tuple[int, int]:
    """(columns, pitch) of a gradient: (0, 0) if its elements lie in one run in
    some order, else its rows' length and distance."""
    if t.is_contiguous():
        return 0, 0
    dims = sorted(((st, n) for st, n in zip(t.stride(), t.shape) if n > 1))
    run = 1
    cols = 0
    for st, n in dims:
        if st == run:
            run *= n
            continue
        if cols or st < run:
            raise ValueError(f"a gradient of shape {tuple(t.shape)} and strides {t.stride()} is "
                             "neither dense nor rows of equal distance")
        cols, pitch, run = run, st, st * n  # rows from here on: every outer step goes on from them
    return (cols, pitch) if cols else (0, 0)


def _disjoint(a: tuple, b: tuple) -> bool:
    """Whether two gradients whose address ranges overlap share no element: rows
    of the same distance whose columns lie beside each other."""
    (p, es, cols, pitch, _), (q, es2, cols2, pitch2, _) = a, b
    if not cols or es != es2 or pitch != pitch2 or not cols2 or (q - p) % es:
        return False
    off = (q - p) // es % pitch
    return off >= cols and off + cols2 <= pitch


# type -> (code of the C ABI, bytes)
_TYPES = {torch.bfloat16: (MT_DTYPE_BF16, 2), torch.float32: (MT_DTYPE_F32, 4)}


def _table(gradients: Sequence[torch.Tensor]):
    """(ctypes tables, count, device) of the distinct gradients."""
    rows = []
    first = None
    for g in gradients:
        if type(g) is not torch.Tensor and hasattr(g, "to_local"):
            raise TypeError("gradients that are shards of a distributed tensor are not supported")
        if g.layout is not torch.strided:
            raise TypeError("sparse gradients are not supported")
        where = g.get_device()
        if where != first:
            _require_device("gradient", g)
            if first is not None:
                raise ValueError(f"gradients lie on devices {first} and {where}: one is supported")
            first = where
        n = g.numel()
        try:
            code, es = _TYPES[g.dtype]
        except KeyError:
            raise TypeError(f"bfloat16 and float32 are supported, got {g.dtype}") from None
        if g.is_contiguous():
            if n:
                rows.append((g.data_ptr(), es, 0, 0, n * es, n, code))
        else:
            cols, pitch = _layout(g)
            span = n if not cols else (n // cols - 1) * pitch + cols
            rows.append((g.data_ptr(), es, cols, pitch, span * es, n, code))
    rows.sort()
    kept: List[tuple] = []
    open_: List[tuple] = []  # gradients whose range may still reach the next one
    end = 0
    for r in rows:
        if kept and r == kept[-1]:
            continue  # the same memory twice: one gradient
        if r[0] < end:
            open_ = [o for o in open_ if o[0] + o[4] > r[0]]
            for o in open_:
                if not _disjoint(o[:5], r[:5]):
                    raise ValueError("two gradients share part of their memory")
        else:
            open_ = []
        open_.append(r)
        kept.append(r)
        end = max(end, r[0] + r[4])
    n = len(kept)
    ptr, _, cols, pitch, _, numel, code = zip(*kept) if n else ((),) * 7
    return ((ctypes.c_void_p * n)(*ptr), (ctypes.c_int64 * n)(*numel), (ctypes.c_int64 * n)(*cols),
            (ctypes.c_int64 * n)(*pitch), (ctypes.c_int32 * n)(*code)), n, gradients[0].device


@torch.no_grad()
def clip_gradients_(gradients: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale gradients (bf16 or fp32 device tensors) in place so that their
    global norm is at most max_norm, and return that norm before the scaling
    (fp32 scalar on the device).

    Every gradient is multiplied by min(1, max_norm / (norm + 1e-6)), and left
    untouched where that is 1; squares are summed in 64 bits in a fixed order.
    norm_type: 2, or math.inf for the largest magnitude.  The same tensor given
    twice counts once; tensors that share part of their memory are refused, as
    are gradients that are neither dense nor rows of equal distance.  With
    error_if_nonfinite a NaN or infinite norm raises RuntimeError before anything
    is scaled (one sync); otherwise it is applied as it is.
    """
    gradients = list(gradients)
    max_norm, norm_type = float(max_norm), float(norm_type)
    if norm_type not in (2.0, math.inf):
        raise ValueError(f"norm_type {norm_type}: 2 and inf are supported")
    if not max_norm >= 0.0:
        raise ValueError("max_norm must be >= 0")
    if not gradients:
        return torch.tensor(0.0)
    tables, n, dev = _table(gradients)
    lib = load()
    out = torch.empty(2, dtype=torch.float32, device=dev)
    ws = torch.empty(lib.mt_grad_norm_workspace_bytes(tables[1], n), dtype=torch.uint8, device=dev)
    _launch(dev, "mt_grad_norm", lib.mt_grad_norm, *tables, n, int(norm_type == math.inf), max_norm,
            ws.data_ptr(), ws.numel(), out.data_ptr())
    if error_if_nonfinite and not bool(torch.isfinite(out[0])):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients is non-finite, so it "
                           "cannot be clipped. To disable this error and scale the gradients by the "
                           "non-finite norm anyway, set `error_if_nonfinite=False`")
    _launch(dev, "mt_grad_scale", lib.mt_grad_scale, *tables, n, out.data_ptr())
    torch.autograd.graph.increment_version(gradients)
    return out[0]


def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach: Optional[bool] = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ over the parameters' gradients, with its
    signature (train.py:24 calls it so); `foreach` is accepted and ignored.  The
    norm comes back in fp32 whatever the gradients' type.  See clip_gradients_.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return clip_gradients_([p.grad for p in parameters if p.grad is not None], max_norm, norm_type,
                           error_if_nonfinite)

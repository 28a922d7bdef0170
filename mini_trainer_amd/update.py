"""The orthogonalised update of weight matrices.

An optimizer that orthogonalises the momentum of a weight matrix before its step takes
it between the clipped gradients (grad_clip) and the weights.  Nothing here
synchronises; there is no CPU or eager-PyTorch fallback: non-device tensors or a missing
library raise.
"""
from __future__ import annotations

import array
import functools
import math
from typing import Sequence, Tuple, Union

import torch

from ._lib import torch_ops
from .flce import _dtype_code, _require_device

__all__ = ["orthogonalize"]

Triple = Tuple[float, float, float]


def _coefficients(given, steps: int) -> array.array:
    """a, b, c of every step in one run."""
    try:
        return _flat_coefficients(tuple(x if isinstance(x, (int, float)) else tuple(x) for x in given), steps)
    except TypeError:
        raise ValueError("coefficients must be numbers") from None


@functools.lru_cache(maxsize=64)  # (an optimizer's are the same at every step)
def _flat_coefficients(given: tuple, steps: int) -> array.array:
    rows = list(given)
    if rows and all(isinstance(x, (int, float)) for x in rows):
        rows = [rows] * steps
    rows = [[float(x) for x in row] for row in rows]
    if len(rows) != steps or any(len(row) != 3 for row in rows):
        raise ValueError(f"coefficients must be (a, b, c), or such a triple for each of {steps} steps")
    flat = array.array("d", [x for row in rows for x in row])
    if not all(math.isfinite(x) for x in flat):
        raise ValueError("coefficients must be finite")
    return flat


def orthogonalize(update: torch.Tensor, steps: int = 5,
                  coefficients: Union[Triple, Sequence[Triple]] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7) -> torch.Tensor:
    """The update [..., m, n] (bf16 or fp32: a momentum, or a stack of them) with its
    singular values brought near 1, by Newton-Schulz steps over each matrix:

        X = update / (norm(update) + eps)
        steps times:  X = a X + (b A + c A^2) X,  A = X X^T

    (over the shorter side: of the transpose where m > n), in the update's dtype and
    contiguous.  coefficients: a, b, c of all steps, or such a triple for each (1 to 64
    steps); those that would carry singular values in [0, 1] beyond 10^6 are refused.

    X is carried in fp32 and rounded once.  bf16 updates go through fp16 matrix products: the
    default five steps are off by about that last rounding, which is 0.0017 of the norm, or
    less, whatever the singular values (bf16 products: 0.02), and so are more steps of
    coefficients that settle; more of the default ones, which do not, carry errors on (12:
    mostly up to 0.003).  fp32 updates, and bf16 ones of up to 32 rows or columns where one workgroup holds
    them, go through products of split values, with the error of fp32 products or less.  A matrix with NaN or infinities gives NaN, a zero
    matrix zeros (with eps > 0).  Matrices of one shape are cheapest as one stack.  Not
    differentiable.

    The workspace of a matrix of sides r <= c (whole 64) is 10 r c + 6 r^2 bytes in bf16
    and 16 r c + 12 r^2 in fp32, with up to 8 MiB more where r is small and c long; of a
    shorter r, 4 (8) of the 10 (16) bytes are as for 64.  A stack's is at most 2 GiB, or one
    matrix's; matrices that one workgroup holds (128 x 352, 16 x 4096 in bf16) need none.
    """
    _require_device("update", update)
    code = _dtype_code(update.dtype)
    if update.dim() < 2:
        raise ValueError(f"update must be [..., m, n], got {tuple(update.shape)}")
    steps = int(steps)
    if not 1 <= steps <= 64:
        raise ValueError(f"steps {steps}: 1 to 64 are supported")
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError("eps must be >= 0 and finite")
    flat = _coefficients(coefficients, steps)
    return torch_ops().orthogonalize(update, flat.buffer_info()[0], steps, eps,
                                     torch._C._cuda_getCurrentRawStream(update.device.index))

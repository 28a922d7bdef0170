"""Residual and RMS norms between two blocks of a decoder, in one pass.

A decoder layer of the models the reference trains adds a block's output to the
residual and normalises the sum for the next block (the norm that
setup_model_for_training.py:98-99 replaces); some normalise the block's output
first, gate it, or scale it or the residual.  There is no CPU or eager-PyTorch
fallback: non-device tensors or a missing library raise.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from ._lib import load, pack_norm_args
from .flce import _backward_once, _dtype_code, _launch, _require_device

__all__ = ["residual_rms_norm"]

GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_ELEMENT = range(4)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[T, H] view with unit stride along H and rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    elif t.is_contiguous():
        return t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


class _ResidualRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, gate, gate_mode, eps, block_scale,
                residual_scale, offset):
        dev, shape = x.device, x.shape
        H = shape[-1]
        ctx.set_materialize_grads(False)
        x2, r2 = _rows(x), _rows(residual)
        w = weight.contiguous()
        pw = None if post_weight is None else post_weight.contiguous()
        g, gate_t = gate, 0
        if gate_mode == GATE_CHANNEL:
            g = gate.contiguous()
        elif gate_mode != GATE_NONE:
            g = _rows(gate)
            gate_t = _pitch(g)
        normed, new_residual = x.new_empty(shape), x.new_empty(shape)
        T = x2.shape[0]
        rstd = torch.empty((2, T), dtype=torch.float32, device=dev)
        x_t = _pitch(x2)
        tail = (eps, block_scale, residual_scale, offset, gate_mode, _dtype_code(x.dtype))
        args = pack_norm_args(x2.data_ptr(), r2.data_ptr(), w.data_ptr(), _at(pw), _at(g),
                              normed.data_ptr(), new_residual.data_ptr(), rstd.data_ptr(),
                              0, 0, 0, 0, 0, 0, 0, x_t, _pitch(r2), gate_t, 0, 0, T, H, *tail)
        _launch(dev, "mt_norm_forward", load().mt_norm_forward, args)
        # x is read again only for the gradients of a gate or of a norm on it
        extra = pw is not None or g is not None
        ctx.save_for_backward(x2 if extra else None, w, pw, g, new_residual, rstd)
        ctx.meta = (T, H, x_t, gate_t, tail, None if gate is None else gate.shape)
        return normed, new_residual

    @_backward_once
    def backward(ctx, dnormed, dnew):
        if dnormed is None and dnew is None:
            return (None,) * 10
        x2, w, pw, g, new_residual, rstd = ctx.saved_tensors
        T, H, x_t, gate_t, tail, gate_shape = ctx.meta
        _, block_scale, residual_scale, _, _, _ = tail
        need_x, need_r, need_w, need_pw, need_g = ctx.needs_input_grad[:5]
        dev = new_residual.device
        dn = _rows(torch.zeros_like(new_residual) if dnormed is None else dnormed)
        dh = None if dnew is None else _rows(dnew)
        # where both are the same number the two inputs share one gradient, as an
        # addition's do
        same = pw is None and g is None and block_scale == residual_scale and need_x and need_r
        new = new_residual.new_empty
        dr = new(new_residual.shape) if need_r else None
        dx = new(new_residual.shape) if need_x and not same else None
        dw = new((H,)) if need_w else None
        dpw = new((H,)) if need_pw else None
        dg = new(gate_shape) if need_g else None
        args = pack_norm_args(_at(x2), 0, w.data_ptr(), _at(pw), _at(g), 0, new_residual.data_ptr(),
                              rstd.data_ptr(), dn.data_ptr(), _at(dh), _at(dx), _at(dr), _at(dw),
                              _at(dpw), _at(dg), x_t, H, gate_t, _pitch(dn),
                              H if dh is None else _pitch(dh), T, H, *tail)
        lib = load()
        nbytes = lib.mt_norm_backward_workspace_bytes(T, H)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _launch(dev, "mt_norm_backward", lib.mt_norm_backward, args, ws.data_ptr(), nbytes)
        if T == 0:
            for t in (dw, dpw, dg):
                if t is not None:
                    t.zero_()
        return (dr if same else dx), dr, dw, dpw, dg, None, None, None, None, None


def residual_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                      eps: float = 1e-6, post_weight: Optional[torch.Tensor] = None,
                      gate: Optional[torch.Tensor] = None, block_scale: float = 1.0,
                      residual_scale: float = 1.0,
                      weight_offset: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(normed, new_residual) of a block's output x [..., H] and the residual
    before it, differentiable in every tensor:

        u            = x, or rms_norm(x) * (weight_offset + post_weight)
        new_residual = residual_scale * residual + block_scale * gate * u
        normed       = rms_norm(new_residual) * (weight_offset + weight)

    rms_norm(t) = t / sqrt(mean(t^2) + eps).  weight and post_weight are [H]
    (weight_offset = 1 for weights stored as differences from 1); gate is [H], or
    x's shape with a last dimension of 1 (one number per token), or x's shape.
    All tensors are bf16, or all fp32; everything is computed in fp32 and rounded
    once (normed comes from the unrounded sum, the gradients from new_residual as
    it was rounded), weight gradients are summed in fp32 in a fixed order.  H is at
    most 32768.
    """
    dtype, dev = x.dtype, x.device
    for name, t in (("x", x), ("residual", residual), ("weight", weight),
                    ("post_weight", post_weight), ("gate", gate)):
        if t is None:
            continue
        _require_device(name, t)
        if t.dtype != dtype:
            raise TypeError(f"{name} ({t.dtype}) and x ({dtype}) must have the same dtype")
        if t.device != dev:
            raise ValueError(f"{name} lies on {t.device}, x on {dev}")
    _dtype_code(x.dtype)
    if x.dim() < 1 or residual.shape != x.shape:
        raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)} must have one shape")
    H = x.shape[-1]
    for name, t in (("weight", weight), ("post_weight", post_weight)):
        if t is not None and t.shape != (H,):
            raise ValueError(f"{name} must be [{H}], got {tuple(t.shape)}")
    if not 1 <= H <= 32768:
        raise ValueError(f"hidden size {H}: 1 to 32768 are supported")
    if not (eps >= 0 and math.isfinite(eps + block_scale + residual_scale + weight_offset)):
        raise ValueError("eps must be >= 0, and it, block_scale, residual_scale and weight_offset "
                         "finite")
    mode = GATE_NONE
    if gate is not None:
        if tuple(gate.shape) == (H,):
            mode = GATE_CHANNEL
        elif gate.shape == x.shape:
            mode = GATE_ELEMENT
        elif gate.shape == x.shape[:-1] + (1,):
            mode = GATE_TOKEN
        else:
            raise ValueError(f"gate must be [{H}], {tuple(x.shape[:-1] + (1,))} or "
                             f"{tuple(x.shape)}, got {tuple(gate.shape)}")
    return _ResidualRmsNorm.apply(x, residual, weight, post_weight, gate, mode, float(eps),
                                  float(block_scale), float(residual_scale), float(weight_offset))

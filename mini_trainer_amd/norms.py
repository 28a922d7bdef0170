"""Residual and RMS norms between two blocks of a decoder, in one pass.

A decoder layer of the models the reference trains adds a block's output to the
residual and normalises the sum for the next block (the norm that
setup_model_for_training.py:98-99 replaces); some normalise the block's output
first, gate it, or scale it or the residual.  There is no CPU or eager-PyTorch
fallback: non-device tensors or a missing library raise.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import NormArgs, check, load
from .flce import _dtype_code, _on_device, _p, _require_device, _stream

__all__ = ["residual_rms_norm"]

GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_ELEMENT = range(4)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[T, H] view with unit stride along H and rows that do not overlap."""
    t = t.reshape(-1, t.shape[-1])
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class _ResidualRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, post_weight, gate, gate_mode, eps, block_scale,
                residual_scale, offset):
        dev, H = x.device, x.shape[-1]
        ctx.set_materialize_grads(False)
        x2, r2 = _rows(x), _rows(residual)
        w = weight.contiguous()
        pw = None if post_weight is None else post_weight.contiguous()
        g = gate
        if gate_mode == GATE_CHANNEL:
            g = gate.contiguous()
        elif gate_mode != GATE_NONE:
            g = _rows(gate)
        normed, new_residual = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
        rstd = torch.empty((2, x2.shape[0]), dtype=torch.float32, device=dev)
        ctx.meta = (gate_mode, eps, block_scale, residual_scale, offset)
        a = _args(ctx.meta, x2, r2, w, pw, g, new_residual, rstd)
        a.normed = _p(normed)
        with _on_device(dev):
            check(load().mt_norm_forward(ctypes.byref(a), _stream(dev)), "mt_norm_forward")
        # x is read again only for the gradients of a gate or of a norm on it
        keep = x2 if (pw is not None or g is not None) else None
        ctx.save_for_backward(keep, w, pw, g, new_residual, rstd)
        ctx.shapes = (x.shape, None if gate is None else gate.shape)
        return normed, new_residual

    @staticmethod
    @once_differentiable
    def backward(ctx, dnormed, dnew):
        x2, w, pw, g, new_residual, rstd = ctx.saved_tensors
        gate_mode, _, block_scale, residual_scale, _ = ctx.meta
        need_x, need_r, need_w, need_pw, need_g = ctx.needs_input_grad[:5]
        if dnormed is None and dnew is None:
            return (None,) * 10
        shape, gate_shape = ctx.shapes
        dev, dt = new_residual.device, new_residual.dtype
        dn = torch.zeros_like(new_residual) if dnormed is None else dnormed
        dn = _rows(dn)
        dh = None if dnew is None else _rows(dnew)
        a = _args(ctx.meta, x2, None, w, pw, g, new_residual, rstd)
        a.dnormed, a.dnormed_t = _p(dn), _pitch(dn)
        a.dresidual_out, a.dresidual_out_t = _p(dh), a.H if dh is None else _pitch(dh)

        def new(needed, like_shape):
            return torch.empty(like_shape, dtype=dt, device=dev) if needed else None

        # where both are the same number the two inputs share one gradient, as an
        # addition's do
        same = pw is None and g is None and block_scale == residual_scale and need_x and need_r
        dr = new(need_r, shape)
        dx = new(need_x and not same, shape)
        dw, dpw, dg = new(need_w, w.shape), new(need_pw, w.shape), new(need_g, gate_shape)
        a.dx, a.dresidual, a.dweight, a.dpost_weight, a.dgate = map(_p, (dx, dr, dw, dpw, dg))
        lib = load()
        ws = torch.empty(lib.mt_norm_backward_workspace_bytes(a.T, a.H), dtype=torch.uint8, device=dev)
        with _on_device(dev):
            check(lib.mt_norm_backward(ctypes.byref(a), _p(ws), ws.numel(), _stream(dev)),
                  "mt_norm_backward")
        if a.T == 0:
            for t in (dw, dpw, dg):
                if t is not None:
                    t.zero_()
        return (dr if same else dx), dr, dw, dpw, dg, None, None, None, None, None


def _args(meta, x2, r2, w, pw, g, new_residual, rstd) -> NormArgs:
    a = NormArgs()
    a.gate_mode, a.eps, a.block_scale, a.residual_scale, a.weight_offset = meta
    a.dtype = _dtype_code(new_residual.dtype)
    a.H = w.shape[0]
    a.T = new_residual.numel() // a.H
    a.x_t = a.H if x2 is None else _pitch(x2)
    a.residual_t = a.H if r2 is None else _pitch(r2)
    if a.gate_mode == GATE_TOKEN:  # [T, 1]: one element per row
        a.gate_t = max(1, g.stride(0)) if g.shape[0] > 1 else 1
    elif a.gate_mode == GATE_ELEMENT:
        a.gate_t = _pitch(g)
    a.x, a.residual, a.weight, a.post_weight, a.gate = map(_p, (x2, r2, w, pw, g))
    a.new_residual, a.rstd = _p(new_residual), _p(rstd)
    return a


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
    once (normed comes from the unrounded sum), weight gradients are summed in
    fp32 in a fixed order.  H is at most 32768.
    """
    tensors = {"x": x, "residual": residual, "weight": weight, "post_weight": post_weight,
               "gate": gate}
    for name, t in tensors.items():
        if t is None:
            continue
        _require_device(name, t)
        if t.dtype != x.dtype:
            raise TypeError(f"{name} ({t.dtype}) and x ({x.dtype}) must have the same dtype")
        if t.device != x.device:
            raise ValueError(f"{name} lies on {t.device}, x on {x.device}")
    _dtype_code(x.dtype)
    if x.dim() < 1 or residual.shape != x.shape:
        raise ValueError(f"x {tuple(x.shape)} and residual {tuple(residual.shape)} must have one shape")
    H = x.shape[-1]
    for name in ("weight", "post_weight"):
        t = tensors[name]
        if t is not None and tuple(t.shape) != (H,):
            raise ValueError(f"{name} must be [{H}], got {tuple(t.shape)}")
    if not 1 <= H <= 32768:
        raise ValueError(f"hidden size {H}: 1 to 32768 are supported")
    for name, s in (("eps", eps), ("block_scale", block_scale), ("residual_scale", residual_scale),
                    ("weight_offset", weight_offset)):
        if not math.isfinite(s) or (name == "eps" and s < 0):
            raise ValueError(f"{name} must be finite" + (" and >= 0" if name == "eps" else ""))
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

"""Token embedding and layer norm in 64 bits on the CPU, from their definitions, and how
far a right kernel may be from them: the sum of the roundings a value goes through, as
step_reference.py counts them (unit, F32, C)."""
from __future__ import annotations

import torch

from step_reference import C, F32, unit


def embedding(ids, weight, dout, scale=1.0, padding=None, accumulator=None):
    """{name: (value, tolerance)} of out and dweight, or of out and accumulator."""
    u = unit(weight.dtype)
    ids = ids.detach().long().cpu().reshape(-1)
    w, d = weight.detach().double().cpu(), dout.detach().double().cpu().reshape(ids.numel(), -1)
    V, H = w.shape
    good = (ids >= 0) & (ids < V)
    out = scale * w[ids.clamp(0, V - 1)]
    out[~good] = float("nan")
    counted = good if padding is None else good & (ids != padding % V)
    at, rows = ids[counted], scale * d[counted]
    total = torch.zeros(V, H, dtype=torch.float64).index_add_(0, at, rows)
    size = torch.zeros(V, H, dtype=torch.float64).index_add_(0, at, rows.abs())
    n = torch.bincount(at, minlength=V).double()[:, None]
    err = (n + C) * F32 * size
    got = {"out": (out, (u + F32) * out.abs())}
    if accumulator is None:
        got["dweight"] = (total, err + u * total.abs())
    else:
        value = accumulator.detach().double().cpu() + total
        got["accumulator"] = (value, err + F32 * value.abs())
    return got


def layer_norm(x, residual, weight, bias, dnormed, dnew, eps, block_scale=1.0, residual_scale=1.0):
    """{name: (value, tolerance)} of every output and gradient; residual, weight, bias and
    dnew may be None."""
    dt = x.dtype
    u = unit(dt)
    H = x.shape[-1]
    f = (H + C) * F32  # relative error of a row's sum and what follows

    def wide(t):
        return None if t is None else t.detach().double().cpu().reshape(-1, t.shape[-1])

    x, r, w, b, dy, dh = (wide(t) for t in (x, residual, weight, bias, dnormed, dnew))
    w = torch.ones(1, H, dtype=torch.float64) if w is None else w
    has_bias, b = b is not None, torch.zeros(1, H, dtype=torch.float64) if b is None else b
    if r is None:
        h, h_err, read_err = x, torch.zeros_like(x), torch.zeros_like(x)
    else:
        h = residual_scale * r + block_scale * x
        h_err = 2 * F32 * ((residual_scale * r).abs() + (block_scale * x).abs())
        # 16 bits of the sum are kept in bf16 (a step of 2^-15 at most), all in fp32
        read_err = (2.0 ** -15 if dt == torch.bfloat16 else 0.0) * h.abs()
    m = h.mean(1, keepdim=True)
    m_err = h_err.mean(1, keepdim=True) + f * h.abs().mean(1, keepdim=True)
    c = h - m
    c_err = h_err + m_err + F32 * (h.abs() + m.abs())
    var = (c * c).mean(1, keepdim=True)
    ir = 1 / torch.sqrt(var + eps)
    rel = ((2 * c.abs() * c_err + c_err * c_err).mean(1, keepdim=True) + f * var) / (2 * (var + eps)) + C * F32
    hn = c * ir
    hn_err = ir * c_err + hn.abs() * rel
    y = hn * w + b
    got = {"normed": (y, u * y.abs() + hn_err * w.abs() + C * F32 * ((hn * w).abs() + b.abs()))}
    if r is not None:
        got["residual"] = (h, u * h.abs() + h_err)
    hn_err = hn_err + ir * read_err
    d = dy * w
    s0, s1 = d.mean(1, keepdim=True), (d * hn).mean(1, keepdim=True)
    s0_err = f * d.abs().mean(1, keepdim=True)
    s1_err = (d.abs() * hn_err).mean(1, keepdim=True) + f * (d * hn).abs().mean(1, keepdim=True)
    inner = d.abs() + s0.abs() + (hn * s1).abs()
    g = ir * (d - s0 - hn * s1)
    # (hn + e)(s1 + f) - hn s1 = hn f + e s1 + e f: the last counts where a row has next to
    # no deviation, e is then 2^-15 |h| / sqrt(eps) against an hn of 0
    g_err = ir * (s0_err + (hn.abs() + hn_err) * s1_err + hn_err * s1.abs() + C * F32 * inner) + rel * ir * inner
    if dh is not None:
        g = g + dh
        g_err = g_err + C * F32 * dh.abs()

    def total(value, err):
        s = value.sum(0)
        return s, err.sum(0) + (value.shape[0] + C) * F32 * value.abs().sum(0) + u * s.abs()

    if weight is not None:
        got["dweight"] = total(dy * hn, dy.abs() * hn_err)
    if has_bias:
        got["dbias"] = total(dy, torch.zeros_like(dy))
    if r is not None:
        got["dresidual"] = (residual_scale * g, abs(residual_scale) * g_err + (u + F32) * (residual_scale * g).abs())
    got["dx"] = (block_scale * g, abs(block_scale) * g_err + (u + F32) * (block_scale * g).abs())
    return got

"""The operators around the loss in 64 bits on the CPU, from their definitions,
and how far a right kernel may be from them.

A tolerance is the sum of the roundings a value goes through: u = eps / 2 of the
inputs' type (2^-8 bf16, 2^-24 fp32) where a result is stored, where the
probabilities and score gradients enter a product in that type (bf16; fp32
keeps them), and where a stored result is read again; plus, for every fp32 sum
of n terms, (n + C) 2^-24 of the sum of their magnitudes; plus FLOOR for every
number below the normal range: exp2 and the matrix instructions take one for
zero, so a probability (or a product with one) may be off by that much outright.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24
FLOOR = 2.0 ** -126
C = 16  # fp32 operations before and after a sum: scaling, exp2, log2, reciprocal


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def seen_mask(lengths, T, window=None, prefix=None):
    """bool [T, T]: key j (column) is seen by query i (row)."""
    mask = torch.zeros(T, T, dtype=torch.bool)
    at = 0
    for s, n in enumerate(lengths):
        i = torch.arange(n)[:, None]
        j = torch.arange(n)[None, :]
        p = 0 if prefix is None else prefix[s]
        m = (j <= i) | (j < p)
        if window is not None:
            m &= i - j < window
        mask[at:at + n, at:at + n] = m
        at += n
    return mask


def attention(q, k, v, dout, mask, scale=None, softcap=None):
    """{name: (value, tolerance)} of out, dq, dk, dv (dout None: out alone) in fp64."""
    dt = q.dtype
    u = unit(dt)
    up = u if dt == torch.bfloat16 else 0.0  # P and dS rounded before their products
    T, Hq, D = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    out, tol_out = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    got = {"out": (out, tol_out)}
    if dout is not None:
        dout = dout.detach().double().cpu()
        for n, t in (("dq", q), ("dk", k), ("dv", v)):
            got[n] = (torch.zeros_like(t), torch.zeros_like(t))
    sees = mask.any(1)
    n = mask.sum(1, keepdim=True).double()  # terms of a row's sums
    m = mask.sum(0).max().double() * G      # of a column's, over the group's heads
    for h in range(Hq):
        c = h // G
        z = scale * (q[:, h] @ k[:, c].T)
        dz = (D + C) * F32 * scale * (q[:, h].abs() @ k[:, c].abs().T)
        cap_grad = torch.ones_like(z)
        if softcap:
            t = torch.tanh(z / softcap)
            z, cap_grad = softcap * t, 1 - t * t
            dz = dz * cap_grad + softcap * 8 * F32
        dz = dz + C * F32 * z.abs()
        z = z.masked_fill(~mask, -math.inf)
        p = torch.where(sees[:, None], torch.softmax(z, -1), torch.zeros(()).double())
        # an error e of every score moves p by at most 2 max(e) relative to itself
        worst = torch.where(mask, dz, torch.zeros(()).double()).amax(1, keepdim=True)
        dp_rel = 2 * worst + (n + C) * F32
        out[:, h] = p @ v[:, c]
        lost = FLOOR * mask.double()  # of each probability
        size = p @ v[:, c].abs()
        tol_out[:, h] = u * out[:, h].abs() + (up + dp_rel + (n + C) * F32) * size \
            + lost @ v[:, c].abs()
        if dout is None:
            continue
        do = dout[:, h]
        d = do @ v[:, c].T
        d_err = (D + C) * F32 * (do.abs() @ v[:, c].abs().T)
        delta = (do * out[:, h]).sum(1, keepdim=True)
        delta_err = (do.abs() * (tol_out[:, h] + (D + C) * F32 * out[:, h].abs())).sum(1, keepdim=True)
        ds = p * (d - delta) * cap_grad
        grad_err = 8 * F32 * (softcap is not None)
        ds_err = p * (cap_grad + grad_err) * (d_err + delta_err) + ds.abs() * (dp_rel + C * F32) \
            + p * (d - delta).abs() * (grad_err + 2 * dz / (softcap or 1.0) * (softcap is not None))
        ds_err = ds_err + up * ds.abs() + lost * ((d - delta).abs() + 1)
        for name, value, err, terms in (
                ("dq", scale * ds @ k[:, c],
                 scale * (ds_err + (n + C) * F32 * ds.abs()) @ k[:, c].abs(), None),
                ("dk", scale * ds.T @ q[:, h],
                 scale * (ds_err + (m + C) * F32 * ds.abs()).T @ q[:, h].abs(), c),
                ("dv", p.T @ do, ((up + dp_rel + (m + C) * F32) * p + lost).T @ do.abs(), c)):
            at = h if terms is None else c
            got[name][0][:, at] += value
            got[name][1][:, at] += err
    for name in got:
        if name != "out":
            got[name] = (got[name][0], got[name][1] + u * got[name][0].abs() + FLOOR)
    return got


def residual_norm(x, residual, weight, dnormed, dnew, eps, post_weight=None, gate=None,
                  block_scale=1.0, residual_scale=1.0, offset=0.0):
    """{name: (value, tolerance)} of every output and gradient in fp64."""
    dt = x.dtype
    u = unit(dt)
    H = x.shape[-1]
    f = (H + C) * F32  # relative error of a row's mean of squares and what follows
    x, r, w, dy, dh = (t.detach().double().cpu().reshape(-1, t.shape[-1])
                       for t in (x, residual, weight, dnormed, dnew))
    w = w.reshape(-1) + offset
    T = x.shape[0]
    g = torch.ones(1, 1, dtype=torch.float64)
    if gate is not None:
        g = gate.detach().double().cpu()
        g = g.reshape(1, H) if tuple(gate.shape) == (H,) else g.reshape(T, -1)
    xn, pw = x, torch.ones(H, dtype=torch.float64)
    ix = torch.ones(T, 1, dtype=torch.float64)
    if post_weight is not None:
        pw = post_weight.detach().double().cpu() + offset
        ix = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
        xn = x * ix
    block = xn * pw
    h = residual_scale * r + block_scale * g * block
    h_err = f * ((residual_scale * r).abs() + (block_scale * g * block).abs())
    ih = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    hn = h * ih
    hn_err = ih * (h_err + hn.abs() * (h_err * hn.abs()).mean(1, keepdim=True)) + f * hn.abs()
    got = {"normed": (hn * w, u * (hn * w).abs() + hn_err * w.abs()), "residual": (h, u * h.abs() + h_err)}
    hn_err = hn_err + u * hn.abs()  # the backward reads the stored sum
    dn = dy * w
    s1 = (dn * hn).mean(1, keepdim=True)
    s1_err = (dn.abs() * hn_err).mean(1, keepdim=True) + f * (dn * hn).abs().mean(1, keepdim=True)
    gh = dh + ih * (dn - hn * s1)
    # ih as the forward formed it from the unrounded sum
    gh_err = ih * (hn.abs() * s1_err + hn_err * s1.abs()) \
        + (f + (h_err * hn.abs()).mean(1, keepdim=True) * ih) * (ih * (dn.abs() + (hn * s1).abs())) \
        + C * F32 * dh.abs()

    def total(value, err, dim):
        n = value.shape[dim]
        s = value.sum(dim)
        return s, err.sum(dim) + (n + C) * F32 * value.abs().sum(dim) + u * s.abs()

    got["dresidual"] = (residual_scale * gh, abs(residual_scale) * gh_err + u * (residual_scale * gh).abs())
    got["dweight"] = total(dy * hn, dy.abs() * hn_err, 0)
    du, du_err = block_scale * g * gh, (block_scale * g).abs() * (gh_err + C * F32 * gh.abs())
    if gate is not None:
        dg, dg_err = block_scale * gh * block, (block_scale * block).abs() * (gh_err + f * gh.abs())
        if tuple(gate.shape) == (H,):
            got["dgate"] = total(dg, dg_err, 0)
        elif gate.shape[-1] == 1 and H > 1:
            got["dgate"] = tuple(t[:, None] for t in total(dg, dg_err, 1))
        else:
            got["dgate"] = (dg, dg_err + u * dg.abs())
    dx, dx_err = du, du_err
    if post_weight is not None:
        xn_err = f * xn.abs()
        got["dpost_weight"] = total(du * xn, du_err * xn.abs() + du.abs() * xn_err, 0)
        a, a_err = du * pw, du_err * pw.abs()
        s2 = (a * xn).mean(1, keepdim=True)
        s2_err = (a_err * xn.abs() + a.abs() * xn_err).mean(1, keepdim=True) \
            + f * (a * xn).abs().mean(1, keepdim=True)
        dx = ix * (a - xn * s2)
        dx_err = ix * (a_err + xn.abs() * s2_err + xn_err * s2.abs() + f * (a.abs() + (xn * s2).abs()))
    got["dx"] = (dx, dx_err + u * dx.abs())
    return got


def assert_within(got, want, name):
    """Every element of a kernel's result within the tolerance of its value."""
    value, tol = want
    x = got.detach().double().cpu().reshape(value.shape)
    assert torch.isfinite(x).all(), f"{name}: not finite"
    off = (x - value).abs()
    at = (off - tol).argmax()
    assert bool((off <= tol).all()), (
        f"{name}: {x.flatten()[at]:.9g} for {value.flatten()[at]:.9g}, off by "
        f"{off.flatten()[at]:.3g} of {tol.flatten()[at]:.3g} allowed")

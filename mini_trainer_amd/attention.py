"""Attention over a packed row: every token sees the tokens of its own document.

The reference packs samples into one row without padding (sampler.py:144-208)
and leaves attention to a library that derives the documents' boundaries from
position_ids (setup_model_for_training.py:91); here the boundaries are the
cu_seqlens the loss's per-sample sums take (causal_lm.cu_seqlens_from_minibatch).
Scores may be capped by a tanh, as the loss caps its logits.  There is no CPU
or eager-PyTorch fallback: non-device tensors or a missing library raise.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ._lib import load, pack_attn_args
from .flce import _backward_once, _dtype_code, _launch, _require_device

__all__ = ["AttentionPlan", "packed_attention", "packed_attention_plan"]

NO_WINDOW = 2 ** 31 - 1


class AttentionPlan:
    """Which rows each workgroup of packed_attention takes; built by
    packed_attention_plan, valid for any number of calls (the layers of a model)
    over the same packed row.  `tokens` rows, `documents` of them bounded by
    cu_seqlens, `window` tokens back at most (None: all)."""

    def __init__(self, tokens: int, documents: int, window: Optional[int], buffer: torch.Tensor,
                 status: torch.Tensor):
        self.tokens, self.documents, self.window = tokens, documents, window
        self.buffer, self.status = buffer, status
        self.device = buffer.device

    def validate(self) -> None:
        """Raise ValueError if cu_seqlens or prefix_lens was malformed (one sync)."""
        st = int(self.status.item())
        if st == 1:
            raise ValueError(f"cu_seqlens must start at 0, be non-decreasing and end at or below "
                             f"{self.tokens}")
        if st == 2:
            raise ValueError("every prefix length must lie within its document")


def packed_attention_plan(cu_seqlens: torch.Tensor, tokens: int, window: Optional[int] = None,
                          prefix_lens: Optional[torch.Tensor] = None, validate: bool = True,
                          device: Optional[torch.device] = None) -> AttentionPlan:
    """The plan of packed_attention over `tokens` rows whose documents are
    bounded by cu_seqlens (int32 [S + 1] from 0 on, non-decreasing, its end at
    most `tokens`: rows behind it belong to no document, give zeros and get zero
    gradients).

    window: a token sees at most that many tokens up to itself (local layers).
    prefix_lens (int32 [S]): the first prefix_lens[s] tokens of document s are
    seen by all of its tokens, within the window (a prompt read as a whole).
    With validate, malformed boundaries raise ValueError (one sync if they lie
    on the device); without it nothing synchronises: all rows of a malformed
    cu_seqlens give zeros and a prefix is clamped to its document.  Boundaries
    on the CPU are copied to `device` (default: the current one).
    """
    lib = load()
    T, S = int(tokens), cu_seqlens.numel() - 1
    if T < 0 or S < 0:
        raise ValueError("tokens must be >= 0 and cu_seqlens needs at least one entry")
    if window is not None and int(window) < 1:
        raise ValueError("window must be at least 1 (or None)")
    if prefix_lens is not None and prefix_lens.numel() != S:
        raise ValueError(f"prefix_lens has {prefix_lens.numel()} elements, expected {S}")
    for name, t in (("cu_seqlens", cu_seqlens), ("prefix_lens", prefix_lens)):
        if t is not None and t.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if cu_seqlens.is_cuda:
        dev = cu_seqlens.device
        if device is not None and torch.device(device) != dev:
            raise ValueError(f"cu_seqlens lies on {dev}, not on {device}")
    else:
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise RuntimeError(f"device must be a ROCm device, got {dev}; packed attention has no "
                               "CPU path")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
    def words(t):  # int64 values that no int32 holds stay malformed
        t = t.reshape(-1)
        if t.dtype == torch.int64:
            t = t.clamp(-2 ** 31, 2 ** 31 - 1)
        return t.to(device=dev, dtype=torch.int32).contiguous()

    cu = cu_seqlens
    if cu.device != dev or cu.dtype != torch.int32 or cu.dim() != 1 or not cu.is_contiguous():
        cu = words(cu)
    pre = None
    if prefix_lens is not None:
        pre = words(prefix_lens)
    nbytes = lib.mt_attn_plan_bytes(T, S)
    buf = cu.new_empty(nbytes // 4)
    status = cu.new_empty(1)
    w = NO_WINDOW if window is None else min(int(window), NO_WINDOW)
    _launch(dev, "mt_attn_plan", lib.mt_attn_plan, cu.data_ptr(), 0 if pre is None else pre.data_ptr(),
            S, T, w, buf.data_ptr(), nbytes, status.data_ptr())
    plan = AttentionPlan(T, S, None if window is None else int(window), buf, status)
    if validate:
        plan.validate()
    return plan


def _heads(t: torch.Tensor):
    """(tensor, address, row stride, head stride) of [T, heads, D] as the kernels
    read it: unit stride along D, whole 16-byte strides and address; a copy
    otherwise."""
    st, sh, sd = t.stride()
    at, es = t.data_ptr(), t.element_size()
    if sd == 1 and (at | st * es | sh * es) & 15 == 0 and st <= 1 << 24:
        return t, at, st, sh
    T, H, D = t.shape
    if T == 1:
        st = H * D
    if H == 1:
        sh = D
    if (sd != 1 and D > 1) or (at | st * es | sh * es) & 15 or st > 1 << 24:
        t = t.clone(memory_format=torch.contiguous_format)
        at, st, sh = t.data_ptr(), H * D, D
    return t, at, st, sh


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, plan, scale, softcap, differentiable):
        dev = query.device
        T, heads, D = query.shape
        q, qp, q_t, q_h = _heads(query)
        k, kp, k_t, k_h = _heads(key)
        v, vp, v_t, v_h = _heads(value)
        out = query.new_empty((T, heads, D))
        # lse [heads, T] and, for a backward, what its rounding took from it and, in bf16,
        # what the rounding of out took from that, a byte for each element (rows of whole
        # 32); `rest` and `low`: the fp32 words that they begin at (16-byte boundaries)
        words, rest, low = heads * T, 0, 0
        if differentiable:  # (needs_input_grad does not say whether gradients are recorded)
            rest = -(-words // 4) * 4
            words += rest
            if out.dtype == torch.bfloat16:
                low = -(-words // 4) * 4
                words = low + T * heads * (-(-D // 32) * 8)
        lse = torch.empty(words, dtype=torch.float32, device=dev)
        lse_at = lse.data_ptr()
        plan_at = plan.buffer.data_ptr()
        w = NO_WINDOW if plan.window is None else min(plan.window, NO_WINDOW)
        tail = (T, plan.documents, heads, key.shape[1], D, w, scale, softcap, _dtype_code(query.dtype))
        args = pack_attn_args(qp, kp, vp, out.data_ptr(), lse_at, 0, 0, 0, 0, plan_at,
                              lse_at + 4 * low if low else 0, lse_at + 4 * rest if rest else 0,
                              q_t, q_h, k_t, k_h, v_t, v_h, 0, 0, *tail)
        _launch(dev, "mt_attn_forward", load().mt_attn_forward, args)
        ctx.save_for_backward(q, k, v, out, lse, plan.buffer)
        ctx.tail, ctx.rest, ctx.low = tail, rest, low
        return out

    @_backward_once
    def backward(ctx, dout):
        query, key, value, out, lse, plan = ctx.saved_tensors
        dev = query.device
        query, qp, q_t, q_h = _heads(query)
        key, kp, k_t, k_h = _heads(key)
        value, vp, v_t, v_h = _heads(value)
        dout, dop, do_t, do_h = _heads(dout)
        dq, dk, dv = (t.new_empty(t.shape) for t in (query, key, value))
        lse_at = lse.data_ptr()
        args = pack_attn_args(qp, kp, vp, out.data_ptr(), lse_at, dop, dq.data_ptr(), dk.data_ptr(),
                              dv.data_ptr(), plan.data_ptr(), lse_at + 4 * ctx.low if ctx.low else 0,
                              lse_at + 4 * ctx.rest if ctx.rest else 0, q_t, q_h, k_t, k_h, v_t, v_h, do_t, do_h, *ctx.tail)
        lib = load()
        nbytes = lib.mt_attn_backward_workspace_bytes(args)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _launch(dev, "mt_attn_backward", lib.mt_attn_backward, args, ws.data_ptr(), nbytes)
        return dq, dk, dv, None, None, None, None


def packed_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                     plan: Union[AttentionPlan, torch.Tensor], scale: Optional[float] = None,
                     softcap: Optional[float] = None) -> torch.Tensor:
    """Attention output [T, heads, D] of query [T, heads, D] over key and value
    [T, kv_heads, D] (heads a multiple of kv_heads: query head h reads key head
    h // (heads / kv_heads)), differentiable in all three.

    plan: from packed_attention_plan, or cu_seqlens (a plan without window or
    prefixes is then built and validated, which synchronises once).  Scores are
    scale * q . k (default 1 / sqrt(D)), and softcap * tanh(score / softcap) with
    a softcap.  bf16 or fp32; scores, softmax and sums are computed in fp32, the
    probabilities, and in the gradients the scores' gradients, rounded to the
    inputs' type for their products.  No
    value of another document, nor of a row behind the last one, enters a
    result; within a document NaN or infinite values reach, as 0 * NaN does, the
    rows whose mask hides them.  D is at most 128; strides are free as long as
    the last is 1 and the others and the address are whole 16-byte steps
    (anything else is copied).  Results do not depend on scheduling.
    """
    for name, t in (("query", query), ("key", key), ("value", value)):
        _require_device(name, t)
        if t.dim() != 3:
            raise ValueError(f"{name} must be [T, heads, D], got {tuple(t.shape)}")
    if not query.dtype == key.dtype == value.dtype:
        raise TypeError(f"query ({query.dtype}), key ({key.dtype}) and value ({value.dtype}) must "
                        "have the same dtype")
    _dtype_code(query.dtype)
    T, heads, D = query.shape
    if key.shape != value.shape or key.shape[0] != T or key.shape[2] != D:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} must be "
                         f"[{T}, kv_heads, {D}] for query {tuple(query.shape)}")
    if key.shape[1] == 0 or heads == 0 or heads % key.shape[1]:
        raise ValueError(f"{heads} query heads are no multiple of {key.shape[1]} key heads")
    if D == 0 or D > 128:
        raise ValueError(f"head dimension {D}: 1 to 128 are supported")
    if not query.device == key.device == value.device:
        raise ValueError("query, key and value must lie on one device")
    cap = 0.0 if softcap is None else float(softcap)
    if not 0.0 <= cap < float("inf"):
        raise ValueError("softcap must be positive and finite (or None)")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite (or None)")
    if isinstance(plan, torch.Tensor):
        plan = packed_attention_plan(plan, T, device=None if plan.is_cuda else query.device)
    if plan.tokens != T:
        raise ValueError(f"the plan is for {plan.tokens} rows, query has {T}")
    if plan.device != query.device:
        raise ValueError(f"the plan lies on {plan.device}, query on {query.device}")
    grad = torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad)
    chunk = 16 // query.element_size()
    if D % chunk:  # whole 16-byte chunks: zero columns add nothing to a product
        pad = (0, -D % chunk)
        query, key, value = (torch.nn.functional.pad(t, pad) for t in (query, key, value))
        return _PackedAttention.apply(query, key, value, plan, scale, cap, grad)[..., :D]
    return _PackedAttention.apply(query, key, value, plan, scale, cap, grad)

"""A transformers decoder's layers on this package's operators: attention over
the packed row, and the residual addition with the norm behind it in one pass.

The reference hands attention to a library (setup_model_for_training.py:91) and
the norms to another (:98-99); patch_causal_lm(packed_layers=True) puts these
here in their place for the labelled forward, which train.py:97 runs.
"""
from __future__ import annotations

import contextlib
import contextvars
import functools
import inspect
import types
from typing import Optional

import torch

from .attention import AttentionPlan, packed_attention, packed_attention_plan
from .norms import residual_rms_norm

__all__ = ["AttentionPlans", "patch_decoder_layers", "unlabelled_forward"]

ATTENTION_NAME = "mt_packed"
PLANS_KWARG = "mt_attention_plans"
# transformers' layers whose forward is norm, attention, addition, norm, MLP, addition,
# and the norms that are rms_norm(x) * weight.
PLAIN_LAYERS = ("LlamaDecoderLayer", "Qwen2DecoderLayer")
PLAIN_NORMS = ("LlamaRMSNorm", "Qwen2RMSNorm")
# Layer types whose mask is packed_attention's, without and with a window.
FULL, SLIDING = "full_attention", "sliding_attention"
# What a layer may hand to its attention beside what _attention reads: none of it
# changes the result (positions are in query and key by then).
HARMLESS = ("position_ids", "cache_position", "use_cache", "position_embeddings", "output_hidden_states",
            "output_router_logits")


# Per thread: whether the modules that run now ask their configuration for packed
# attention, and whether the unlabelled forward of a patched model is running.
_packed = contextvars.ContextVar("mt_packed", default=False)
_unlabelled = contextvars.ContextVar("mt_unlabelled", default=False)


@contextlib.contextmanager
def _set(var, value=True):
    token = var.set(value)
    try:
        yield
    finally:
        var.reset(token)


@contextlib.contextmanager
def unlabelled_forward():
    """A context in which a patched decoder runs as it was, within another's labelled
    forward too."""
    with _set(_packed, False), _set(_unlabelled):
        yield


class AttentionPlans:
    """The plans of one packed minibatch, one for each window its layers use.  With
    `validate`, malformed boundaries raise ValueError: here where they lie on the CPU;
    on the device with the first plan, which then synchronises once.  Without it every
    attention of a minibatch malformed there gives zeros, and status (int32 [1], 0 or
    1) says so."""

    def __init__(self, cu_seqlens: torch.Tensor, tokens: int, device: torch.device,
                 validate: bool = True):
        if not cu_seqlens.is_cuda:
            cu = cu_seqlens.reshape(-1).to(torch.int64)
            if cu.numel() == 0 or cu[0] != 0 or cu[-1] > tokens or bool((cu.diff() < 0).any()):
                raise ValueError("cu_seqlens must start at 0, be non-decreasing and end at or below "
                                 f"{tokens}, the row's tokens")
        self._validate = validate and cu_seqlens.is_cuda
        self.status: Optional[torch.Tensor] = None
        self._args = (cu_seqlens, tokens, device)
        self._plans: dict = {}
        self._attended: set = set()
        self._calls = 0

    def get(self, window: Optional[int]) -> AttentionPlan:
        if window not in self._plans:
            cu, tokens, device = self._args
            plan = self._plans[window] = packed_attention_plan(
                cu, tokens, window=window, validate=False, device=None if cu.is_cuda else device)
            if self.status is None:
                self.status = plan.status
                if self._validate:
                    plan.validate()
        return self._plans[window]

    def attended(self, module: torch.nn.Module) -> None:
        """Note that this attention module has run as packed attention."""
        self._attended.add(id(module))
        self._calls += 1

    def check_layers(self, decoder: torch.nn.Module) -> None:
        """Raise ValueError unless every layer of the decoder went through packed
        attention: one that mixes tokens in another way has mixed the documents."""
        layers, ran = getattr(decoder.config, "num_hidden_layers", None), len(self._attended)
        dropped = decoder.training and getattr(decoder.config, "layerdrop", 0.0)
        # (two calls in a layer count once; a module that several layers share, for each)
        if layers not in (ran, self._calls) and not (dropped and layers and 0 < ran < layers):
            raise ValueError(f"packed layers: {ran} of {type(decoder).__name__}'s {layers} layers run "
                             "their attention as packed attention; the others would mix the documents")


def _has_window(module) -> bool:
    """Whether the model's configuration gives an attention module's layer a window."""
    config = getattr(module, "config", None)
    kinds, layer = getattr(config, "layer_types", None), getattr(module, "layer_idx", None)
    if kinds and layer is not None and layer < len(kinds):
        return kinds[layer] == SLIDING
    return getattr(config, "sliding_window", None) is not None and \
        getattr(config, "use_sliding_window", True)


def _attention(module, query, key, value, attention_mask=None, scaling=None, dropout=0.0,
               softcap=None, sliding_window=None, is_causal=None, **kwargs):
    """The attention function of a layer: query [B, heads, T, D], key and value
    [B, kv_heads, T, D] -> ([B, T, heads, D], None).  What packed_attention does not
    compute (a mask of the layer's own, sinks, attention that is not causal, any
    keyword that is not known to change nothing) is refused."""
    plans = kwargs.pop(PLANS_KWARG, None)
    where = type(module).__name__
    if plans is None:
        raise ValueError(f"packed layers: {where} is not handed the keywords of the decoder's forward")
    if dropout:
        raise ValueError("packed attention has no dropout")
    if attention_mask is not None:
        raise ValueError(f"packed attention takes no attention mask; {where} passes its own")
    if is_causal is False or not getattr(module, "is_causal", True):
        raise ValueError(f"packed attention is causal; {where} is not")
    if kwargs.get("output_attentions") is False:
        del kwargs["output_attentions"]
    unknown = sorted(n for n, x in kwargs.items() if x is not None and n not in HARMLESS)
    if unknown:
        raise ValueError(f"packed attention does not compute {', '.join(unknown)} of {where}")
    if key.shape[2] != query.shape[2]:
        raise ValueError("packed attention takes no cache of earlier keys")
    if sliding_window is None and _has_window(module):
        raise ValueError(f"{where} has a sliding window that it does not pass to its attention")
    plans.attended(module)
    B, heads, T, D = query.shape
    q, k, v = (t.transpose(1, 2).reshape(B * T, t.shape[1], D) for t in (query, key, value))
    out = packed_attention(q, k, v, plans.get(sliding_window), scale=scaling, softcap=softcap)
    return out.view(B, T, heads, D), None


def _is_plain(module: torch.nn.Module, names) -> bool:
    """Whether the module is transformers' own of that name and its forward the class's:
    not another class that is called so, nor one whose forward has been replaced, in
    the class or in this module."""
    cls = type(module)
    forward = inspect.unwrap(cls.forward)
    return (cls.__name__ in names and cls.__module__.startswith("transformers.models.")
            and "forward" not in module.__dict__
            and (forward.__module__, forward.__qualname__) == (cls.__module__, cls.__name__ + ".forward"))


def _has_hooks(module: torch.nn.Module) -> bool:
    """Whether something wants to see the module called."""
    every = torch.nn.modules.module
    return bool(module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                or module._backward_pre_hooks or every._global_forward_hooks
                or every._global_forward_pre_hooks or every._global_backward_hooks
                or every._global_backward_pre_hooks)


def _layer_forward(self, hidden_states, attention_mask=None, position_ids=None,
                   past_key_values=None, use_cache=False, position_embeddings=None, **kwargs):
    """A PLAIN_LAYERS forward with the addition after attention and the norm
    behind it in one pass."""
    residual = hidden_states
    hidden_states, _ = self.self_attn(
        hidden_states=self.input_layernorm(hidden_states), attention_mask=attention_mask,
        position_ids=position_ids, past_key_values=past_key_values, use_cache=use_cache,
        position_embeddings=position_embeddings, **kwargs)
    norm = self.post_attention_layernorm
    if PLANS_KWARG in kwargs and _is_plain(norm, PLAIN_NORMS) and not _has_hooks(norm) and \
            hidden_states.dtype == residual.dtype == norm.weight.dtype:
        hidden_states, residual = residual_rms_norm(hidden_states, residual, norm.weight,
                                                    eps=norm.variance_epsilon)
    else:
        residual = residual + hidden_states
        hidden_states = norm(residual)
    return residual + self.mlp(hidden_states)


def _refuse_other_mixers(decoder: torch.nn.Module) -> None:
    """Raise ValueError for a decoder that mixes tokens, or places them, in a way that
    packed attention does not bound by the documents.  (Attention modules that never
    ask for the configured attention show in AttentionPlans.check_layers.)"""
    name = type(decoder).__name__
    if "position_ids" not in inspect.signature(decoder.forward).parameters:
        raise ValueError(f"packed layers: {name} takes no position_ids, so that no document but the "
                         "first would start at position 0")
    other = set(getattr(decoder.config, "layer_types", None) or ()) - {FULL, SLIDING}
    if other:
        raise ValueError(f"packed layers: {name} has layers of {', '.join(sorted(other))}")
    for path, module in decoder.named_modules():
        conv = isinstance(module, torch.nn.modules.conv._ConvNd) and max(module.kernel_size) > 1
        if conv or isinstance(module, torch.nn.RNNBase):
            raise ValueError(f"packed layers: {name}.{path} ({type(module).__name__}) mixes tokens "
                             "across documents")


@functools.lru_cache(maxsize=None)
def _config_view_cls(cls: type) -> type:
    def get(self):
        return ATTENTION_NAME if _packed.get() else super(view, self)._attn_implementation

    def put(self, value):
        cls._attn_implementation.fset(self, value)

    view = type(cls.__name__, (cls,), {"__module__": cls.__module__, "mt_view": True,
                                       "_attn_implementation": property(get, put)})
    return view


def _config_view(config):
    """The same configuration (one dictionary), which names packed attention to the
    modules of a labelled forward and what it names to all others: nothing that
    another thread, or a checkpoint's recomputation, reads is changed for a call."""
    if getattr(type(config), "mt_view", False):
        return config
    view = object.__new__(_config_view_cls(type(config)))
    object.__setattr__(view, "__dict__", config.__dict__)
    return view


OWN_FORWARD = "_mt_own_forward"  # a module's attribute: the forward it had of its own


@functools.lru_cache(maxsize=None)
def _packed_forward(own, is_decoder: bool):
    @functools.wraps(own)
    def forward(self, *args, **kwargs):
        run = self.__dict__.get(OWN_FORWARD) or functools.partial(own, self)
        if kwargs.get(PLANS_KWARG) is not None:
            with _set(_packed):
                return run(*args, **kwargs)
        if is_decoder and not _unlabelled.get():
            raise RuntimeError("the decoder of a model patched with patch_causal_lm(packed_layers=True) "
                               "runs in the model's own forward only: the labelled forward for packed "
                               "attention")
        return run(*args, **kwargs)

    return forward


def patch_decoder_layers(decoder: torch.nn.Module) -> None:
    """Give the decoder's modules, where they run with plans among their keywords, a
    configuration that names packed attention, and its plain layers the fused
    forward.  Without plans the modules run as before."""
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    _refuse_other_mixers(decoder)
    ALL_ATTENTION_FUNCTIONS.register(ATTENTION_NAME, _attention)
    for module in decoder.modules():
        if _is_plain(module, PLAIN_LAYERS):
            module.forward = types.MethodType(_layer_forward, module)
            continue
        config = module.__dict__.get("config")
        if config is None or getattr(type(config), "mt_view", False) or \
                not hasattr(type(config), "_attn_implementation"):
            continue
        parameters = inspect.signature(module.forward).parameters.values()
        if module is not decoder and all(p.kind is not p.VAR_KEYWORD for p in parameters):
            continue  # (no plans reach it)
        module.config = _config_view(config)
        if "forward" in module.__dict__:
            module.__dict__[OWN_FORWARD] = module.forward
        module.forward = types.MethodType(_packed_forward(type(module).forward, module is decoder), module)


def minibatch_plans(tokens: torch.Tensor, position_ids: Optional[torch.Tensor],
                    cu_seqlens: Optional[torch.Tensor], validate: bool = True) -> AttentionPlans:
    """The plans of a minibatch of `tokens` [B, T, ...]: documents by cu_seqlens, or
    where position_ids restart (one sync) and with each row."""
    from .causal_lm import cu_seqlens_from_lengths, cu_seqlens_from_position_ids

    B, T = tokens.shape[:2]
    if B > 1 and cu_seqlens is not None:
        raise ValueError(f"cu_seqlens bounds the samples of one packed row; got {B} rows")
    if cu_seqlens is None:
        validate = False  # (made here)
        if position_ids is None:
            cu_seqlens = cu_seqlens_from_lengths([T] * B)
        else:
            starts = position_ids.reshape(-1, T).expand(B, T).clone()
            starts[:, :1] = 0  # a row is no continuation of the one before
            cu_seqlens = cu_seqlens_from_position_ids(starts)
    return AttentionPlans(cu_seqlens, B * T, tokens.device, validate)


def positions_within(cu_seqlens: torch.Tensor, tokens: int, device: torch.device) -> torch.Tensor:
    """[1, tokens] int64 on `device`: each token's place in its document, the rows behind
    the last one counted as one.  No sync; within the row for malformed boundaries too,
    so that no embedding is read out of range before they are checked."""
    rows = torch.arange(tokens, device=cu_seqlens.device)
    cu = cu_seqlens.reshape(-1).to(torch.int64)
    document = torch.searchsorted(cu, rows, right=True) - 1
    return (rows - cu[document]).clamp(0, max(tokens - 1, 0)).to(device, non_blocking=True)[None]

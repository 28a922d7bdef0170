"""patch_causal_lm(packed_layers=True, embedding_and_norms=True) on the CPU: the host side
of the patched forward, with the operators replaced by their definitions
(test_packed_layers_cpu.py's, and the embedding's and layer norms')."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from mini_trainer_amd import decoder, patch_causal_lm

tf = pytest.importorskip("transformers")

import test_packed_layers_cpu as base  # noqa: E402
from test_packed_layers_cpu import TOL, alone, batch, build, operators, rel  # noqa: E402,F401

base.MODELS.setdefault("starcoder2", ("Starcoder2ForCausalLM", "Starcoder2Config",
                                      dict(base.BASE, residual_dropout=0.0, embedding_dropout=0.0,
                                           attention_dropout=0.0, bos_token_id=0, eos_token_id=0)))
base.MODELS.setdefault("gemma3", ("Gemma3ForCausalLM", "Gemma3TextConfig",
                                  dict(base.BASE, head_dim=16, sliding_window=8,
                                       layer_types=["sliding_attention", "full_attention"])))


@pytest.fixture
def ends(operators, monkeypatch):  # noqa: F811
    """The calls of each operator by its name."""
    calls = {"embedding": [], "norm": 0, "residual": 0}

    def embedding(ids, weight, scale=1.0, padding_idx=None, dw_accumulator=None, validate=True):
        calls["embedding"].append((scale, padding_idx, dw_accumulator))
        assert not validate
        return weight[ids] * scale

    def norm(x, weight=None, bias=None, eps=1e-5):
        calls["norm"] += 1
        return F.layer_norm(x, x.shape[-1:], weight, bias, eps)

    def residual(x, r, weight=None, bias=None, eps=1e-5):
        calls["residual"] += 1
        return F.layer_norm(x + r, x.shape[-1:], weight, bias, eps), x + r

    monkeypatch.setattr(decoder, "token_embedding", embedding)
    monkeypatch.setattr(decoder, "layer_norm", norm)
    monkeypatch.setattr(decoder, "residual_layer_norm", residual)
    return calls


@torch.no_grad()
@pytest.mark.parametrize("name,norms,fused", [("llama", 0, 0), ("gpt2", 5, 0), ("starcoder2", 3, 2),
                                              ("gemma3", 0, 0)])
def test_documents_are_as_alone(ends, name, norms, fused):
    model, kw = build(name), batch()
    want = alone(model, kw["input_ids"])
    logits = model(input_ids=kw["input_ids"]).logits
    patch_causal_lm(model, packed_layers=True, embedding_and_norms=True)
    assert rel(model(**kw).loss, want) <= TOL
    scale = 8.0 if name == "gemma3" else 1.0
    assert [c[0] for c in ends["embedding"]] == [scale] and ends["norm"] == norms and ends["residual"] == fused
    # unlabelled: as before
    assert torch.equal(model(input_ids=kw["input_ids"]).logits, logits)
    assert len(ends["embedding"]) == 1 and ends["norm"] == norms


@torch.no_grad()
def test_without_the_argument_nothing_changes(ends):
    model, kw = build("gpt2"), batch()
    patch_causal_lm(model, packed_layers=True)(**kw)
    assert not ends["embedding"] and not ends["norm"]


@pytest.mark.parametrize("name", ["gpt2", "starcoder2"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_layers_run_the_same_operators_again(ends, name, reentrant):
    model, kw = build(name), batch()
    patch_causal_lm(model, packed_layers=True, embedding_and_norms=True)
    model.train()
    model(**kw).loss.sum().backward()
    want = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    once = dict(ends)
    model.zero_grad()
    model.gradient_checkpointing_enable({"use_reentrant": reentrant})
    if reentrant:
        model.get_input_embeddings().weight.requires_grad_(True)
        model.enable_input_require_grads()
    model(**kw).loss.sum().backward()
    for n, p in model.named_parameters():
        if n in want:
            assert rel(p.grad, want[n]) <= TOL, n
    # every norm of a layer twice, the decoder's last one once
    assert ends["norm"] - once["norm"] == 2 * (once["norm"] - 1) + 1
    assert ends["residual"] == 3 * once["residual"]


@torch.no_grad()
@pytest.mark.parametrize("what", ["hook", "forward", "max_norm", "sparse", "class"])
def test_other_embeddings_keep_theirs(ends, what):
    model, kw = build("llama"), batch()
    want, emb, seen = alone(model, kw["input_ids"]), model.model.embed_tokens, []
    if what == "forward":
        own = emb.forward
        emb.forward = lambda ids: seen.append(True) or own(ids)
    elif what == "max_norm":
        emb.max_norm = 1e6
    elif what == "sparse":
        emb.sparse = True
    elif what == "class":
        emb.__class__ = type("Embedding", (torch.nn.Embedding,), {})
    patch_causal_lm(model, packed_layers=True, embedding_and_norms=True)
    if what == "hook":
        emb.register_forward_hook(lambda *_: seen.append(True))
    assert rel(model(**kw).loss, want) <= TOL and not ends["embedding"]
    assert bool(seen) == (what in ("hook", "forward"))


@torch.no_grad()
@pytest.mark.parametrize("what", ["hook", "forward", "class"])
def test_other_norms_keep_theirs(ends, what):
    model, kw = build("starcoder2"), batch()
    want, layer, seen = alone(model, kw["input_ids"]), model.model.layers[1], []
    norm = layer.post_attention_layernorm
    if what == "forward":
        own = norm.forward
        norm.forward = lambda x: seen.append(True) or own(x)
    elif what == "class":
        norm.__class__ = type("LayerNorm", (torch.nn.LayerNorm,), {})
    patch_causal_lm(model, packed_layers=True, embedding_and_norms=True)
    if what == "hook":
        norm.register_forward_hook(lambda *_: seen.append(True))
    assert rel(model(**kw).loss, want) <= TOL
    assert ends["residual"] == 1
    assert bool(seen) == (what in ("hook", "forward"))


def test_the_embeddings_gradient_in_the_accumulator(ends):
    acc = torch.zeros(100, 64)
    model = build("llama", tie_word_embeddings=True)
    patch_causal_lm(model, dw_accumulator=acc, packed_layers=True, embedding_and_norms=True,
                    accumulate_embedding=True)
    model(**batch())
    assert ends["embedding"][0][2] is acc
    model.get_input_embeddings().register_forward_hook(lambda *_: None)
    with pytest.raises(RuntimeError, match="dw_accumulator"):
        model(**batch())


def test_refusals():
    acc = torch.zeros(100, 64)
    with pytest.raises(ValueError, match="packed_layers"):
        patch_causal_lm(build("llama"), embedding_and_norms=True)
    for kw in (dict(embedding_and_norms=True), dict(dw_accumulator=acc)):
        with pytest.raises(ValueError, match="accumulate_embedding"):
            patch_causal_lm(build("llama", tie_word_embeddings=True), packed_layers=True,
                            accumulate_embedding=True, **kw)
    with pytest.raises(ValueError, match="shares"):
        patch_causal_lm(build("llama", tie_word_embeddings=False), packed_layers=True, dw_accumulator=acc,
                        embedding_and_norms=True, accumulate_embedding=True)
    model = build("llama", tie_word_embeddings=True)
    model.model.embed_tokens.sparse = True
    with pytest.raises(ValueError, match="dw_accumulator"):
        patch_causal_lm(model, packed_layers=True, dw_accumulator=acc, embedding_and_norms=True,
                        accumulate_embedding=True)

"""The operators of a packed step together, as patch_causal_lm(packed_layers=True)
and a clip run them: a two-layer Llama in fp32 over a packed row on the GPU
against the unpatched model on the CPU in 64 bits, one document at a time."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from mini_trainer_amd import clip_grad_norm_, cu_seqlens_from_lengths, patch_causal_lm

transformers = pytest.importorskip("transformers")

LENGTHS = [37, 150, 5, 64, 1, 90]
VOCAB = 500


def tiny(kind="llama", seed=0, **more):
    torch.manual_seed(seed)
    kw = dict(vocab_size=VOCAB, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
              num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=1024,
              tie_word_embeddings=False, attn_implementation="eager", **more)
    if kind == "llama":
        m = transformers.LlamaForCausalLM(transformers.LlamaConfig(**kw))
    else:
        m = transformers.Qwen2ForCausalLM(transformers.Qwen2Config(**kw))
    return m.float()


def packed(seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (1, sum(LENGTHS)), generator=g)
    labels = ids.clone()
    at = 0
    for n in LENGTHS:
        labels[0, at:at + n // 3] = -100
        at += n
    pos = torch.cat([torch.arange(n) for n in LENGTHS])[None]
    return ids, labels, pos


def reference(model, ids, labels):
    """(per-token loss, gradients by name, their norm) document by document in 64 bits."""
    model = copy.deepcopy(model).double()
    hidden, at = [], 0
    for n in LENGTHS:
        hidden.append(model.model(input_ids=ids[:, at:at + n]).last_hidden_state[0])
        at += n
    logits = F.linear(torch.cat(hidden), model.lm_head.weight)
    shifted = F.pad(labels, (0, 1), value=-100)[0, 1:]
    loss = F.cross_entropy(logits, shifted, ignore_index=-100, reduction="none")
    loss.sum().backward()
    grads = {n: p.grad for n, p in model.named_parameters()}
    return loss.detach(), grads, torch.cat([g.flatten() for g in grads.values()]).norm()


def rel(a, b):
    return float((a.double().cpu() - b).norm() / b.norm())


# fp32 through two layers of some 300-term sums: each product's relative error is
# a few sqrt(300) 2^-24 = 1e-6 and a gradient goes through some ten of them; 1e-4
# leaves room for cancellation in sums over the row, and is a tenth of what a
# wrong mask, scale or missing term of one token in 347 would give
TOL = 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["llama", "qwen2"])
@pytest.mark.parametrize("bounds", ["cu_seqlens", "position_ids"])
def test_packed_step_matches_each_document_alone(gpu, kind, bounds):
    model = tiny(kind)
    ids, labels, pos = packed()
    loss_ref, grads_ref, norm_ref = reference(model, ids, labels)
    model = patch_causal_lm(model.to(gpu), packed_layers=True)
    kw = {"cu_seqlens": cu_seqlens_from_lengths(LENGTHS).to(gpu)} if bounds == "cu_seqlens" else {}
    out = model(input_ids=ids.to(gpu), labels=labels.to(gpu), position_ids=pos.to(gpu), **kw)
    assert rel(out.loss.detach(), loss_ref) <= TOL
    out.loss.sum().backward()
    for name, p in model.named_parameters():
        if grads_ref[name].norm() > 1e-9 * norm_ref:
            assert rel(p.grad, grads_ref[name]) <= TOL, name
    before = {n: p.grad.clone() for n, p in model.named_parameters()}
    norm = clip_grad_norm_(model.parameters(), 0.5 * float(norm_ref))
    assert abs(float(norm) - float(norm_ref)) <= TOL * float(norm_ref)
    c = 0.5 * float(norm_ref) / (float(norm) + 1e-6)
    for name, p in model.named_parameters():
        assert torch.allclose(p.grad, before[name] * c, rtol=1e-6, atol=0), name


@pytest.mark.gpu
def test_bf16_step_runs_with_checkpointing_and_accumulator(gpu):
    """bf16, gradient checkpointing of the layers, the head's gradient in an fp32
    accumulator that the clip takes beside the other gradients."""
    ref_model = tiny()
    ids, labels, pos = packed()
    loss_ref, grads_ref, _ = reference(ref_model, ids, labels)
    model = copy.deepcopy(ref_model).to(gpu, torch.bfloat16)
    acc = torch.zeros(VOCAB, 128, device=gpu)
    patch_causal_lm(model, dw_accumulator=acc, packed_layers=True)
    model.train()
    model.gradient_checkpointing_enable({"use_reentrant": False})
    cu = cu_seqlens_from_lengths(LENGTHS)
    out = model(input_ids=ids.to(gpu), labels=labels.to(gpu), position_ids=pos.to(gpu), cu_seqlens=cu)
    out.loss.float().sum().backward()
    # bf16 weights and activations carry 2^-8 each through two layers
    assert rel(out.loss.detach(), loss_ref) <= 2e-2
    assert rel(acc, grads_ref["lm_head.weight"]) <= 5e-2
    name = "model.layers.0.self_attn.q_proj.weight"
    assert rel(dict(model.named_parameters())[name].grad, grads_ref[name]) <= 0.15
    from mini_trainer_amd import clip_gradients_

    grads = [p.grad for p in model.parameters() if p.grad is not None] + [acc]
    want = torch.cat([g.double().flatten() for g in grads]).norm()
    assert abs(float(clip_gradients_(grads, 1.0)) - float(want)) <= 1e-6 * float(want)
    assert float(torch.cat([g.double().flatten() for g in grads]).norm()) <= 1.0 + 2.0 ** -8


@pytest.mark.gpu
def test_rows_window_and_unlabelled_calls(gpu):
    """Several rows are documents of their own; a sliding window reaches the plan;
    without labels the model's own attention runs."""
    model = tiny("qwen2", seed=3, use_sliding_window=True, sliding_window=16, max_window_layers=0,
                 layer_types=["sliding_attention"] * 2)
    ids = torch.randint(0, VOCAB, (3, 40), generator=torch.Generator().manual_seed(4))
    with torch.no_grad():
        logits = model.double()(input_ids=ids).logits
    want = F.cross_entropy(logits[:, :-1].reshape(-1, VOCAB), ids[:, 1:].reshape(-1), reduction="none")
    model = patch_causal_lm(model.float().to(gpu), packed_layers=True)
    loss = model(input_ids=ids.to(gpu), labels=ids.to(gpu)).loss.detach().view(3, 40)
    assert rel(loss[:, :-1].reshape(-1), want) <= TOL and not loss[:, -1].any()
    with torch.no_grad():
        again = model(input_ids=ids.to(gpu)).logits
    assert rel(again, logits) <= TOL
    with pytest.raises(ValueError, match="no attention_mask"):
        model(input_ids=ids.to(gpu), labels=ids.to(gpu), attention_mask=torch.ones_like(ids).to(gpu))
    with pytest.raises(ValueError, match="one packed row"):
        model(input_ids=ids.to(gpu), labels=ids.to(gpu), cu_seqlens=torch.tensor([0, 120]))


@pytest.mark.gpu
def test_another_norm_keeps_its_own_forward(gpu):
    """A layer whose norm was replaced does not go through residual_rms_norm."""
    model = tiny(seed=7)
    for layer in model.model.layers:
        layer.post_attention_layernorm = torch.nn.LayerNorm(128)
    ids, labels, pos = packed()
    loss_ref, _, _ = reference(model, ids, labels)
    model = patch_causal_lm(model.to(gpu), packed_layers=True)
    out = model(input_ids=ids.to(gpu), labels=labels.to(gpu), position_ids=pos.to(gpu))
    assert rel(out.loss.detach(), loss_ref) <= TOL


def test_patched_layers_without_a_gpu():
    model = tiny(seed=5)
    ids, labels, pos = packed()
    with torch.no_grad():
        logits = model(input_ids=ids).logits
    model = patch_causal_lm(model, packed_layers=True)
    with torch.no_grad():  # unlabelled: as before, the fused layers included
        assert torch.equal(model(input_ids=ids).logits, logits)
    with pytest.raises(RuntimeError, match="ROCm device"):
        model(input_ids=ids, labels=labels, cu_seqlens=cu_seqlens_from_lengths(LENGTHS))
    with pytest.raises(RuntimeError, match="labelled forward"):
        model.model(input_ids=ids)

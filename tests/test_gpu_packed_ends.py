"""A packed step with its embedding, layer norms and an orthogonalised update, as
patch_causal_lm(packed_layers=True, embedding_and_norms=True), a clip and orthogonalize run
them together, on the GPU against the unpatched model on the CPU in 64 bits."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from mini_trainer_amd import (clip_gradients_, cu_seqlens_from_lengths, orthogonalize, patch_causal_lm,
                              token_embedding)

import test_gpu_packed_step as step
import update_reference
from test_gpu_packed_step import LENGTHS, TOL, VOCAB, packed, rel

transformers = pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu


def tiny(kind, seed=0, **more):
    if kind == "llama":
        return step.tiny(seed=seed, **more)
    torch.manual_seed(seed)
    kw = dict(vocab_size=VOCAB, attn_implementation="eager", bos_token_id=0, eos_token_id=0,
              tie_word_embeddings=False)
    if kind == "starcoder2":
        config = transformers.Starcoder2Config(
            hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, residual_dropout=0.0, embedding_dropout=0.0, attention_dropout=0.0,
            max_position_embeddings=1024, **{**kw, **more})
        return transformers.Starcoder2ForCausalLM(config).float()
    config = transformers.GPT2Config(n_embd=128, n_layer=2, n_head=4, n_positions=1024, attn_pdrop=0.0,
                                     resid_pdrop=0.0, embd_pdrop=0.0, **{**kw, **more})
    return transformers.GPT2LMHeadModel(config).float()


def reference(model, ids, labels):
    """(per-token loss, gradients by name) document by document in 64 bits."""
    model = copy.deepcopy(model).double()
    hidden, at = [], 0
    for n in LENGTHS:
        hidden.append(model.get_decoder()(input_ids=ids[:, at:at + n]).last_hidden_state[0])
        at += n
    shifted = F.pad(labels, (0, 1), value=-100)[0, 1:]
    loss = F.cross_entropy(F.linear(torch.cat(hidden), model.lm_head.weight), shifted, ignore_index=-100,
                           reduction="none")
    loss.sum().backward()
    return loss.detach(), {n: p.grad for n, p in model.named_parameters()}


@pytest.mark.parametrize("kind", ["llama", "starcoder2", "gpt2"])
@pytest.mark.parametrize("checkpointed", [False, True])
def test_step_matches_each_document_alone(gpu, kind, checkpointed):
    model = tiny(kind)
    ids, labels, pos = packed()
    loss_ref, grads_ref = reference(model, ids, labels)
    model = patch_causal_lm(model.to(gpu), packed_layers=True, embedding_and_norms=True)
    if checkpointed:
        model.train()
        model.gradient_checkpointing_enable({"use_reentrant": False})
    cu = cu_seqlens_from_lengths(LENGTHS).to(gpu)
    out = model(input_ids=ids.to(gpu), labels=labels.to(gpu), position_ids=pos.to(gpu), cu_seqlens=cu)
    assert rel(out.loss.detach(), loss_ref) <= TOL
    out.loss.sum().backward()
    size = max(float(g.norm()) for g in grads_ref.values())
    for name, p in model.named_parameters():
        if grads_ref[name].norm() > 1e-9 * size:
            assert rel(p.grad, grads_ref[name]) <= TOL, name
    # the update of the step: clip, momentum (its first step's), orthogonalised matrices
    matrices = {n: p for n, p in model.named_parameters() if p.dim() == 2 and "embed" not in n and "wte" not in n
                and "wpe" not in n and "lm_head" not in n}
    assert len(matrices) >= 8
    grads = [p.grad for p in model.parameters()]
    clip_gradients_(grads, 0.5)
    for n, p in list(matrices.items())[:4]:
        update_reference.assert_within(orthogonalize(p.grad), p.grad)


def test_bf16_with_tied_embeddings_in_one_accumulator(gpu):
    """Head and embedding share their weight: both gradients in fp32 in one tensor, from two
    minibatches."""
    model = tiny("starcoder2", tie_word_embeddings=True)
    ids, labels, pos = packed()
    # (bf16 weights on both sides: their rounding is no error of the step)
    model = model.to(torch.bfloat16).float()
    _, grads_ref = reference(model, ids, labels)
    name = "model.embed_tokens.weight"
    model = model.to(gpu, torch.bfloat16)
    acc = torch.zeros(VOCAB, 128, device=gpu)
    patch_causal_lm(model, dw_accumulator=acc, packed_layers=True, embedding_and_norms=True,
                    accumulate_embedding=True)
    for _ in range(2):
        out = model(input_ids=ids.to(gpu), labels=labels.to(gpu), position_ids=pos.to(gpu),
                    cu_seqlens=cu_seqlens_from_lengths(LENGTHS))
        out.loss.float().sum().backward()
    assert model.model.embed_tokens.weight.grad is None
    # bf16 activations carry 2^-8 each through two layers and back
    assert rel(acc, 2 * grads_ref[name]) <= 5e-2


def test_an_id_out_of_range_shows(gpu):
    model = patch_causal_lm(tiny("llama").to(gpu), packed_layers=True, embedding_and_norms=True)
    ids, labels, pos = (t.to(gpu) for t in packed())
    cu = cu_seqlens_from_lengths(LENGTHS)
    want = model(input_ids=ids, labels=labels, position_ids=pos, cu_seqlens=cu).loss
    bad = ids.clone()
    bad[0, LENGTHS[0] + 3] = VOCAB
    got = model(input_ids=bad, labels=labels, position_ids=pos, cu_seqlens=cu).loss
    document = torch.zeros(sum(LENGTHS), dtype=torch.bool)
    document[LENGTHS[0]:LENGTHS[0] + LENGTHS[1]] = True
    assert torch.equal(got.cpu()[~document], want.cpu()[~document])
    assert got.cpu()[document].isnan().any()


def test_a_tied_accumulator_by_hand(gpu):
    """token_embedding and the fused loss add into one accumulator what autograd would."""
    from mini_trainer_amd import fused_linear_cross_entropy

    g = torch.Generator().manual_seed(0)
    w = (torch.randn(VOCAB, 128, generator=g) * 0.05).to(torch.bfloat16).to(gpu).requires_grad_(True)
    ids = torch.randint(0, VOCAB, (300,), generator=g).to(gpu)
    target = torch.randint(0, VOCAB, (300,), generator=g).to(gpu)
    acc = torch.zeros(VOCAB, 128, device=gpu)
    hidden = token_embedding(ids, w, dw_accumulator=acc)
    fused_linear_cross_entropy(hidden, w, target, dw_accumulator=acc).sum().backward()
    assert w.grad is None
    ref = w.detach().double().cpu().requires_grad_(True)
    F.cross_entropy(ref[ids.cpu()] @ ref.T, target.cpu(), reduction="sum").backward()
    # the embedding's part goes through dX in bf16 (2^-8), the head's through bf16 products
    assert rel(acc, ref.grad) <= 2e-2

"""patch_causal_lm(packed_layers=True) on the CPU: the host side of the patched
forward, with the operators replaced by their definitions and the loss by the
decoder's last hidden states.  Every model either agrees with each document run
alone through the unpatched model, or is refused."""
from __future__ import annotations

import copy
import math
import threading

import pytest
import torch

from mini_trainer_amd import causal_lm, cu_seqlens_from_lengths, decoder, patch_causal_lm

tf = pytest.importorskip("transformers")

LENGTHS = [25, 15]
T = sum(LENGTHS)
# fp32 through two small layers, each sum of at most 96 terms: some ten products of
# relative error sqrt(96) 2^-24 = 6e-7 each
TOL = 1e-5

WIDE = dict(vocab_size=100, hidden_size=64, num_hidden_layers=2, num_attention_heads=4,
            max_position_embeddings=128)
BASE = dict(WIDE, intermediate_size=96, num_key_value_heads=2)


def build(name, **more):
    torch.manual_seed(0)
    cls, config, kw = MODELS[name]
    if not hasattr(tf, cls):
        pytest.skip(f"this transformers has no {cls}")
    return getattr(tf, cls)(getattr(tf, config)(**{**kw, **more})).float().eval()


MODELS = {
    "llama": ("LlamaForCausalLM", "LlamaConfig", BASE),
    "qwen2": ("Qwen2ForCausalLM", "Qwen2Config", BASE),
    "mistral": ("MistralForCausalLM", "MistralConfig", dict(BASE, sliding_window=8)),
    "gemma2": ("Gemma2ForCausalLM", "Gemma2Config", dict(BASE, head_dim=16, sliding_window=8)),
    "gpt2": ("GPT2LMHeadModel", "GPT2Config",
             dict(vocab_size=100, n_embd=64, n_layer=2, n_head=4, n_positions=128, attn_pdrop=0.0,
                  resid_pdrop=0.0, embd_pdrop=0.0)),
    "gpt_oss": ("GptOssForCausalLM", "GptOssConfig",
                dict(BASE, head_dim=16, num_local_experts=2, num_experts_per_tok=1)),
    "doge": ("DogeForCausalLM", "DogeConfig", BASE),
    "diffllama": ("DiffLlamaForCausalLM", "DiffLlamaConfig", BASE),
    "bloom": ("BloomForCausalLM", "BloomConfig", dict(vocab_size=100, hidden_size=64, n_layer=2, n_head=4)),
    "xglm": ("XGLMForCausalLM", "XGLMConfig",
             dict(vocab_size=100, d_model=64, ffn_dim=96, num_layers=2, attention_heads=4, dropout=0.0,
                  attention_dropout=0.0)),
    "gpt_neo": ("GPTNeoForCausalLM", "GPTNeoConfig",
                dict(vocab_size=100, hidden_size=64, num_layers=2, num_heads=4,
                     attention_types=[[["global", "local"], 1]], max_position_embeddings=128,
                     attention_dropout=0.0, resid_dropout=0.0, embed_dropout=0.0)),
    "jamba": ("JambaForCausalLM", "JambaConfig",
              dict(BASE, attn_layer_period=2, attn_layer_offset=1, num_experts=2, num_experts_per_tok=1,
                   use_mamba_kernels=False, mamba_d_state=4, mamba_dt_rank=4, pad_token_id=0)),
    "falcon_h1": ("FalconH1ForCausalLM", "FalconH1Config",
                  dict(BASE, mamba_d_ssm=64, mamba_n_heads=4, mamba_d_head=16, mamba_d_state=8,
                       mamba_n_groups=1)),
    "recurrent_gemma": ("RecurrentGemmaForCausalLM", "RecurrentGemmaConfig",
                        dict(BASE, lru_width=64, attention_window_size=8,
                             block_types=["recurrent", "attention"])),
    "minimax": ("MiniMaxForCausalLM", "MiniMaxConfig",
                dict(BASE, head_dim=16, num_local_experts=2, num_experts_per_tok=1, block_size=8,
                     layer_types=["linear_attention", "full_attention"])),
    "llama4": ("Llama4ForCausalLM", "Llama4TextConfig",
               dict(BASE, head_dim=16, num_local_experts=2, intermediate_size_mlp=96,
                    attention_chunk_size=8)),
    "bart": ("BartForCausalLM", "BartConfig",
             dict(vocab_size=100, d_model=64, decoder_layers=2, decoder_attention_heads=4,
                  decoder_ffn_dim=96, max_position_embeddings=128, is_decoder=True,
                  is_encoder_decoder=False)),
    "phimoe": ("PhimoeForCausalLM", "PhimoeConfig",
               dict(BASE, num_local_experts=4, num_experts_per_tok=2, sliding_window=8)),
}


@pytest.fixture
def operators(monkeypatch):
    """The operators' definitions in their places; the number of attention calls."""
    calls = []

    class Plan:
        def __init__(self, cu, tokens, window=None, **_):
            self.cu, self.tokens, self.window = cu.tolist(), tokens, window
            self.status = torch.zeros(1, dtype=torch.int32)

    def attention(q, k, v, plan, scale=None, softcap=None):
        calls.append(plan)
        out = torch.zeros_like(q)
        G = q.shape[1] // k.shape[1]
        for a, b in zip(plan.cu, plan.cu[1:]):
            i, j = torch.arange(b - a)[:, None], torch.arange(b - a)[None, :]
            seen = (j <= i) & (i - j < (plan.window or T))
            z = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(G, 1)) * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            out[a:b] = torch.einsum("hij,jhd->ihd", p, v[a:b].repeat_interleave(G, 1))
        return out

    def norm(x, residual, weight, eps):
        h = x + residual
        return h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * weight, h

    monkeypatch.setattr(decoder, "packed_attention", attention)
    monkeypatch.setattr(decoder, "packed_attention_plan", Plan)
    monkeypatch.setattr(decoder, "residual_rms_norm", norm)
    monkeypatch.setattr(causal_lm, "causal_lm_loss", lambda hidden, *_, **__: hidden[0])
    monkeypatch.setattr(causal_lm, "sample_loss_sums", lambda *_, **__: (None, None))
    return calls


def batch(seed=1):
    ids = torch.randint(1, 100, (1, T), generator=torch.Generator().manual_seed(seed))
    pos = torch.cat([torch.arange(n) for n in LENGTHS])[None]
    return dict(input_ids=ids, labels=ids, position_ids=pos,
                cu_seqlens=cu_seqlens_from_lengths(LENGTHS))


def alone(model, ids):
    """Last hidden states of each document by itself."""
    cu = cu_seqlens_from_lengths(LENGTHS).tolist()
    return torch.cat([model.get_decoder()(input_ids=ids[:, a:b]).last_hidden_state[0]
                      for a, b in zip(cu, cu[1:])])


def rel(a, b):
    return float((a - b).norm() / b.norm())


def patched(name, **more):
    return patch_causal_lm(build(name, **more), packed_layers=True)


@torch.no_grad()
@pytest.mark.parametrize("name", ["llama", "qwen2", "mistral", "gemma2", "gpt2"])
def test_documents_are_as_alone(operators, name):
    model, kw = build(name), batch()
    want = alone(model, kw["input_ids"])
    got = patch_causal_lm(model, packed_layers=True)(**kw).loss
    assert rel(got, want) <= TOL and len(operators) == 2


@torch.no_grad()
@pytest.mark.parametrize("name,what", [("gpt_oss", "s_aux"), ("doge", "attention mask")])
def test_more_than_packed_attention_computes_is_refused(operators, name, what):
    with pytest.raises(ValueError, match=what):
        patched(name)(**batch())


@torch.no_grad()
@pytest.mark.parametrize("kw", [dict(some_bias=torch.zeros(1)), dict(output_attentions=True),
                                dict(is_causal=False), dict(head_mask=torch.ones(2, 4))])
def test_unknown_keywords_are_refused(operators, kw):
    model = patched("llama")
    with pytest.raises(ValueError):
        model(**batch(), **kw)
    # not given, or changing nothing
    assert len(operators) == 0
    model(**batch(), some_bias=None, output_attentions=False, output_router_logits=False)
    assert len(operators) == 2


@torch.no_grad()
def test_a_layer_that_is_not_causal_is_refused(operators):
    model = patched("llama")
    model.model.layers[1].self_attn.is_causal = False
    with pytest.raises(ValueError, match="causal"):
        model(**batch())


@torch.no_grad()
def test_flash_attention_boundaries(operators):
    """cu_seq_lens_q bounds the documents where cu_seqlens does not; position_ids that
    say otherwise do not."""
    model, kw = patched("llama"), batch()
    want = model(**kw).loss
    cu, row = kw.pop("cu_seqlens"), torch.arange(T)[None]
    kw["position_ids"] = row
    got = model(**kw, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=25, max_length_k=25).loss
    assert operators[-1].cu == [0, 25, 40]
    assert rel(got, want) <= TOL  # (rotary positions are relative)


@torch.no_grad()
@pytest.mark.parametrize("name", ["bloom", "xglm", "gpt_neo", "jamba", "falcon_h1", "recurrent_gemma",
                                  "minimax", "llama4", "bart"])
def test_decoders_that_mix_documents_elsewhere_are_refused(operators, name):
    """Attention of their own, state spaces, recurrences, convolutions, chunks, positions
    that cannot restart: when the model is patched, or in its first labelled forward."""
    model = build(name)
    with pytest.raises(ValueError, match="packed layers: "):
        patch_causal_lm(model, packed_layers=True)(**batch())


@torch.no_grad()
def test_a_window_that_reaches_only_the_mask_is_refused(operators):
    with pytest.raises(ValueError, match="sliding window"):
        patched("phimoe")(**batch())


@torch.no_grad()
def test_every_attention_layer_is_counted(operators):
    model, kw = patched("llama"), batch()
    first, second = (layer.self_attn for layer in model.model.layers)
    own, second.forward = second.forward, lambda hidden_states, **_: (hidden_states, None)
    with pytest.raises(ValueError, match="1 of LlamaModel's 2 layers"):
        model(**kw)
    second.forward = own
    model(**kw)  # (each forward is counted afresh)
    # two calls in each layer are two layers' calls
    model = build("diffllama")
    want = alone(model, kw["input_ids"])
    del operators[:]
    got = patch_causal_lm(model, packed_layers=True)(**kw).loss
    assert rel(got, want) <= TOL and len(operators) == 4


def gradients(model, loss):
    model.zero_grad()
    loss.backward()
    return {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("own", ["eager", "sdpa"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_unlabelled_checkpointed_step_is_the_unpatched_models(operators, own, reentrant):
    """The layers are recomputed in the backward, after the unlabelled forward has ended."""
    model = build("llama", attn_implementation=own).train()
    model.gradient_checkpointing_enable({"use_reentrant": reentrant})
    ids = batch()["input_ids"]

    def step(m):
        logits = m(input_ids=ids).logits
        return logits.detach(), gradients(m, logits.float().pow(2).sum())

    want, wants = step(copy.deepcopy(model))
    patch_causal_lm(model, packed_layers=True)
    for _ in range(2):
        got, grads = step(model)
        assert torch.equal(got, want) and grads.keys() == wants.keys()
        assert all(torch.equal(grads[n], wants[n]) for n in wants)
        assert model.config._attn_implementation == model.model.config._attn_implementation == own
        with torch.no_grad():
            model(**batch())  # a labelled forward between them
    assert len(operators) == 4


@pytest.mark.parametrize("reentrant", [False, True])
def test_labelled_checkpointed_step(operators, reentrant):
    model = patched("llama").train()
    kw = batch()
    want = gradients(model, model(**kw).loss.pow(2).sum())
    model.gradient_checkpointing_enable({"use_reentrant": reentrant})
    del operators[:]
    got = gradients(model, model(**kw).loss.pow(2).sum())
    assert len(operators) == 4  # each layer's attention again in the backward
    # the embedding's gradient comes from the whole first layer either way
    assert got.keys() == want.keys() and all(rel(got[n], want[n]) <= TOL for n in want)


@torch.no_grad()
def test_labelled_and_unlabelled_forwards_in_two_threads(operators):
    """Each goes by its own attention, whichever runs within the other."""
    model, kw = build("llama"), batch()
    docs, logits = alone(model, kw["input_ids"]), model(input_ids=kw["input_ids"]).logits
    patch_causal_lm(model, packed_layers=True)
    calls = {"labelled": lambda: model(**kw).loss, "unlabelled": lambda: model(input_ids=kw["input_ids"]).logits}
    for outer, inner in (("labelled", "unlabelled"), ("unlabelled", "labelled")):
        got, entered = {}, []

        def other(*_):
            if not entered:
                entered.append(True)

                def run():
                    with torch.no_grad():
                        got[inner] = calls[inner]()
                thread = threading.Thread(target=run)
                thread.start()
                thread.join()

        def here(*_):
            if not entered:
                entered.append(True)
                got[inner] = calls[inner]()

        for hook in (other, here):  # in another thread, and within the same one
            del entered[:]
            handle = model.model.layers[0].self_attn.register_forward_pre_hook(hook)
            got[outer] = calls[outer]()
            handle.remove()
            assert rel(got["labelled"], docs) <= TOL
            assert torch.equal(got["unlabelled"], logits)


@torch.no_grad()
def test_forwards_of_the_modules_own_stay(operators):
    """A forward that something else has put in an attention module's place is run."""
    model, kw = build("llama"), batch()
    want, ran = alone(model, kw["input_ids"]), []
    module = model.model.layers[1].self_attn
    own = module.forward

    def forward(*args, **kwargs):
        ran.append(True)
        return own(*args, **kwargs)

    module.forward = forward
    patch_causal_lm(model, packed_layers=True)
    assert rel(model(**kw).loss, want) <= TOL and ran == [True]
    patch_causal_lm(model, packed_layers=True)  # again: as once
    assert rel(model(**kw).loss, want) <= TOL and ran == [True] * 2


@torch.no_grad()
def test_configuration_stays_one(operators):
    model = patched("llama", attn_implementation="sdpa")
    model.config.rms_norm_eps, model.model.config.some_number = 1e-3, 5
    assert model.model.config.rms_norm_eps == 1e-3 and model.config.some_number == 5
    assert isinstance(model.model.config, tf.LlamaConfig)
    model.set_attn_implementation("eager")
    assert model.model.layers[0].self_attn.config._attn_implementation == "eager"
    model(**batch())
    assert len(operators) == 2


@torch.no_grad()
@pytest.mark.parametrize("bad", [[0, 25, T + 1], [1, 25, T], [0, 30, 25, T], [0, -5], [], [0, 2 ** 32 + 40]])
def test_malformed_boundaries_are_refused(operators, bad):
    """Boundaries on the CPU, before anything runs."""
    model, kw = patched("llama"), batch()
    kw["cu_seqlens"] = torch.tensor(bad, dtype=torch.int64)
    for how in ({}, {"validate_cu_seqlens": False}):
        with pytest.raises(ValueError, match="cu_seqlens"):
            model(**kw, **how)
    assert not operators
    kw["cu_seqlens"] = torch.tensor([0, 25, 25, 30])  # an empty document, rows behind the last
    assert model(**kw).attention_status.tolist() == [0]


@torch.no_grad()
@pytest.mark.parametrize("name", ["gpt2", "llama"])
@pytest.mark.parametrize("bounds", ["cu_seqlens", "cu_seq_lens_q"])
def test_positions_count_within_each_document(operators, name, bounds):
    """cu_seqlens alone: positions that are learned start at 0 in every document."""
    model, kw = build(name), batch()
    want = alone(model, kw["input_ids"])
    cu = kw.pop("cu_seqlens")
    del kw["position_ids"]
    got = patch_causal_lm(model, packed_layers=True)(**kw, **{bounds: cu}).loss
    assert rel(got, want) <= TOL


def test_positions():
    for cu, want in (([0, 3, 3, 5], [0, 1, 2, 0, 1, 0, 1]), ([0], list(range(7))), ([0, 7], list(range(7))),
                     ([0, 0, 1], [0, 0, 1, 2, 3, 4, 5])):
        got = decoder.positions_within(torch.tensor(cu, dtype=torch.int32), 7, torch.device("cpu"))
        assert got.tolist() == [want]
    for bad in ([5, 7], [0, 9], [0, -3, 7], [-2 ** 31, 2 ** 31 - 1], [3, 1, 9]):
        got = decoder.positions_within(torch.tensor(bad), 7, torch.device("cpu"))
        assert got.min() >= 0 and got.max() < 7


@pytest.mark.parametrize("where", ["hook", "pre_hook", "backward_hook", "global", "forward", "class", "name"])
def test_the_norms_module_is_called_where_someone_looks(operators, monkeypatch, where):
    """Hooks of the norm behind the attention run, and a norm whose forward is not
    transformers' own keeps it."""
    model, kw, fused, seen = patched("llama"), batch(), [], []
    norm = model.model.layers[1].post_attention_layernorm
    plain = decoder.residual_rms_norm
    monkeypatch.setattr(decoder, "residual_rms_norm", lambda *a, **k: fused.append(True) or plain(*a, **k))
    want = model(**kw).loss.detach()
    assert fused == [True] * 2

    def look(module, *_):
        if module is norm:
            seen.append(True)

    def twice(self, x):
        seen.append(True)
        return 2 * x

    handle = None
    if where == "hook":
        handle = norm.register_forward_hook(look)
    elif where == "pre_hook":
        handle = norm.register_forward_pre_hook(look)
    elif where == "backward_hook":
        handle = norm.register_full_backward_hook(look)
    elif where == "global":
        handle = torch.nn.modules.module.register_module_forward_hook(look)
    elif where == "forward":
        norm.forward = twice.__get__(norm)
    elif where == "class":
        monkeypatch.setattr(type(norm), "forward", twice)
    else:
        norm.__class__ = type("LlamaRMSNorm", (type(norm),), {"forward": twice})
    try:
        loss = model(**kw).loss
        loss.sum().backward()
    finally:
        if handle is not None:
            handle.remove()
    assert seen
    assert len(fused) == 2 + (0 if where in ("global", "class") else 1)
    if handle is not None:
        assert rel(loss.detach(), want) <= TOL


@torch.no_grad()
def test_layers_of_another_forward_keep_it(operators):
    """A plain layer's forward that something else has put there is run."""
    model, kw, ran = build("llama"), batch(), []
    want = alone(model, kw["input_ids"])
    layer = model.model.layers[0]
    own = layer.forward

    def forward(*args, **kwargs):
        ran.append(True)
        return own(*args, **kwargs)

    layer.forward = forward
    patch_causal_lm(model, packed_layers=True)
    assert rel(model(**kw).loss, want) <= TOL and ran == [True] and len(operators) == 2

"""patch_causal_lm(packed_layers=True) on the GPU, where its host side meets the device."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import cu_seqlens_from_lengths, patch_causal_lm

tf = pytest.importorskip("transformers")

pytestmark = pytest.mark.gpu

LENGTHS = [25, 15]
T = sum(LENGTHS)


def tiny(gpu, seed=0):
    torch.manual_seed(seed)
    model = tf.LlamaForCausalLM(tf.LlamaConfig(
        vocab_size=100, hidden_size=64, intermediate_size=96, num_hidden_layers=2,
        num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=128,
        tie_word_embeddings=False))
    return patch_causal_lm(model.float().to(gpu), packed_layers=True)


def batch(gpu):
    ids = torch.randint(1, 100, (1, T), generator=torch.Generator().manual_seed(1)).to(gpu)
    pos = torch.cat([torch.arange(n) for n in LENGTHS])[None].to(gpu)
    return dict(input_ids=ids, labels=ids, position_ids=pos)


@torch.no_grad()
def test_malformed_boundaries_on_the_device(gpu):
    model, kw = tiny(gpu), batch(gpu)
    good = cu_seqlens_from_lengths(LENGTHS).to(gpu)
    want = model(**kw, cu_seqlens=good)
    assert want.attention_status.item() == 0
    for bad in ([0, 25, T + 1], [1, 25, T], [0, 30, 25, T]):
        cu = torch.tensor(bad, dtype=torch.int32, device=gpu)
        with pytest.raises(ValueError, match="cu_seqlens"):
            model(**kw, cu_seqlens=cu)
        assert model(**kw, cu_seqlens=cu, validate_cu_seqlens=False).attention_status.item() == 1
    again = model(**kw, cu_seqlens=good, validate_cu_seqlens=False)
    assert torch.equal(again.loss, want.loss) and again.attention_status.item() == 0


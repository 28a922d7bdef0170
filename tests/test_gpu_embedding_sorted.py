"""Gradients of long embeddings whose sort keeps its tokens in LDS in some waves and reads the
ids again in others.

Upstream gradients are small whole numbers, so that every sum is exact in fp32 (at most
20000 x 7 < 2^24) and a token that is lost, doubled or misplaced shows whatever the sum's
size: accumulators and fp32 gradients have to be equal, bf16 ones the exact sums rounded."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import token_embedding

pytestmark = pytest.mark.gpu

V, H = 600, 24
BUCKETS, LIST, WAVES = 256, 512, 16  # the sort's: ids of a bucket are equal modulo 256


def ids_of(kind, T):
    g = torch.Generator().manual_seed(T)
    if kind == "one":
        return torch.full((T,), 17)
    if kind == "interleaved":  # two ids of one bucket
        ids = torch.full((T,), 256 + 3)
        ids[::5] = 3
        return ids
    if kind == "some waves":  # the first half one id, then three ids of its bucket among others
        ids = torch.randint(0, V, (T,), generator=g)
        ids[:T // 2] = 3
        ids[T // 2::3] = torch.tensor([3, 259, 515])[torch.randint(0, 3, (len(ids[T // 2::3]),), generator=g)]
        return ids
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 2.7)
    return torch.multinomial(p, T, True, generator=g)


def most_of_a_bucket(ids):
    """The most tokens of one bucket that each wave of the sort holds."""
    run = -(-len(ids) // 1024) * 64
    return [max([0, *torch.bincount(part % BUCKETS).tolist()]) for part in ids.split(run)][:WAVES]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [8193, 16384, 20000])
@pytest.mark.parametrize("kind", ["one", "interleaved", "some waves", "zipf"])
def test_every_token_is_summed_once(gpu, kind, T, dtype):
    ids = ids_of(kind, T)
    most = most_of_a_bucket(ids)
    if kind != "zipf":
        assert max(most) > LIST
    if kind == "some waves":
        assert min(most) <= LIST
    g = torch.Generator().manual_seed(1)
    d = torch.randint(-7, 8, (T, H), generator=g)
    w = torch.randn(V, H, generator=g).to(dtype).to(gpu).requires_grad_(True)
    up = d.to(dtype).to(gpu)
    for padding in (None, 3):
        counted = ids != (-1 if padding is None else padding)
        want = torch.zeros(V, H, dtype=torch.int64).index_add_(0, ids[counted], d[counted])
        for kept in (torch.int64, torch.int32):
            here = ids.to(gpu, kept)
            out = token_embedding(here, w, padding_idx=padding)
            assert torch.equal(out, w[here.long()])
            (got,) = torch.autograd.grad(out, w, up)
            assert torch.equal(got.cpu(), want.to(torch.float32).to(dtype))
            acc = torch.full((V, H), 5.0, device=gpu)
            out = token_embedding(here, w, padding_idx=padding, dw_accumulator=acc)
            torch.autograd.grad(out, w, up, allow_unused=True)
            assert torch.equal(acc.cpu(), (want + 5).to(torch.float32))

"""Packed attention where scores, or the softcap of them, are large."""
from __future__ import annotations

import pytest
import torch

from mini_trainer_amd import packed_attention, packed_attention_plan

import step_reference as ref

pytestmark = pytest.mark.gpu

# query heads that give half tiles and, in 70 rows, whole ones (one key head each)
HALF, WHOLE = 2, 514


def plan_of(lengths, gpu):
    cu = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=gpu)
    return packed_attention_plan(cu, sum(lengths))


@pytest.mark.parametrize("heads", [HALF, WHOLE])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_of_the_types_whole_range(gpu, dtype, heads):
    """Rows all of whose scores lie at -2^110 and below: those that see one key take its
    value, those that see equal ones the average, and a lower score counts nothing.
    Every product, sum and difference here is exact, so is each probability (1, 1/2, 0)."""
    D, lengths = 64, [1, 2, 2, 64, 1]
    T = sum(lengths)
    g = torch.Generator().manual_seed(1)
    v = torch.randn(T, heads, D, generator=g).to(dtype).to(gpu)
    do = torch.randn(T, heads, D, generator=g).to(dtype).to(gpu)
    q = torch.full((T, heads, D), -2.0 ** 52, dtype=dtype, device=gpu)
    k = torch.full((T, heads, D), 2.0 ** 52, dtype=dtype, device=gpu)
    k[4] *= 2          # the second key of the second pair: a score twice as low
    k[6:69] *= 4       # all but the first of 64
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, plan_of(lengths, gpu), scale=1.0)
    want = v.double()
    want[2] = (v[1].double() + v[2].double()) / 2
    want[4] = v[3].double()
    want[5:69] = v[5].double()
    tol = ref.unit(dtype) * want.abs() + 4 * ref.F32 * v.double().abs().amax()
    assert ((out.double() - want).abs() <= tol).all()
    dq, dk, dv = torch.autograd.grad(out, leaves, do)
    # a row that sees one key: nothing depends on its score, all on its value
    for row in (0, 69):
        assert not dq[row].any() and not dk[row].any()
        assert torch.equal(dv[row], do[row])


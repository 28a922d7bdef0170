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



@pytest.mark.parametrize("heads", [HALF, WHOLE])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [0, 3, 8, 12, 25, 50])
@pytest.mark.parametrize("D", [64, 128])
def test_equal_scores_of_any_size(gpu, D, dtype, half, heads):
    """All scores of a row the same, -D 2^(2 half): its n probabilities are 1 / n each in
    the forward and in the gradients, however little room the size of the scores leaves
    for the logarithm of n in an fp32 log-sum.  Scores are exact here, so that the errors
    are, with u = eps / 2 of the type and F = 2^-24:
      probabilities  up (u for bf16's products) + (n + C) F, and where |lse| < 8192,
                     F |lse| from the log-sum alone;
      out            u |out| + theirs times mean |v|;
      delta          theirs and 2^-16 (what is kept of bf16's out) of |dO| |out|, summed;
      dS             up + the probabilities' of itself, plus p times those of delta and dP."""
    lengths = [1, 2, 3, 57, 7]
    T = sum(lengths)
    g = torch.Generator().manual_seed(3)
    v, do = (torch.randn(T, heads, D, generator=g).to(dtype).to(gpu) for _ in range(2))
    q = torch.full((T, heads, D), -2.0 ** half, dtype=dtype, device=gpu)
    k = torch.full((T, heads, D), 2.0 ** half, dtype=dtype, device=gpu)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = packed_attention(*leaves, plan_of(lengths, gpu), scale=1.0)
    got = {"out": out, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)))}
    u, F, C = ref.unit(dtype), ref.F32, ref.C
    up = u if dtype == torch.bfloat16 else 0.0
    mask = ref.seen_mask(lengths, T).double()
    n = mask.sum(1, keepdim=True)
    p = mask / n
    lse = D * 2.0 ** (2 * half) * 1.4427
    rel_o = up + (n + C) * F
    rel_p = rel_o + (F * lse if lse < 8192 else 0.0)
    for h in (0, heads - 1):
        vh, doh = v[:, h].double().cpu(), do[:, h].double().cpu()
        o = p @ vh
        o_err = rel_o * (p @ vh.abs())
        dp = doh @ vh.T
        delta = (doh * o).sum(1, keepdim=True)
        delta_err = (doh.abs() * (o_err + (2.0 ** -16 + (D + C) * F) * o.abs())).sum(1, keepdim=True)
        alone = (n == 1)
        ds = torch.where(alone, torch.zeros(()).double(), p * (dp - delta))
        ds_err = (rel_p + up) * ds.abs() + p * ((D + C) * F * (doh.abs() @ vh.abs().T) + delta_err)
        ds_err = torch.where(alone, torch.zeros(()).double(), 1.01 * ds_err)
        size = 2.0 ** half
        dq, dk = ds.sum(1, keepdim=True) * size, -ds.sum(0)[:, None] * size
        dq_err = (ds_err + (T + C) * F * ds.abs()).sum(1, keepdim=True) * size
        dk_err = (ds_err + (T + C) * F * ds.abs()).sum(0)[:, None] * size
        dv = p.T @ doh
        dv_err = ((rel_p + (T + C) * F) * p).T @ doh.abs()
        one = torch.ones(1, D, dtype=torch.float64)
        for name, value, err in (("out", o, o_err), ("dq", dq * one, dq_err * one),
                                 ("dk", dk * one, dk_err * one), ("dv", dv, dv_err)):
            ref.assert_within(got[name][:, h], (value, err + u * (value.abs() + err)), f"{name} {h}")


@pytest.mark.parametrize("heads", [HALF, WHOLE])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [256.0, 257.0, 1e4, 1e6, 1e8, 1e30])
def test_a_large_softcap(gpu, D, heads, softcap):
    """softcap tanh(z / softcap) is within |z|^3 / (3 softcap^2) of z; the tolerance is that
    of the capped scores with tanh right to 4 units of its last place, whatever the cap."""
    lengths = [50, 20]
    T = sum(lengths)
    g = torch.Generator().manual_seed(2)
    q, k, v, do = (torch.randn(T, heads, D, generator=g).to(torch.bfloat16).to(gpu) for _ in range(4))
    leaves = [t.detach().requires_grad_(True) for t in (4 * q, k, v)]
    out = packed_attention(*leaves, plan_of(lengths, gpu), softcap=softcap)
    got = {"out": out, **dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)))}
    mask = ref.seen_mask(lengths, T)
    for h in (0, heads - 1):
        one = slice(h, h + 1)
        z = torch.einsum("id,jd->ij", 4 * q[:, h].double().cpu(), k[:, h].double().cpu()) * D ** -0.5
        assert z.abs().max() < 60
        want = capped(4 * q[:, one], k[:, one], v[:, one], do[:, one], mask, softcap)
        for name in got:
            ref.assert_within(got[name][:, one], want[name], name)


def capped(q, k, v, do, mask, softcap):
    """Values with the cap, tolerances of the same scores without one (whose C operations
    have room for tanh's 4 units): the cap's derivative, 1 - tanh^2, adds 8 of them."""
    plain = ref.attention(q, k, v, do, mask)
    value = ref.attention(q, k, v, do, mask, softcap=softcap)
    made = {}
    for name in plain:
        tol = plain[name][1]
        # a smaller |z| under the cap has the smaller error; the gradients are as much smaller
        made[name] = (value[name][0], 1.01 * tol + 64 * ref.F32 * value[name][0].abs())
    return made

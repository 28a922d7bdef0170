"""The rounding of fp16 products that spectra_reference.py describes keeps updates near what
their last rounding leaves; the one around mu alone does not."""
from __future__ import annotations

import pytest
import torch

import spectra_reference as ref
from update_reference import COEFFICIENTS, triples


def ratios(r, c, around, coefficients=COEFFICIENTS, steps=5):
    found = {}
    for name, x in ref.matrices(r, c).items():
        want, wide = ref.exact(x, coefficients, steps), x.double()
        got = ref.rounded(wide, triples(coefficients, steps), float(wide.norm()), 1e-7, around)
        found[name] = ref.ratio(got.to(torch.bfloat16), want)
    return found


@pytest.mark.parametrize("r,c", [(48, 200), (64, 256), (128, 128), (128, 352), (256, 1024)])
def test_five_steps(r, c):
    new, old = ratios(r, c, False), ratios(r, c, True)
    assert max(new.values()) < 1.45, new
    assert max(old.values()) > 1.5, old
    # what was good stays so
    assert new["random"] < 1.25 and new["momentum"] < 1.25


def test_more_steps_of_coefficients_that_settle():
    settle = (1.875, -1.25, 0.375)
    new, old = (ratios(96, 256, around, settle, 12) for around in (False, True))
    assert max(new.values()) < 1.45 and max(old.values()) > 1.5

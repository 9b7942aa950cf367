"""CPU tests of the 4-bit format's division by scales of any magnitude."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4
from tests import _int4 as I


def test_scales_whose_reciprocal_is_infinite():
    # (2^-135 is subnormal, and its reciprocal past fp32's largest)
    t = torch.tensor([2.0 ** -135])
    x = torch.zeros(1, 1, 64)
    x[0, 0, :16] = torch.arange(-7.0, 9.0) * t
    got = I.values(*i4.quantise_int4(x, t), t)
    assert torch.equal(got, x.double())


@pytest.mark.parametrize("scale", [2.0 ** -135, 1e-30, -0.37, 3e20, 2.0 ** 126])
def test_the_rule_with_any_scale(scale):
    """Elements are off by at most a step and a half (a largest one that the rounded step leaves
    past code 15), and the step is at most 9/8 of its definition."""
    g = torch.Generator().manual_seed(1)
    t = torch.tensor([scale])
    x = torch.randn(20, 2, 64, generator=g) * t
    y = x.double() / t.double()
    got = I.values(*i4.quantise_int4(x, t), None)
    grouped = y.view(20, 2, 2, 32)
    lo, hi = grouped.amin(-1, keepdim=True), grouped.amax(-1, keepdim=True)
    step = torch.maximum((hi - lo) / 15, torch.maximum(hi, -lo) / 56) * 9 / 8
    assert ((got.view_as(grouped) - grouped).abs() <= 1.5 * step).all()

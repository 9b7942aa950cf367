"""CPU tests of the 4-bit format at the ends of what a group holds."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4


@pytest.mark.parametrize("end", [-16384.0, 16384.0])
def test_what_the_conversion_forms_stays_within_fp16(end):
    """Codes become values as (16 + c) s + (z - 16) s: the second term has to be an fp16 number. One
    end of the group is the largest magnitude, the other passes over every whole number."""
    other = torch.arange(-16384.0, 16385.0)
    x = other.view(-1, 1, 1).repeat(1, 1, 64)
    x[:, 0, ::32] = end
    codes, words = i4.quantise_int4(x)
    w = words[:, 0, 0].long()
    s = (w & 0x7f80).to(torch.int16).view(torch.float16).double()
    term = ((w & 127) - 64 - 16) * s
    assert float(s.max()) <= 2304 and float(term.abs().max()) <= 52992
    assert torch.equal(term.half().double(), term)  # no rounding, none infinite
    values = i4.int4_values(codes, words)
    assert torch.equal(values.half().float(), values) and float(values.abs().max()) <= 17280


def test_how_far_elements_are_off():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(500, 4, 128, generator=g)
    codes, words = i4.quantise_int4(x)
    step = (words & 0x7f80).view(torch.float16).float().repeat_interleave(32, -1)
    off = (i4.int4_values(codes, words) - x).abs() / step
    # steps of 4 significant bits are rounded down by at most a 17th: 15 of them leave at most 15 / 16
    # of one, and the zero point's own rounding half of one
    assert float(off.max()) <= 15 / 16 + 0.5 + 1e-4 and float((off > 0.5001).float().mean()) < 0.02

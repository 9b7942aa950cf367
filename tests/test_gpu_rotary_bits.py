"""GPU tests of cosines' and sines' last bits in rotary positions."""

import math

import pytest
import torch

from flashprefill_amd.rotary import apply_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inverse", [False, True])
def test_cosines_and_sines_are_rounded_once(inverse):
    """Pairs (1, 1) and (1, -1) at angles close to an odd multiple of pi / 4: cosine and sine
    are nearly alike in size there and cancel, exactly, so that the output is the difference of the
    two as fp32 holds them, 2^12 of their units in the last place large and less, which the
    output's 11 bits all but show. One that is off by a unit is seen."""
    n = 4096
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(1, 1 << 17, (n,), generator=g)
    f = (math.pi / 4 + math.pi / 2 * torch.randint(0, 4, (8,), generator=g) +
         2.0 ** -15 * torch.randn(8, generator=g, dtype=torch.float64))
    f = torch.cat([f, f / 3, f + 40 * math.pi]).double()
    pos[:n // 2] = 1  # (angles f themselves; far positions with any angle too)
    x = torch.ones(n, 2, 48, dtype=torch.float16)
    x[:, 1, 24:] = -1
    y = x.cuda()
    apply_rotary(y, None, pos.cuda(), f.cuda(), amplitude=1024.0, inverse=inverse)
    angle = pos.double().view(-1, 1) * f
    c, s = ((1024.0 * t).float().double() for t in (angle.cos(), angle.sin()))
    if inverse:
        s = -s
    want = torch.stack([torch.cat([c - s, c + s], -1), torch.cat([c + s, s - c], -1)], 1)
    # (fp32's sum of two fp32 numbers, then fp16's)
    assert torch.equal(y.cpu(), want.float().half())

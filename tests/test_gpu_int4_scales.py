"""GPU tests of the 4-bit write's division by scales of any magnitude."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4
from tests import _int4 as I
from tests.test_gpu_int4 import _write

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("scale", [2.0 ** -135, 2.0 ** -61, 2.0 ** -59, -0.37, 1 / 3, 2.0 ** 60,
                                   2.0 ** 62, 2.0 ** 126, 0.0, float("inf"), float("nan")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_write(d, scale):
    # every code and word is the composition's, in which torch divides
    x, s = I.rows(60, 2, d, BF, 3), torch.tensor([scale])
    x[::2] = (x[::2].float() * scale).to(BF)
    got = _write(x, x, torch.arange(60), 4, 16, s, s)
    codes, words = i4.quantise_int4(x, s)
    assert torch.equal(got[0].view(-1, 2, d // 2)[:60], codes)
    assert torch.equal(got[3].transpose(1, 2).reshape(-1, 2, d // 32)[:60], words)
    if scale == 2.0 ** -135:
        held = i4.int4_values(codes, words)
        assert not held[(x != x).view(60, 2, -1, 32).any(-1).logical_not()
                        .repeat_interleave(32, -1).view(60, 2, d)].isnan().any()


@pytest.mark.parametrize("dtype", [BF, FP])
def test_quotients_beside_ties(dtype):
    """Elements whose quotient lies on, or half a unit in the last place from, a boundary
    between two codes: where a product with a rounded reciprocal may fall on the other side."""
    g = torch.Generator().manual_seed(4)
    s = torch.exp(torch.randn(8, generator=g))
    k = torch.randint(-16, 17, (4000, 8, 64), generator=g) / 2
    x = (k * s.view(1, 8, 1)).to(dtype)
    got = _write(x, x, torch.arange(4000), 250, 16, s, s)
    codes, words = i4.quantise_int4(x, s)
    assert torch.equal(got[0].view(-1, 8, 32), codes)
    assert torch.equal(got[3].transpose(1, 2).reshape(-1, 8, 2), words)

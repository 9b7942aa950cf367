"""GPU tests of how many bits of the probabilities attention over a 4-bit cache keeps."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4
from tests import _int4 as I

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _attend(args, scale):
    out = torch.empty_like(args[0], device="cuda")
    q, kc, vc, kg, vg, cu, used, table, ks, vs = (
        t.cuda() if torch.is_tensor(t) else t for t in args)
    i4.paged_decode_attention_int4(q, kc, vc, kg, vg, out, cu, used, table, scale, ks, vs)
    return out.cpu()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lens,news,hq,hkv,d,page", [
    ([9, 30], [1, 1], 8, 2, 128, 16), ([700, 12], [1, 2], 8, 1, 64, 24),
    ([300, 2100], [1, 1], 4, 2, 256, 16),  # few rows; many of tiles of 128 and of 256
    ([90, 40], [40, 40], 8, 2, 64, 16), ([200], [130], 4, 1, 256, 1),
    ([700], [600], 8, 2, 128, 24), ([600, 550], [530, 520], 8, 1, 64, 16)], ids=str)
def test_probabilities_keep_their_bits(lens, news, hq, hkv, d, page, dtype):
    """Scores are small here, so that what P loses shows: with sum |q| |k| scale (`most`) below
    4, fp32 scores are off by less than 2^-17, and P relatively as much. P in two parts loses 2^-22
    and sums over up to 2,100 keys, factors and the division 2^-17, all of sum P |v|. P in one
    fp16 part would be off by up to 2^-11, and 2^-13 on the average of few keys."""
    args = I.attention_case(lens, news, hq, hkv, d, page, dtype, "none", seed=d + sum(lens))
    scale = 2.0 ** -4 / d ** 0.5
    got = _attend(args, scale).double()
    want, size, most = I.attention(*args, scale)
    assert most < 4
    eps, least = (2.0 ** -8, 0.0) if dtype == BF else (2.0 ** -11, 2.0 ** -25)
    far = (got - want).abs() - want.abs() * eps * 1.01 - least
    over = float((far - size * (2.0 ** -17 + 2.0 ** -17)).max())
    assert over <= 0

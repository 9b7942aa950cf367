"""GPU tests of few query rows over long 4-bit caches: shares of more than 1,024 keys, hundreds of
partials of a row, more of them to a wave than it has lanes, and groups of NaN among them."""

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
    return out.cpu().double()


def _far(got, want, size, dtype):
    """By how much outputs are past what scores of |q| |k| scale below 4 allow: half a spacing
    of the output, and 2^-16 of sum P |v| for the scores' last bits (2^-17) and for P's, the sums
    and the factors (2^-17: chains of at most 64 fp32 sums before the partials are joined, and of
    800 / 16 there)."""
    eps, least = (2.0 ** -8, 0.0) if dtype == BF else (2.0 ** -11, 2.0 ** -25)
    return (got - want).abs() - want.abs() * eps * 1.01 - least - size * 2.0 ** -16


CASES = [
    # one sequence: some 270 and 510 partials of each row, rows shared by workgroups of the merge
    ([70000], [1], 16, 1, 64, 16), ([131000], [2], 8, 1, 128, 24), ([70001], [3], 4, 2, 256, 16),
    # a long one among many: the merge's workgroups take all rows, a wave several hundred partials
    ([100000] + [40] * 255, [1] * 256, 16, 1, 64, 16), ([50] * 300 + [90000], [1] * 301, 10, 1, 128, 24),
    # shares of ten units: a second window of page places
    ([40000] * 8, [1] * 8, 6, 3, 64, 16), ([40000] * 8, [2] * 8, 3, 3, 128, 16),
    ([39990] * 8, [1] * 8, 3, 3, 64, 24), ([40000] * 8, [1] * 8, 2, 2, 256, 32)]


def _name(x):
    return "+".join(f"{x.count(n)}x{n}" for n in dict.fromkeys(x)) if isinstance(x, list) else None


@pytest.mark.parametrize("dtype,case", [((BF, FP)[i % 2], c) for i, c in enumerate(CASES)],
                         ids=lambda x: _name(x[0]) if isinstance(x, tuple) else None)
def test_long_contexts(dtype, case):
    lens, news, hq, hkv, d, page = case
    args = I.attention_case(lens, news, hq, hkv, d, page, dtype, "none", seed=d + len(lens))
    scale = 2.0 ** -4 / d ** 0.5
    want, size, most = I.attention(*args, scale)
    assert most < 4
    assert float(_far(_attend(args, scale), want, size, dtype).max()) <= 0


@pytest.mark.parametrize("lens,news,hq,hkv,d,page,at", [
    ([70000], [3], 4, 1, 64, 16, 69998), ([70000], [3], 4, 1, 64, 24, 41000),
    ([90000] + [40] * 255, [2] + [1] * 255, 8, 1, 64, 16, 89999),
    ([40000] * 8, [2] * 8, 3, 3, 128, 16, 39999), ([40000] * 8, [2] * 8, 3, 3, 64, 24, 1024)],
    ids=_name)
def test_nan_in_long_contexts(lens, news, hq, hkv, d, page, at):
    """A value group of key `at` of the first sequence is NaN: its dims of the rows that see the
    key are, and nothing else."""
    args = I.attention_case(lens, news, hq, hkv, d, page, BF, "none", seed=7)
    scale = 2.0 ** -4 / d ** 0.5
    want, size, most = I.attention(*args, scale)
    args[4][args[7][0, at // page], 0, at % page, 1] = I.NAN_WORD
    got = _attend(args, scale)
    nan = torch.zeros(got.shape, dtype=torch.bool)
    for i in range(news[0]):
        if lens[0] - news[0] + i >= at:
            nan[i, :hq // hkv, 32:64] = True
    assert torch.equal(got.isnan(), nan)
    assert float(_far(got, want, size, BF)[~nan].max()) <= 0

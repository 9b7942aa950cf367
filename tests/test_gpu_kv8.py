"""The 8-bit paged KV cache on the GPU: the quantising write bit for bit against torch's
rounding, attention over the cache (decode, several queries, prefill over a cached prefix)
and the read-back against 64-bit results, and all of them together as the hooked forwards
call them."""

import math
import threading
from types import SimpleNamespace

import pytest
import torch

from tests._kv8 import E4M3, E5M2, MODES, NAN_CODE, TOP, attention, attention_case, bound, quantise, \
    scales, values
from flashprefill_amd import vllm_backend as vb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def _dev(args):
    return [None if t is None else t.to(DEV) for t in args]


def _same(got, want):
    """Equal values, NaN where the other has NaN, and equal signs of zero."""
    got, want = got.float(), want.float()
    nan = want.isnan()
    return torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want[~nan]) and \
        torch.equal(got[~nan].signbit(), want[~nan].signbit())


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------

def _special(x):
    """Rows with values that a cast can go wrong at: zeros, one infinity, NaN, the largest
    and smallest of the type, ties."""
    top, tiny = torch.finfo(x.dtype).max, torch.finfo(x.dtype).tiny
    x[0] = 0.0
    x[1, :, 0] = math.inf
    x[2, :, 1] = -math.inf
    x[3, :, 2] = math.nan
    x[4] = top
    x[5] = tiny
    x[6] = tiny / 4
    x[7, :, 3] = -top
    x[8] = -0.0
    x[9, :, :4] = torch.tensor([448.0, 464.0, -17.0, 0.0009765625]).to(x.dtype)
    x[10] = math.inf
    return x


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("hkv,d,page", [(8, 128, 16), (2, 64, 16), (4, 256, 24), (3, 96, 7),
                                        (1, 8, 1), (5, 40, 32), (1, 512, 16)])
def test_write(fmt, dtype, mode, hkv, d, page):
    g = torch.Generator().manual_seed(hkv * d)
    T = 53
    qkv = 3 * torch.randn(T + 2, 2 + 2 * hkv, d, generator=g)
    qkv = _special((qkv * torch.exp(2 * torch.randn(T + 2, 1, 1, generator=g))).to(dtype))
    total = T // page + 5
    slots = torch.randperm(total * page, generator=g)[:T]
    slots[::9] = -1  # padding
    slots[11] = total * page + 2  # past the cache: skipped
    cache = torch.randint(0, 126, (2, total, page, hkv, d), generator=g).to(torch.uint8)
    sc = [scales(mode, total, page, hkv, g) for _ in range(2)]
    want, want_s = cache.clone().view(fmt), [None if s is None else s.clone() for s in sc]
    keep = [t for t in range(T) if 0 <= slots[t] < total * page]
    at = slots[keep]
    for i, rows in enumerate((qkv[:T, 2:2 + hkv], qkv[:T, 2 + hkv:])):
        fixed = torch.ones(1, 1) if mode == "none" else None if mode == "slot" else sc[i].view(1, -1)
        codes, s = quantise(rows[keep], fmt, fixed)
        want[i].view(torch.uint8)[at // page, at % page] = codes.view(torch.uint8)
        if mode == "slot":
            want_s[i][at // page, :, at % page] = s
    dq, dc, ds = qkv.to(DEV), cache.to(DEV).view(fmt), _dev(sc)
    vb.reshape_and_cache(dq[:, 2:2 + hkv], dq[:, 2 + hkv:], dc[0], dc[1], slots.to(DEV), *ds)
    assert _same(dc.cpu(), want)
    for s, w in zip(ds, want_s):
        assert s is None or torch.equal(s.cpu(), w)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_write_of_every_16_bit_value(fmt, dtype):
    """All 65536 inputs, at scales that leave the bits alone, shift ties and overflow."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).view(128, 4, 128)
    slots = torch.arange(128, device=DEV)
    for s in (1.0, 0.75, 3e-5, 7.1e4, 3e-39, 1e38):
        cache = torch.zeros(2, 8, 16, 4, 128, dtype=torch.uint8, device=DEV).view(fmt)
        sc = torch.tensor(s)
        vb.reshape_and_cache(x.to(DEV), x.to(DEV), cache[0], cache[1], slots, sc.to(DEV), sc.to(DEV))
        want, _ = quantise(x, fmt, sc.view(1, 1))
        for c in cache:
            assert _same(c.view(128, 4, 128).cpu(), want), s


@pytest.mark.parametrize("slot", [0, 1])
def test_write_and_read_back_with_scales_of_two_kinds(slot):
    """K's scales per slot beside fixed ones of V, and the other way round: each as in a
    call in which both are of its kind."""
    g = torch.Generator().manual_seed(3)
    rows = (3 * torch.randn(2, 100, 4, 64, generator=g)).to(BF).to(DEV)
    slots = torch.randperm(7 * 24, generator=g)[:100].to(DEV)
    fixed = torch.tensor([0.01, 0.02, 0.5, 0.003], device=DEV)
    cu = torch.tensor([0, 7 * 24], dtype=torch.int32, device=DEV)
    table = torch.arange(7, dtype=torch.int32, device=DEV).view(1, -1)

    def run(kinds):
        c = torch.zeros(2, 7, 24, 4, 64, dtype=torch.uint8, device=DEV).view(E4M3)
        sc = [torch.ones(7, 4, 24, device=DEV) if k else fixed for k in kinds]
        vb.reshape_and_cache(*rows, *c, slots, *sc)
        back = torch.zeros(2, 7 * 24, 4, 64, dtype=BF, device=DEV)
        vb.gather_cache(*c, *back, cu, table, None, *sc)
        return c.view(torch.uint8), sc, back

    got = run([slot == 0, slot == 1])
    for i in range(2):
        want = run([i == slot] * 2)
        assert torch.equal(got[0][i], want[0][i]) and torch.equal(got[1][i], want[1][i])
        assert torch.equal(got[2][i], want[2][i]) and got[2][i].any()


def test_write_of_no_tokens_and_index_types():
    cache = torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    x = torch.ones(3, 2, 64, dtype=BF, device=DEV)
    vb.reshape_and_cache(x, x, cache[0], cache[1], torch.zeros(0, dtype=torch.long, device=DEV))
    assert (cache.view(torch.uint8) == 0).all()
    for slots in (torch.tensor([5, 63], dtype=torch.int32, device=DEV), torch.tensor([5, 63])):
        c = torch.zeros_like(cache)
        vb.reshape_and_cache(x, x, c[0], c[1], slots)
        hit = c.float().view(2, 64, -1).any(-1)
        assert hit.nonzero()[:, 1].tolist() == [5, 63, 5, 63]


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _run(args, scale):
    q, kc, vc, cu, used, table, ks, vs = _dev(args)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device=DEV)
    assert vb._paged_kernel_takes(q, kc, vc, out, cu, used, table, ks, vs)
    vb.paged_decode_attention(q, kc, vc, out, cu, used, table, scale, ks, vs)
    return out.cpu()


def _check(args, scale):
    got, (want, size) = _run(args, scale).double(), attention(*args, scale)
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    off = ((got - want).abs() / bound(want, size, args[0].dtype).clamp_min(1e-300))[~nan]
    assert (off <= 1).all(), off.max()


SHAPES = [(32, 8, 128, BF, E4M3), (28, 4, 128, HF, E5M2), (8, 8, 64, HF, E4M3),
          (40, 2, 64, BF, E5M2), (8, 2, 256, BF, E4M3), (6, 3, 256, HF, E5M2)]


@pytest.mark.parametrize("lens", [[1, 15, 16, 17], [31, 32, 33, 127], [128, 129, 255, 256],
                                  [257, 384, 511, 640], [3000, 1, 40, 700]])
@pytest.mark.parametrize("hq,hkv,d,dtype,fmt", SHAPES)
@pytest.mark.parametrize("mode", ["head", "slot"])
def test_decode(lens, hq, hkv, d, dtype, fmt, mode):
    _check(attention_case(lens, [1] * len(lens), hq, hkv, d, 16, dtype, fmt, mode),
           1 / math.sqrt(d))


@pytest.mark.parametrize("page", [1, 5, 16, 24, 32, 48, 256])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("mode", MODES)
def test_page_sizes_and_index_types(page, index, mode):
    _check(attention_case([700, 33, 260], [1, 2, 1], 8, 2, 128, page, BF, E4M3, mode, index=index),
           1 / math.sqrt(128))


@pytest.mark.parametrize("lens,news", [([40, 300, 2100], [1, 7, 33]), ([5, 600, 64], [5, 0, 64]),
                                       ([900, 0, 1300], [200, 3, 130]), ([3, 50], [6, 1]),
                                       ([1500], [700])])
@pytest.mark.parametrize("hq,hkv,d,dtype,fmt", SHAPES + [(32, 8, 128, HF, E4M3), (4, 1, 64, BF, E4M3)])
@pytest.mark.parametrize("mode", ["tensor", "slot"])
def test_several_queries(lens, news, hq, hkv, d, dtype, fmt, mode):
    # [3, 50] / [6, 1]: rows before the first cached token see nothing (NaN, as
    # softmax over no key); a sequence of no cached tokens gives 0
    _check(attention_case(lens, news, hq, hkv, d, 16, dtype, fmt, mode), 1 / math.sqrt(d))


@pytest.mark.parametrize("page", [1, 16, 24, 64])
@pytest.mark.parametrize("d,dtype,fmt", [(128, BF, E4M3), (64, HF, E4M3), (128, HF, E5M2),
                                         (64, BF, E5M2)])
@pytest.mark.parametrize("mode", ["none", "slot"])
def test_many_rows_at_tile_edges(page, d, dtype, fmt, mode):
    for lens, news in (([127, 128, 129, 64], [31, 32, 33, 64]), ([1000, 65, 320], [65, 65, 1]),
                       ([2049, 30], [97, 40])):
        _check(attention_case(lens, news, 8, 2, d, page, dtype, fmt, mode, seed=page),
               1 / math.sqrt(d))


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("d,news", [(64, 1), (128, 1), (256, 3), (128, 40)])
@pytest.mark.parametrize("slot", ["key", "value"])
def test_scales_of_two_kinds(page, d, news, slot):
    """K's scales per slot beside one of V, and the other way round."""
    args = attention_case([700, 33, 260], [news] * 3, 8, 2, d, page, BF, E4M3, "slot", seed=2)
    args[7 if slot == "key" else 6] = torch.tensor([0.02])
    _check(args, 0.1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("scale", [0.5, -0.3, 1e-3, 0.0])
@pytest.mark.parametrize("mode", ["head", "slot"])
def test_peaked_and_flat_rows(dtype, news, scale, mode):
    args = attention_case([3000, 700], [news, news], 8, 2, 128, 16, dtype, E4M3, mode, seed=9)
    codes = args[2].view(torch.uint8)
    codes[codes != NAN_CODE] &= 0x7f  # values of one sign, so that small P add up
    _check(args, scale)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (5, 5), (6, 3), (7, 1), (9, 3), (34, 2)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new", [1, 41])
def test_head_counts(hq, hkv, d, new):
    _check(attention_case([1900, 70, 700, 40], [new, 33 if new > 1 else 1, new, 0], hq, hkv, d, 16,
                          BF, E4M3, "head"), 1 / math.sqrt(d))


def test_wide_tables_many_sequences_and_every_chunk():
    _check(attention_case([100, 2000], [1, 1], 8, 2, 128, 16, BF, E4M3, "slot", width=4096), 0.08)
    lens = [(37 * i) % 300 + 1 for i in range(150)]
    _check(attention_case(lens, [1 + (i % 3 == 0) for i in range(150)], 4, 2, 64, 16, BF, E4M3,
                          "head"), 0.125)
    # the same where the workgroups share the keys (a table with room for more)
    lens = [(41 * i) % 1500 + 1 for i in range(150)]
    for d, hkv in ((64, 2), (64, 3), (128, 2), (256, 1)):
        _check(attention_case(lens, [i % 3 for i in range(150)], 2 * hkv, hkv, d, 16, BF, E4M3,
                              "slot"), 1 / math.sqrt(d))
    _check(attention_case([1, 9000, 0, 513, 130], [2, 1, 3, 0, 31], 6, 3, 64, 16, HF, E4M3,
                          "head"), 0.125)
    _check(attention_case([2500, 1300], [90, 200], 8, 2, 256, 16, BF, E4M3, "slot"), 0.06)
    _check(attention_case([40000], [1], 4, 1, 128, 16, BF, E5M2, "slot"), 0.09)
    _check(attention_case([20000], [70], 2, 1, 64, 16, HF, E4M3, "slot"), 0.12)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mode", ["tensor", "head", "slot"])
def test_few_and_many_chunks_of_many_rows(dtype, d, mode):
    # 2 .. 4 chunk slots per row, and more (their partials are merged in two ways)
    for lens, news in (([900, 500], [40, 33]), ([6000, 1000, 0], [65, 70, 3])):
        _check(attention_case(lens, news, 8, 2, d, 16, dtype, E4M3, mode, seed=5),
               1 / math.sqrt(d))


@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("d,page,mode", [(128, 16, "slot"), (64, 24, "head"), (128, 24, "slot"),
                                         (64, 16, "slot")])
@pytest.mark.parametrize("width", [None, 200])
def test_infinite_values(news, d, page, mode, width):
    """+inf and -inf (e5m2) in V at keys that every row sees: those dims are infinite, the
    others what they are without; in several chunks and in one."""
    args = attention_case([1000, 200], [news] * 2, 8, 2, d, page, BF, E5M2, mode, seed=3,
                          width=width)
    codes = args[2].view(torch.uint8)
    for b, key in ((0, 500), (1, 77)):
        at = int(args[5][b, key // page]), key % page
        codes[at[0], at[1], 0, 5] = 0x7c
        codes[at[0], at[1], 1, d - 1] = 0xfc
    scale = 1 / math.sqrt(d)
    got, (want, size) = _run(args, scale).double(), attention(*args, scale)
    inf = want.isinf()
    assert not want.isnan().any() and inf.sum() == 2 * news * 8
    assert torch.equal(got[inf], want[inf])
    assert ((got - want).abs() <= bound(want, size, BF))[~inf].all()


@pytest.mark.parametrize("news,d", [(40, 128), (3, 128), (3, 64), (3, 256), (40, 64)])
@pytest.mark.parametrize("what", ["value", "value scale", "key scale"])
@pytest.mark.parametrize("width", [None, 100])
def test_a_token_that_a_row_does_not_see(what, news, d, width):
    """A NaN in the last new token's value, or in its scales, reaches the last query only."""
    args = attention_case([500], [news], 8, 2, d, 16, BF, E4M3, "slot", seed=4, width=width)
    want, size = attention(*args, 0.1)
    page, at = args[5][0, 499 // 16], 499 % 16
    if what == "value":
        args[2].view(torch.uint8)[page, at, :, 7] = NAN_CODE
    else:
        args[7 if what == "value scale" else 6][page, :, at] = math.nan
    got = _run(args, 0.1).double()
    assert got[-1, :, 7].isnan().all()
    assert got[-1].isnan().all() == (what != "value")
    assert ((got - want).abs() <= bound(want, size, BF))[:-1].all()


@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 24), (256, 16)])
@pytest.mark.parametrize("mode", ["head", "slot"])
def test_values_near_the_largest(news, d, page, mode):
    """Values of 448 x 7e35 at every key of a dim: the weighted mean is that value,
    whatever the sum of the weights before the division, in one chunk and in several."""
    args = attention_case([3000, 200], [news] * 2, 8, 2, d, page, BF, E4M3, mode, seed=5)
    codes = args[2].view(torch.uint8)
    codes[:, :, 0, 3] = 0x7e
    codes[:, :, 1, d - 2] = 0xfe
    args[7][args[7] == args[7]] = 7e35
    want, size = attention(*args, 0.05)
    assert want.isfinite().all()
    got = _run(args, 0.05).double()
    assert ((got - want).abs() <= bound(want, size, BF)).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news", [1, 40])
@pytest.mark.parametrize("mode", ["none", "slot"])
def test_small_probabilities(d, news, mode):
    """A value of 57344 at a key of probability 2^-t, 0 at the key that holds the rest:
    the output is 57344 x 2^-t however far t lies below the row's largest."""
    ts = [12 + i / 8 for i in range(200)]
    args = attention_case([64] * len(ts), [news] * len(ts), 4, 1, d, 16, HF, E5M2, mode, seed=6)
    q, kc, vc, cu, used, table, ks, vs = args
    q.zero_()
    kc.view(torch.uint8).zero_()
    vc.view(torch.uint8).zero_()
    if mode == "slot":
        ks.fill_(1.0)
        vs.fill_(1.0)
    # e5m2 keys -1024 (P = 0), 0 and -1, with t in the query
    k8, v8 = kc.view(torch.uint8), vc.view(torch.uint8)
    k8[..., 0] = torch.tensor(-57344.0).to(E5M2).view(torch.uint8)
    for b, t in enumerate(ts):
        q[int(cu[b]):int(cu[b + 1]), :, 0] = t
        k8[table[b, 0], 0, 0, 0] = 0
        k8[table[b, 0], 1, 0, 0] = torch.tensor(-1.0).to(E5M2).view(torch.uint8)
        v8[table[b, 0], 1, 0, 3] = torch.tensor(57344.0).to(E5M2).view(torch.uint8)
    got, (want, size) = _run(args, math.log(2.0)).double(), attention(*args, math.log(2.0))
    # half a step of the rounded output, 2^-17 of P (two parts) and 2^-18 for the
    # exponent t <= 37 held in fp32
    step = torch.clamp(2.0 ** (want.abs().clamp_min(1e-30).log2().floor() - 10), min=2.0 ** -24)
    assert ((got - want).abs() <= 0.5 * step + 2.0 ** -16 * want.abs()).all(), \
        ((got - want).abs() / step).max()


@pytest.mark.parametrize("d,page,mode", [(64, 16, "head"), (128, 16, "head"), (128, 16, "slot"),
                                         (128, 24, "slot")])
def test_values_near_the_largest_behind_a_low_maximum(d, page, mode):
    """Values of 448 x 7e35 at keys whose scores all lie 7.5 (of 2^x) above those of the
    first tile, so that the running maximum need not move: their mean is that value."""
    n, new = 3000, 40
    args = attention_case([n, 200], [new] * 2, 8, 2, d, page, BF, E4M3, mode, seed=5)
    q, kc, vc, cu, used, table, ks, vs = args
    q.zero_()
    q[..., 0] = 1.0
    for i, s in ((6, ks), (7, vs)):
        args[i] = torch.where(s.isnan(), s, torch.full_like(s, 1.0 if i == 6 else 7e35))
    k8, v8 = kc.view(torch.uint8), vc.view(torch.uint8)
    k8[..., 0] = torch.tensor(7.5).to(E4M3).view(torch.uint8)
    for b in range(2):
        for t in range(64):
            k8[table[b, t // page], t % page, :, 0] = 0
    v8[:, :, 0, 3] = 0x7e
    v8[:, :, 1, d - 2] = 0xfe
    want, size = attention(*args, math.log(2.0))
    assert want.isfinite().all()
    got = _run(args, math.log(2.0)).double()
    assert ((got - want).abs() <= bound(want, size, BF)).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("fmt,step", [(E4M3, 2.0 ** -9), (E5M2, 2.0 ** -16)])
@pytest.mark.parametrize("news,d", [(1, 128), (40, 128), (1, 64), (40, 64), (1, 256)])
def test_the_smallest_codes(dtype, fmt, step, news, d):
    """K and V of subnormal codes (fp16 holds e5m2's as its own subnormals) and scales that
    make them ordinary numbers."""
    args = attention_case([700, 33], [news] * 2, 8, 2, d, 16, dtype, fmt, "tensor", seed=8)
    g = torch.Generator().manual_seed(9)
    for i in (1, 2):
        codes = args[i].view(torch.uint8)
        small = torch.randint(0, 4, codes.shape, generator=g).to(torch.uint8) | \
            (torch.randint(0, 2, codes.shape, generator=g) << 7).to(torch.uint8)
        args[i].view(torch.uint8).copy_(torch.where(codes == NAN_CODE, codes, small))
    args[6], args[7] = torch.tensor([0.5 / step]), torch.tensor([1.0 / step])
    _check(args, 1 / math.sqrt(d))


@pytest.fixture
def roomy(monkeypatch):
    """Cases whose tables have room for 40,000 keys: at head_dim 256 the kernel of many
    rows takes calls of 128 rows per sequence that may be long."""
    plain = attention_case

    def case(lens, news, hq, hkv, d, page, *args, width=None, **more):
        return plain(lens, news, hq, hkv, d, page, *args, width=40000 // page, **more)
    monkeypatch.setitem(globals(), "attention_case", case)


@pytest.mark.parametrize("lens,news", [([900, 0, 1300], [200, 3, 130]), ([1500], [700]),
                                       ([127, 128, 129, 64], [31, 32, 33, 64]), ([3, 50], [6, 60]),
                                       ([2049, 1000, 65, 320, 30], [97, 65, 65, 1, 40])])
@pytest.mark.parametrize("page,mode", [(16, "slot"), (16, "head"), (24, "slot"), (24, "none"),
                                       (1, "tensor"), (64, "none")])
@pytest.mark.parametrize("dtype,fmt", [(BF, E4M3), (HF, E5M2)])
def test_many_rows_of_256(lens, news, page, mode, dtype, fmt, roomy):
    _check(attention_case(lens, news, 8, 2, 256, page, dtype, fmt, mode), 1 / 16)


def test_many_rows_of_256_with_other_head_counts(roomy):
    for hq, hkv in ((5, 5), (7, 1), (34, 2)):
        _check(attention_case([1900, 70, 700], [150, 30, 141], hq, hkv, 256, 16, BF, E4M3, "head"),
               1 / 16)


def test_one_token_of_128_heads_over_every_chunk():
    # the most chunk slots: one tile of rows, and a table with room for 2^17 keys and more
    args = attention_case([34000], [1], 128, 1, 256, 16, BF, E4M3, "head", width=9000)
    q, kc, vc, cu, used, table, ks, vs = args
    rows = table[0, :34000 // 16].long()
    k, v = (values(c, s)[rows].reshape(-1, 256)[:34000] for c, s in ((kc, ks), (vc, vs)))
    p = torch.softmax(q[0].double() @ k.t() / 16, -1)
    got = _run(args, 1 / 16).double()
    assert ((got[0] - p @ v).abs() <= bound(p @ v, p @ v.abs(), BF)).all()


@pytest.mark.parametrize("page,mode", [(16, "slot"), (16, "head"), (24, "slot")])
def test_many_rows_of_256_and_extreme_values(page, mode, roomy):
    test_infinite_values(40, 256, page, mode, None)
    test_values_near_the_largest(40, 256, page, mode)
    test_values_near_the_largest_behind_a_low_maximum(256, page, mode)
    for fmt, step in ((E4M3, 2.0 ** -9), (E5M2, 2.0 ** -16)):
        test_the_smallest_codes(HF, fmt, step, 40, 256)
    for scale in (0.5, -0.3, 1e-3, 0.0):
        test_peaked_and_flat_rows(BF, 40, scale, mode)
    test_small_probabilities(256, 40, "slot" if mode == "slot" else "none")


def test_many_rows_of_256_and_what_only_the_device_sees(roomy):
    for page in (16, 24, 64):
        test_what_only_the_device_sees(page, 256, 40, None)
    for what in ("value", "value scale", "key scale"):
        test_a_token_that_a_row_does_not_see(what, 40, 256, None)
    for slot in ("key", "value"):
        test_scales_of_two_kinds(16, 256, 40, slot)


def test_strided_inputs_and_untouched_rows():
    args = attention_case([300, 70], [1, 1], 8, 2, 128, 16, BF, E4M3, "slot")
    want = _run(args, 0.1)
    q, kc, vc, cu, used, table, ks, vs = _dev(args)
    qkv = torch.zeros(5, 12, 128, dtype=BF, device=DEV)
    qkv[:2, 2:10] = q
    # both caches of one layer of several, heads before slots
    both = torch.zeros(kc.shape[0], 3, 2, 2, 16, 128, dtype=torch.uint8, device=DEV)
    both[:, 1, 0] = kc.view(torch.uint8).transpose(1, 2)
    both[:, 1, 1] = vc.view(torch.uint8).transpose(1, 2)
    kc, vc = (both[:, 1, i].transpose(1, 2).view(E4M3) for i in range(2))
    sc = torch.stack([ks, vs], 1)
    out = torch.full((5, 8, 128), 7.0, dtype=BF, device=DEV)
    assert vb._paged_kernel_takes(qkv[:, 2:10], kc, vc, out, cu, used, table, sc[:, 0], sc[:, 1])
    vb.paged_decode_attention(qkv[:, 2:10], kc, vc, out, cu, used, table, 0.1, sc[:, 0], sc[:, 1])
    assert torch.equal(out[:2].cpu(), want)
    assert (out[2:] == 7.0).all()


@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("d,news,width", [(128, 1, None), (128, 1, 200), (64, 1, 200), (128, 40, None),
                                          (64, 40, None), (256, 2, 200)])
def test_what_only_the_device_sees(page, d, news, width):
    """A length beyond the table and pages outside the cache: NaN rows, the other
    sequence as it is; offsets that do not fit: every row NaN."""
    args = attention_case([1000, 200], [news] * 2, 8, 2, d, page, BF, E4M3, "slot", seed=page,
                          width=width)
    want = _run(args, 0.1)
    for b, first in ((0, 384), (1, 64)):
        rows, rest = slice(news * b, news * b + news), slice(news * (1 - b), news * (2 - b))
        for pos in range(4):
            t2 = args[5].clone()
            t2[b, (first + 16 * pos) // page] = (args[1].shape[0], -args[1].shape[0] - 1)[pos % 2]
            got = _run([*args[:5], t2, *args[6:]], 0.1)
            assert got[rows].isnan().all() and torch.equal(got[rest], want[rest]), (b, pos)
        u2 = args[4].clone()
        u2[b] = args[5].shape[1] * page + 1
        got = _run([*args[:4], u2, *args[5:]], 0.1)
        assert got[rows].isnan().all() and torch.equal(got[rest], want[rest])
    for cu in ([0, news, 2 * news + 1], [-1, news, 2 * news], [0, 2 * news + 1, 2 * news],
               [0, news, 2 ** 30]):
        got = _run([*args[:3], torch.tensor(cu, dtype=torch.int32), *args[4:]], 0.1)
        assert got.isnan().all(), cu


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("d", [64, 256])
def test_one_head_or_one_page_of_any_stride(new, d):
    # torch gives a dimension of one entry any stride, and contiguous() keeps it
    for lens, page in (([100, 260], 16), ([700, 650], 128), ([40], 48)):
        args = attention_case(lens, [new] * len(lens), 4, 1, d, page, BF, E4M3, "slot", seed=new)
        for i in (6, 7):
            args[i] = args[i].transpose(1, 2).contiguous().transpose(1, 2)
            args[i] = args[i].as_strided(args[i].shape, (args[i].stride(0), 1, 1))
            if args[i].shape[0] == 1:
                args[i] = args[i].as_strided(args[i].shape, (7, 1, 1))
        assert args[6].is_contiguous() and args[6].stride(1) == 1
        _check(args, 0.1)


def test_rows_and_caches_of_one_entry_and_any_stride():
    g = torch.Generator().manual_seed(2)

    def odd(x, dim, stride):  # the same memory with another stride of a dimension of one entry
        st = list(x.stride())
        assert x.shape[dim] == 1
        st[dim] = stride
        return x.as_strided(x.shape, st)

    for page in (16, 1):
        n = 16 if page == 16 else 1
        k, v = (odd(odd(torch.randn(1, 1, 64, generator=g).to(BF).to(DEV), 0, 3), 1, 1)
                for _ in range(2))
        caches = [torch.full((1, page, 1, 64), NAN_CODE, dtype=torch.uint8, device=DEV).view(E4M3)
                  for _ in range(2)]
        caches = [odd(odd(c, 0, 5), 2, 1) for c in caches]
        if page == 1:
            caches = [odd(c, 1, 7) for c in caches]
        sc = [odd(odd(torch.ones(1, 1, page, device=DEV), 0, 3), 1, 1) for _ in range(2)]
        vb.reshape_and_cache(k, v, *caches, torch.tensor([n - 1], device=DEV), *sc)
        kw, ks = quantise(k.cpu(), E4M3, None)
        assert torch.equal(caches[0][0, n - 1].view(torch.uint8).cpu(), kw[0].view(torch.uint8))
        assert torch.equal(sc[0][0, :, n - 1].cpu(), ks[0])
        table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
        back = [odd(torch.zeros(1, 1, 64, dtype=BF, device=DEV), 0, 3) for _ in range(2)]
        vb.gather_cache(*caches, *back, torch.tensor([0, 1], device=DEV), table,
                        torch.tensor([n - 1], device=DEV), *sc)
        vw, vs = quantise(v.cpu(), E4M3, None)
        want = (vw.float() * vs.unsqueeze(-1)).to(BF)
        assert torch.equal(back[1].cpu(), want)
        if page == 16:
            caches = [c[:, n - 1:].contiguous().expand(1, 16, 1, 64).contiguous() for c in
                      (x.view(torch.uint8) for x in caches)]
            caches = [odd(c.view(E4M3), 2, 1) for c in caches]
            sc = [odd(s[:, :, n - 1:].expand(1, 1, 16).contiguous(), 1, 1) for s in sc]
        q = odd(torch.randn(1, 2, 64, generator=g).to(BF).to(DEV), 0, 1)
        out = odd(torch.zeros(1, 2, 64, dtype=BF, device=DEV), 0, 1)
        meta = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1], [1])]
        assert vb._paged_kernel_takes(q, *caches, out, *meta, table, *sc)
        vb.paged_decode_attention(q, *caches, out, *meta, table, 0.1, *sc)
        assert torch.equal(out.cpu(), want.expand(1, 2, 64))  # (one key: its value)


def test_offsets_past_32_bits():
    """Pages behind the first 4 GiB of a cache, written, attended and read back."""
    hkv, d, page, n = 8, 128, 16, 200
    total = (1 << 32) // (hkv * d * page) + 40
    kc, vc = (torch.zeros(total, page, hkv, d, dtype=torch.uint8, device=DEV).view(E4M3)
              for _ in range(2))
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, hkv, d, generator=g).to(BF) for _ in range(2))
    table = torch.arange(total - 1, total - 14, -1, dtype=torch.int32).view(1, -1)
    t = torch.arange(n)
    slots = table[0, t // page].long() * page + t % page
    vb.reshape_and_cache(k.to(DEV), v.to(DEV), kc, vc, slots.to(DEV))
    kk, kv = torch.empty(n, hkv, d, dtype=BF, device=DEV), torch.empty(n, hkv, d, dtype=BF, device=DEV)
    vb.gather_cache(kc, vc, kk, kv, torch.tensor([0, n], device=DEV), table.to(DEV))
    assert torch.equal(kk.cpu(), k.to(E4M3).to(BF)) and torch.equal(kv.cpu(), v.to(E4M3).to(BF))
    for new in (1, 40):
        q = torch.randn(new, 32, d, generator=g).to(BF)
        out = torch.empty_like(q, device=DEV)
        vb.paged_decode_attention(q.to(DEV), kc, vc, out, torch.tensor([0, new], device=DEV),
                                  torch.tensor([n], device=DEV), table.to(DEV), 0.08)
        small = torch.arange(13).view(1, -1)
        pages = torch.zeros(2, 13 * page, hkv, d)
        pages[0, :n], pages[1, :n] = k.to(E4M3).float(), v.to(E4M3).float()
        pages = pages.view(2, 13, page, hkv, d)
        want, size = attention(q, pages[0], pages[1], torch.tensor([0, new]), torch.tensor([n]),
                               small, None, None, 0.08)
        assert ((out.cpu().double() - want).abs() <= bound(want, size, BF)).all()


def test_other_layouts_take_the_torch_composition():
    """A head dim that the kernels do not have, unaligned scales, fp32 queries: the
    composition's result."""
    args = attention_case([300, 70], [1, 1], 8, 2, 80, 16, BF, E4M3, "slot")
    q, kc, vc, cu, used, table, ks, vs = _dev(args)
    out = torch.empty_like(q)
    assert not vb._paged_kernel_takes(q, kc, vc, out, cu, used, table, ks, vs)
    vb.paged_decode_attention(q, kc, vc, out, cu, used, table, 0.1, ks, vs)
    want, size = attention(*args, 0.1)
    assert ((out.cpu().double() - want).abs() <= bound(want, size, BF)).all()
    args = attention_case([300, 70], [1, 1], 8, 2, 64, 16, BF, E4M3, "slot")
    q, kc, vc, cu, used, table, ks, vs = _dev(args)
    shifted = torch.empty(ks.numel() + 1, device=DEV)[1:].view(ks.shape).copy_(ks)
    assert not vb._paged_kernel_takes(q, kc, vc, torch.empty_like(q), cu, used, table, shifted, vs)
    out = torch.empty_like(q)
    vb.paged_decode_attention(q, kc, vc, out, cu, used, table, 0.1, shifted, vs)
    want, size = attention(*args, 0.1)
    assert ((out.cpu().double() - want).abs() <= bound(want, size, BF)).all()


# ---------------------------------------------------------------------------
# read-back
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [E4M3, E5M2, None])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hkv,d,page", [(8, 128, 16), (2, 64, 24), (4, 256, 16), (3, 96, 7),
                                        (1, 8, 1), (1, 512, 64)])
@pytest.mark.parametrize("mode", MODES)
def test_read_back(fmt, dtype, hkv, d, page, mode):
    if fmt is None and mode != "none":
        mode = "none"  # 16-bit caches have no scales
    g = torch.Generator().manual_seed(page * d)
    lens, first = [70, 0, 1, 33, 129], [5, 0, 0, 40, 17]
    room = [n + f for n, f in zip(lens, first)]
    per = [(n + page - 1) // page for n in room]
    total = sum(per) + 2
    perm = torch.randperm(total, generator=g)
    table = torch.full((5, max(per)), 10 ** 6, dtype=torch.int64)
    at = 0
    for b, m in enumerate(per):
        table[b, :m] = perm[at:at + m]
        at += m
    table[0, 0] -= total  # a page counted from the end
    if fmt is None:
        caches = [torch.randn(total, page, hkv, d, generator=g).to(dtype) for _ in range(2)]
    else:  # every code, NaN and infinities included
        caches = [torch.randint(0, 256, (total, page, hkv, d), generator=g).to(torch.uint8).view(fmt)
                  for _ in range(2)]
    sc = [scales(mode, total, page, hkv, g) for _ in range(2)]
    cu = torch.tensor([2] + [2 + sum(lens[:i + 1]) for i in range(5)], dtype=torch.int32)
    T = int(cu[-1]) + 3
    rows = [torch.full((T, 2 * hkv, d), 7.0, dtype=dtype, device=DEV)[:, :hkv] for _ in range(2)]
    vb.gather_cache(*_dev(caches), *rows, cu.to(DEV), table.to(DEV), torch.tensor(first).to(DEV),
                    *_dev(sc))
    for x, c, s in zip(rows, caches, sc):
        want = torch.full((T, hkv, d), 7.0, dtype=dtype)
        v = c.float()
        if s is not None:
            v = v * (s.transpose(1, 2).unsqueeze(-1) if s.dim() == 3 else s.view(-1, 1))
        for b, n in enumerate(lens):
            t = torch.arange(n) + first[b]
            want[cu[b]:cu[b + 1]] = v[table[b][t // page], t % page].to(dtype)
        assert _same(x.cpu(), want)


def test_read_back_of_what_only_the_device_sees():
    g = torch.Generator().manual_seed(0)
    cache = torch.randn(6, 16, 2, 64, generator=g).to(BF).to(DEV)
    table = torch.tensor([[0, 1, 2], [3, 99, -7]], dtype=torch.int32, device=DEV)

    def run(cu, starts=None):
        x, y = torch.full((2, 80, 2, 64), 7.0, dtype=BF, device=DEV)
        vb.gather_cache(cache, cache, x, y, torch.tensor(cu, device=DEV, dtype=torch.int32), table,
                        None if starts is None else torch.tensor(starts, device=DEV))
        assert _same(x, y)
        return x.float().cpu()

    flat = cache.view(96, 2, 64).float().cpu()
    x = run([0, 30, 70])  # sequence 1: page 3, then two outside the cache
    assert torch.equal(x[:46], torch.cat([flat[:30], flat[48:64]]))
    assert x[46:70].isnan().all() and (x[70:] == 7).all()
    x = run([0, 50, 66])  # past the table's room, and a row of no sequence
    assert torch.equal(x[:48], flat[:48]) and x[48:50].isnan().all()
    assert torch.equal(x[50:66], flat[48:64]) and (x[66:] == 7).all()
    x = run([0, 3, 6], [47, -1])
    assert torch.equal(x[:1], flat[47:48]) and x[1:6].isnan().all() and (x[6:] == 7).all()
    x = run([0, 3, 6], [2 ** 62, 2])
    assert x[:3].isnan().all() and torch.equal(x[3:6], flat[50:53])
    for cu in ([0, 81, 81], [-1, 3, 5], [0, 5, 3]):
        assert run(cu).isnan().all(), cu
    many = torch.arange(0, 81, dtype=torch.int32, device=DEV)  # more sequences than one round
    x, y = torch.full((2, 80, 2, 64), 7.0, dtype=BF, device=DEV)
    vb.gather_cache(cache, cache, x, y, many, (torch.arange(80, device=DEV) % 6).view(80, 1))
    assert torch.equal(x.float().cpu(), flat.view(6, 16, 2, 64)[torch.arange(80) % 6, 0])


def test_read_back_of_no_sequence_and_no_rows():
    cache = torch.ones(2, 16, 2, 64, dtype=BF, device=DEV)
    x = torch.full((4, 2, 64), 7.0, dtype=BF, device=DEV)
    y = x.clone()
    vb.gather_cache(cache, cache, x, y, torch.tensor([0], device=DEV),
                    torch.zeros(0, 3, dtype=torch.int32, device=DEV))
    vb.gather_cache(cache, cache, x, y, torch.tensor([1, 1], device=DEV),
                    torch.zeros(1, 0, dtype=torch.int32, device=DEV))
    vb.gather_cache(cache, cache, x[:0], y[:0], torch.tensor([0, 0], device=DEV),
                    torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    assert (x == 7).all() and (y == 7).all()
    vb.gather_cache(cache, cache, x, y, torch.tensor([1, 3], device=DEV),
                    torch.zeros(1, 0, dtype=torch.int32, device=DEV))
    assert x[1:3].isnan().all() and (x[3:] == 7).all()


# ---------------------------------------------------------------------------
# as they are used
# ---------------------------------------------------------------------------

def _cached(lens, hkv, d, page, fmt, mode, seed, dtype=BF):
    """Rows, a table with room for them, and an empty cache with its scales."""
    g = torch.Generator().manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(sum(per) + 2, generator=g)
    table = torch.zeros(len(lens), max(per), dtype=torch.int32)
    slots, at = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = perm[at:at + per[b]].to(torch.int32)
        at += per[b]
        t = torch.arange(n)
        slots.append(table[b, t // page].long() * page + t % page)
    total = sum(per) + 2
    kv = torch.zeros(2, total, page, hkv, d, dtype=torch.uint8)
    sc = [scales(mode, total, page, hkv, g) for _ in range(2)]
    rows = [torch.randn(sum(lens), hkv, d, generator=g).to(dtype) for _ in range(2)]
    return rows, table, slots, kv, sc, g


@pytest.mark.parametrize("mode", MODES)
def test_written_then_attended_and_read_back(mode):
    """Prompts written in two steps, a decode step and a drafted one over them, and the
    rows read back."""
    lens, hq, hkv, d, page = [700, 33, 129], 8, 2, 128, 16
    rows, table, slots, kv, sc, g = _cached(lens, hkv, d, page, E4M3, mode, 11)
    cache, dsc = kv.to(DEV).view(E4M3), _dev(sc)
    all_slots = torch.cat(slots)
    for part in (slice(0, 400), slice(400, None)):
        vb.reshape_and_cache(rows[0][part].to(DEV), rows[1][part].to(DEV), cache[0], cache[1],
                             all_slots[part].to(DEV), *dsc)
    cpu, csc = cache.cpu(), [None if s is None else s.cpu() for s in dsc]
    used = torch.tensor(lens)
    for news in ([1, 1, 1], [4, 1, 33]):
        q = torch.randn(sum(news), hq, d, generator=g).to(BF)
        cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)))
        args = [q, cpu[0], cpu[1], cu, used, table, *csc]
        _check(args, 0.09)
    cu = torch.tensor([0] + list(used.cumsum(0)))
    back = [torch.empty(sum(lens), hkv, d, dtype=BF, device=DEV) for _ in range(2)]
    vb.gather_cache(cache[0], cache[1], *back, cu.to(DEV), table.to(DEV), None, *dsc)
    for i in range(2):
        v = values(cpu[i], csc[i]).float().view(-1, hkv, d)[all_slots]
        assert torch.equal(back[i].cpu(), v.to(BF))
        # a value lies within half a step of its 8 bits (2^-4 of it, or the smallest
        # step 2^-9 of the scale), then within half a step of bf16; beyond the range of
        # a fixed scale it saturates
        if mode == "slot":
            s = csc[i].transpose(1, 2).reshape(-1, hkv)[all_slots].unsqueeze(-1)
            x = rows[i].float()
            assert ((back[i].cpu().float() - x).abs()
                    <= x.abs() * (2.0 ** -4 + 2.0 ** -7) + s * 2.0 ** -10 * 1.01).all()


def _meta(lens, news, table, slots):
    cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32, device=DEV)
    return SimpleNamespace(num_actual_tokens=sum(news), query_start_loc=cu, max_query_len=max(news),
                           seq_lens=torch.tensor(lens, device=DEV), block_table=table.to(DEV),
                           slot_mapping=slots.to(DEV), use_cascade=False)


@pytest.mark.parametrize("name,fmt", [("fp8", E4M3), ("fp8_e5m2", E5M2)])
def test_a_prompt_and_a_decode_step_through_the_hooked_forward(name, fmt):
    lens, hq, hkv, d, page = [701, 34, 130], 8, 2, 128, 16
    rows, table, slots, kv, _, g = _cached(lens, hkv, d, page, fmt, "none", 12)
    cache = kv.to(DEV)  # bytes, as vLLM allocates it
    layer = SimpleNamespace(_k_scale=torch.tensor(0.02, device=DEV),
                            _v_scale=torch.tensor(0.013, device=DEV))
    impl = SimpleNamespace(attn_type="decoder", kv_sharing_target_layer_name=None,
                           kv_cache_dtype=name, dcp_world_size=1, scale=1 / math.sqrt(d))
    fwd = vb.make_forward(vb.ATTENTION_CONFIGS["flashprefill_llama"])
    first = [n - 1 for n in lens]
    starts = [sum(lens[:b]) for b in range(3)]
    pre = torch.cat([torch.arange(n) + s for n, s in zip(first, starts)])
    last = torch.tensor([s + n for n, s in zip(first, starts)])
    all_slots = torch.cat(slots)
    q = torch.randn(sum(lens), hq, d, generator=g).to(BF).to(DEV)
    k, v = _dev(rows)
    out = torch.empty_like(q)
    sub = [t[pre.to(DEV)] for t in (q, k, v, out)]
    fwd(impl, layer, *sub[:3], cache, _meta(first, first, table, all_slots[pre]), output=sub[3])
    want = torch.empty_like(sub[3])
    cu = torch.tensor([0] + list(torch.tensor(first).cumsum(0)), dtype=torch.int32, device=DEV)
    vb.flash_prefill_varlen_func(*sub[:3], want, cu, max(first), 0.18, 128, 2, 4, 2)
    assert torch.equal(sub[3], want)  # prefill reads the step's own rows
    sub = [t[last.to(DEV)] for t in (q, k, v, out)]
    fwd(impl, layer, *sub[:3], cache, _meta(lens, [1, 1, 1], table, all_slots[last]), output=sub[3])
    cpu = cache.cpu().view(fmt)
    sc = [torch.tensor(0.02), torch.tensor(0.013)]
    for i in range(2):
        codes, _ = quantise(rows[i], fmt, sc[i].view(1, 1))
        assert _same(cpu[i].view(-1, hkv, d)[all_slots], codes)
    want, size = attention(sub[0].cpu(), cpu[0], cpu[1], torch.arange(4), torch.tensor(lens), table,
                           *sc, 1 / math.sqrt(d))
    assert ((sub[3].cpu().double() - want).abs() <= bound(want, size, BF)).all()


def test_v0_prefix_cached_prefill_and_decode_rows():
    lens, hq, hkv, d, page = [600, 90, 300, 44], 8, 2, 128, 16
    rows, table, slots, kv, _, g = _cached(lens, hkv, d, page, E4M3, "none", 13)
    cache = kv.to(DEV)
    layer = SimpleNamespace(_k_scale=torch.tensor([0.02], device=DEV), _v_scale=None)
    old = [n - m for n, m in zip(lens, (64, 50, 1, 1))]
    starts = [sum(lens[:b]) for b in range(4)]
    had = torch.cat([torch.arange(n) + s for n, s in zip(old, starts)])
    new = torch.cat([torch.arange(o, n) + s for o, n, s in zip(old, lens, starts)])
    all_slots = torch.cat(slots)
    vb.reshape_and_cache(rows[0][had].to(DEV), rows[1][had].to(DEV), cache[0].view(E4M3),
                         cache[1].view(E4M3), all_slots[had].to(DEV), layer._k_scale)
    q = torch.randn(116, hq, d, generator=g).to(BF)
    cu = torch.tensor([0, 64, 114], dtype=torch.int32, device=DEV)
    used = torch.tensor(lens, device=DEV)
    dt = table.to(DEV)
    pm = SimpleNamespace(seq_start_loc=cu, max_prefill_seq_len=64, query_start_loc=cu,
                         seq_lens_tensor=used[:2], block_tables=dt[:2])
    dm = SimpleNamespace(seq_lens_tensor=used[2:], max_decode_query_len=1, query_start_loc=None,
                         block_tables=dt[2:])
    meta = SimpleNamespace(num_prefill_tokens=114, num_decode_tokens=2,
                           slot_mapping=all_slots[new].to(DEV), prefill_metadata=pm,
                           decode_metadata=dm)
    impl = SimpleNamespace(attn_type="decoder", kv_cache_dtype="fp8_e4m3", scale=0.08)
    fwd = vb.make_forward_v0(vb.ATTENTION_CONFIGS["flashprefill_qwen2"])
    out = torch.empty(116, hq, d, dtype=BF, device=DEV)
    fwd(impl, layer, q.to(DEV), rows[0][new].to(DEV), rows[1][new].to(DEV), cache, meta, output=out)
    cpu = cache.cpu().view(E4M3)
    want, size = attention(q, cpu[0], cpu[1], torch.tensor([0, 64, 114, 115, 116]),
                           torch.tensor(lens), table, torch.tensor(0.02), None, 0.08)
    assert ((out.cpu().double() - want).abs() <= bound(want, size, BF)).all()


def test_capture_and_replay():
    """One graph of write, attention and read-back, replayed over changing rows, lengths
    and slots, with the same calls made eagerly in between."""
    lens, hq, hkv, d, page = [900, 70], 8, 2, 128, 16
    rows, table, slots, kv, sc, g = _cached(lens, hkv, d, page, E4M3, "slot", 14)
    cache, dsc = kv.to(DEV).view(E4M3), _dev(sc)
    vb.reshape_and_cache(rows[0].to(DEV), rows[1].to(DEV), cache[0], cache[1],
                         torch.cat(slots).to(DEV), *dsc)
    dt, cu = table.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    used = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(2, h, d, generator=g).to(BF).to(DEV) for h in (hq, hkv, hkv))
    at = torch.stack([s[-1] for s in slots]).to(DEV)
    out, bk, bv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)

    def step(cache, dsc, out, bk, bv):
        vb.reshape_and_cache(k, v, cache[0], cache[1], at, *dsc)
        vb.paged_decode_attention(q, cache[0], cache[1], out, cu, used, dt, 0.1, *dsc)
        vb.gather_cache(cache[0], cache[1], bk, bv, cu, dt, used - 1, *dsc)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(cache, dsc, out, bk, bv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, dsc, out, bk, bv)
    for n in (900, 300, 897, 1):
        used[0] = n
        at[0] = slots[0][n - 1]
        k.normal_()
        q.normal_()
        mine = (cache.view(torch.uint8).clone().view(E4M3), [x.clone() for x in dsc],
                *(torch.zeros_like(x) for x in (out, bk, bv)))
        step(*mine)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mine[2]) and torch.equal(bk, mine[3]) and torch.equal(bv, mine[4])
        assert torch.equal(cache.view(torch.uint8), mine[0].view(torch.uint8))
        assert torch.equal(dsc[0], mine[1][0]) and torch.equal(dsc[1], mine[1][1])


def test_another_stream_and_threads():
    """Calls on a stream of their own and from two threads on one give the same bits."""
    cases = [_dev(attention_case([3000 + 500 * i, 700], [1, 1], 8, 2, 128, 16, BF, E4M3, "slot",
                                 seed=60 + i)) for i in range(2)]

    def call(c):
        out = torch.empty_like(c[0])
        vb.paged_decode_attention(*c[:3], out, *c[3:6], 0.09, *c[6:])
        return out

    want = [call(c) for c in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        aside = [call(c) for c in cases]
    got = [[], []]

    def work(i):
        for _ in range(100):
            got[i].append(call(cases[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(aside[i], want[i])
        assert len(got[i]) == 100 and all(torch.equal(o, want[i]) for o in got[i])


def test_a_write_counts_as_an_in_place_change():
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    other = torch.zeros_like(cache)
    sc = [torch.ones(2, 2, 16, device=DEV) for _ in range(2)]
    x = torch.ones(3, 2, 64, dtype=BF, device=DEV)
    before = [t._version for t in (cache, other, *sc)]
    vb.reshape_and_cache(x, x, cache, other, torch.arange(3, device=DEV), *sc)
    assert all(t._version > v for t, v in zip((cache, other, *sc), before))
    w = torch.ones_like(x, requires_grad=True)
    y = (w * x).sum()  # saves x
    vb.gather_cache(cache, other, x, x.clone(), torch.tensor([0, 3], device=DEV),
                    torch.zeros(1, 1, dtype=torch.int32, device=DEV), None, *sc)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_refusals():
    cache = torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    x = torch.ones(3, 2, 64, dtype=BF, device=DEV)
    slots = torch.arange(3, device=DEV)
    sc = torch.ones(4, 2, 16, device=DEV)
    with pytest.raises(RuntimeError, match="one memory"):
        vb.reshape_and_cache(x, x, cache[0], cache[1], slots, sc, sc[:1].expand(4, 2, 16))
    with pytest.raises(RuntimeError, match="one memory"):
        vb.reshape_and_cache(x, x, cache[0], cache[1, :1].expand(4, 16, 2, 64), slots)
    with pytest.raises(ValueError, match="one GPU"):
        vb.reshape_and_cache(x, x.cpu(), cache[0], cache[1], slots)
    for kc, vc, ks, vs in ((cache[0], cache[0], sc, sc.clone()), (cache[0], cache[1], sc, sc)):
        with pytest.raises(ValueError, match="of their own"):
            vb.reshape_and_cache(x, x, kc, vc, slots, ks, vs)
    with pytest.raises(RuntimeError, match="gradient"):
        vb.reshape_and_cache(x, x, cache[0], cache[1], slots, sc.clone().requires_grad_(), sc)
    with pytest.raises(ValueError, match="device"):
        vb.reshape_and_cache(x, x, cache[0], cache[1], slots, sc.cpu(), sc)
    with torch.inference_mode():
        frozen = torch.zeros(4, 16, 2, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    with pytest.raises(RuntimeError, match="inference"):
        vb.reshape_and_cache(x, x, cache[0], frozen, slots)
    with torch.inference_mode():
        vb.reshape_and_cache(x, x, frozen, frozen.clone(), slots)
    odd = torch.zeros(4 * 16 * 2 * 64 + 4, dtype=torch.uint8, device=DEV)[4:].view(4, 16, 2, 64)
    with pytest.raises(ValueError, match="aligned"):
        vb.reshape_and_cache(x, x, odd.view(E4M3), cache[1], slots)
    cu, table = torch.tensor([0, 3], device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="one memory"):
        vb.gather_cache(cache[0], cache[1], x, x[:1].expand(3, 2, 64), cu, table)
    with pytest.raises(ValueError, match="of their own"):
        vb.gather_cache(cache[0], cache[1], x, x, cu, table)
    y = torch.ones_like(x, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        vb.gather_cache(cache[0], cache[1], x, y, cu, table)
    assert TOP[E4M3] == 448.0

"""GPU tests of the 4-bit KV cache: write, read-back, attention with few and many rows,
each against 64 bits, and a run of them together, captured and replayed."""

import math
from types import SimpleNamespace

import pytest
import torch

from flashprefill_amd import int4_cache as i4
from flashprefill_amd import vllm_backend as vb
from tests import _int4 as I

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _cuda(x):
    return x.cuda() if torch.is_tensor(x) else x


def _write(x, y, slots, nb, page, scale=None, v_scale=None):
    """Written caches, on the CPU: k codes, v codes, k words, v words."""
    n, hkv, d = x.shape
    caches = [torch.full((nb, page, hkv, d // 2), 0xa5, dtype=torch.uint8, device="cuda")
              for _ in range(2)]
    words = [torch.full((nb, hkv, page, d // 32), 0x1234, dtype=torch.int16, device="cuda")
             for _ in range(2)]
    i4.reshape_and_cache_int4(_cuda(x), _cuda(y), *caches, *words, _cuda(slots), _cuda(scale),
                              _cuda(v_scale))
    return [t.cpu() for t in caches + words]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("mode", I.MODES)
@pytest.mark.parametrize("n,hkv,d,page", [(1, 1, 64, 16), (77, 3, 128, 16), (300, 8, 128, 24),
                                          (41, 5, 256, 1), (130, 2, 64, 7)])
def test_write(n, hkv, d, page, dtype, mode):
    # every code and word is the composition's, which is the rule's in 64 bits (a CPU test)
    g = torch.Generator().manual_seed(n)
    x, y = I.rows(n, hkv, d, dtype, n), I.rows(n, hkv, d, dtype, n + 1)
    ks, vs = I.scales(mode, hkv, g), I.scales(mode, hkv, g)
    nb = n // page + 3
    slots = torch.randperm(nb * page, generator=g)[:n]
    slots[::5] = -1
    slots[3::11] = nb * page + 2
    got = _write(x, y, slots, nb, page, ks, vs)
    put = (slots >= 0) & (slots < nb * page)
    at = slots[put]
    left = torch.ones(nb * page, dtype=torch.bool)
    left[at] = False
    for c, w, r, s in ((got[0], got[2], x, ks), (got[1], got[3], y, vs)):
        codes, words = i4.quantise_int4(r[put], s)
        assert torch.equal(c.view(-1, hkv, d // 2)[at], codes)
        flat = w.transpose(1, 2).reshape(-1, hkv, d // 32)
        assert torch.equal(flat[at], words)
        assert (c.view(-1, hkv, d // 2)[left] == 0xa5).all() and (flat[left] == 0x1234).all()


@pytest.mark.parametrize("scale", [1e-30, -0.37, 3e20])
def test_write_with_scales_out_of_the_ordinary(scale):
    x, s = I.rows(50, 2, 128, BF, 3), torch.tensor([scale])
    if abs(scale) != 0.37:
        x = (x.float() * scale).to(BF)
    got = _write(x, x, torch.arange(50), 4, 16, s, s)
    codes, words = i4.quantise_int4(x, s)
    assert torch.equal(got[0].view(-1, 2, 64)[:50], codes)
    assert torch.equal(got[3].transpose(1, 2).reshape(-1, 2, 4)[:50], words)


def test_views_of_one_projection_and_of_one_page_tensor():
    qkv = I.rows(60, 10, 128, BF, 5).cuda()
    key, value = qkv[:, 6:8], qkv[:, 8:]
    pages = torch.zeros(2, 6, 16, 2, i4.int4_row_bytes(128), dtype=torch.uint8, device="cuda")
    (kc, kg), (vc, vg) = (i4.int4_cache_views(p) for p in pages)
    slots = torch.randperm(96, device="cuda")[:60]
    i4.reshape_and_cache_int4(key, value, kc, vc, kg, vg, slots)
    for x, c, w in ((key, kc, kg), (value, vc, vg)):
        codes, words = i4.quantise_int4(x)
        assert torch.equal(c[slots // 16, slots % 16], codes)
        assert torch.equal(w[slots // 16, :, slots % 16], words)
    assert int((pages != 0).sum()) <= 2 * 60 * 2 * 72
    q = torch.randn(2, 4, 128, device="cuda", dtype=BF)
    out, want = torch.empty_like(q), torch.empty_like(q)
    args = (torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"),
            torch.tensor([33, 96], dtype=torch.int32, device="cuda"),
            torch.arange(6, dtype=torch.int32, device="cuda").repeat(2, 1), 0.1)
    # (slots that nothing was written to hold zeros; groups of NaN came from the rows)
    kg[kg == I.NAN_WORD] = 64
    vg[vg == I.NAN_WORD] = 64
    i4.paged_decode_attention_int4(q, kc, vc, kg, vg, out, *args)
    i4.paged_attention_int4_reference(q, kc, vc, kg, vg, want, *args)
    assert torch.allclose(out.float(), want.float(), rtol=2 ** -6, atol=1e-2)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("mode", I.MODES)
@pytest.mark.parametrize("hkv,d,page,from_first", [(3, 128, 16, True), (8, 64, 7, False),
                                                   (1, 256, 64, False), (5, 128, 1, True)])
def test_read_back(hkv, d, page, from_first, dtype, mode):
    g = torch.Generator().manual_seed(d + page)
    lens = [0, 1, 40, 129, 3]
    starts = [0] * 5 if from_first else [0, 5, 17, 0, page]
    per = [(n + s + page - 1) // page + 1 for n, s in zip(lens, starts)]
    total = sum(per)
    perm = torch.randperm(total, generator=g)
    table = torch.full((5, max(per)), total + 5, dtype=torch.int64)
    at = 0
    for b, m in enumerate(per):
        table[b, :m] = perm[at:at + m]
        at += m
    table[3, 0] -= total  # (from the end)
    cu = torch.tensor([2] + (2 + torch.tensor(lens).cumsum(0)).tolist(), dtype=torch.int32)
    n = int(cu[-1]) + 4
    (kc, kg), (vc, vg) = (I.random_cache(total, page, hkv, d, g) for _ in range(2))
    ks, vs = I.scales(mode, hkv, g), I.scales(mode, hkv, g)
    out = [torch.full((n, hkv, d), 7.0, dtype=dtype) for _ in range(4)]
    first = None if from_first else torch.tensor(starts)
    got = [t.cuda() for t in out[:2]]
    i4.gather_cache_int4(*map(_cuda, (kc, vc, kg, vg)), *got, cu.cuda(), table.cuda(), _cuda(first),
                         _cuda(ks), _cuda(vs))
    i4.gather_cache_int4_reference(kc, vc, kg, vg, *out[2:], cu, table, first, ks, vs)
    for a, b in zip(got, out[2:]):
        assert torch.equal(a.cpu(), b)
        assert (b[:2] == 7).all() and (b[-4:] == 7).all()
    for b in range(5):
        for i in range(lens[b]):
            pos = starts[b] + i
            pg, o = int(table[b, pos // page]), pos % page
            want = I.values(kc[pg, o], kg[pg, :, o], ks).float().to(dtype)
            assert torch.equal(got[0][int(cu[b]) + i].cpu(), want)


def test_read_back_of_what_does_not_fit():
    g = torch.Generator().manual_seed(0)
    kc, kg = (t.cuda() for t in I.random_cache(4, 16, 2, 64, g))
    table = torch.tensor([[0, 9], [1, -5], [2, 3]], dtype=torch.int32, device="cuda")
    key, value = (torch.ones(60, 2, 64, dtype=BF, device="cuda") for _ in range(2))

    def call(cu, starts=None):
        key.fill_(1.0)
        i4.gather_cache_int4(kc, kc, kg, kg, key, value,
                             torch.tensor(cu, dtype=torch.int32, device="cuda"), table,
                             None if starts is None else torch.tensor(starts, device="cuda"))
        return key.isnan().all(-1).all(-1).cpu()

    nan = call([0, 20, 40, 58])
    want = torch.zeros(60, dtype=torch.bool)
    want[16:20] = want[36:40] = True
    assert torch.equal(nan, want) and (key[58:] == 1).all()
    nan = call([0, 2, 4, 6], [32, -1, 31])  # past the room, before the first, one past the room
    assert nan[:6].tolist() == [True, True, True, True, False, True]
    assert call([0, 20, 10, 30]).all() and call([0, 20, 40, 61]).all()


FEW = [([1], [1], 4, 4, 64, 16), ([0, 5, 333], [1, 1, 1], 8, 2, 128, 16),
       ([1, 15, 16, 17, 31, 33, 127, 129], [1] * 8, 8, 1, 128, 16),
       ([700, 2, 1300], [2, 1, 3], 6, 3, 64, 24), ([257, 0, 64], [4, 2, 1], 4, 4, 256, 32),
       ([2100, 90], [1, 1], 28, 4, 128, 64), ([530], [1], 40, 2, 64, 1),
       ([65, 1000], [5, 1], 12, 12, 64, 16), ([2500], [3], 5, 1, 256, 5)]
MANY = [([40], [40], 4, 1, 64, 16), ([700, 129, 64], [130, 129, 33], 8, 2, 128, 16),
        ([1, 300], [1, 300], 32, 8, 128, 24), ([2300], [500], 4, 4, 64, 64),
        ([1500, 40], [256, 40], 4, 1, 256, 16), ([5, 0, 90], [64, 40, 64], 4, 2, 128, 1),
        ([900, 700], [290, 300], 8, 1, 64, 16), ([1000, 530], [530, 530], 4, 1, 128, 24),
        ([2100], [520], 8, 2, 128, 16), ([600, 0, 7], [600, 300, 300], 16, 2, 64, 1)]


def _attend(args, dtype, scale, spread=False):
    """The output on the CPU. spread: queries and outputs with strides of their own."""
    q = args[0].cuda()
    out = torch.full_like(q, 5.0)
    if spread:
        q = torch.cat([q, q], -1)[:, :, :q.shape[-1]]
        out = torch.full((q.shape[0] + 2, 3 * q.shape[1], q.shape[2]), 5.0, dtype=dtype,
                         device="cuda")[:, ::3]
    i4.paged_decode_attention_int4(q, *map(_cuda, args[1:5]), out, *map(_cuda, args[5:8]), scale,
                                   *map(_cuda, args[8:]))
    if spread:
        assert (out[-2:] == 5).all()
    return out[:q.shape[0]].cpu()


@pytest.mark.parametrize("dtype,mode,index", [(BF, "none", torch.int32), (FP, "head", torch.int64),
                                              (BF, "tensor", torch.int64)])
@pytest.mark.parametrize("case", FEW + MANY, ids=str)
def test_attention(case, dtype, mode, index):
    lens, news, hq, hkv, d, page = case
    args = I.attention_case(lens, news, hq, hkv, d, page, dtype, mode, seed=sum(lens), index=index)
    got = _attend(args, dtype, 1 / math.sqrt(d), spread=index == torch.int64)
    want, size, most = I.attention(*args, 1 / math.sqrt(d))
    cu = args[5].tolist()
    for b, n in enumerate(lens):
        for i in range(news[b]):
            o, r = got[cu[b] + i].double(), cu[b] + i
            if n == 0:
                assert (o == 0).all()
            elif n - news[b] + i < 0:
                assert o.isnan().all()  # a row with no cached token to attend to
            else:
                assert ((o - want[r]).abs() <= bound(want[r], size[r], most, dtype)).all(), \
                    (b, i, float((o - want[r]).abs().max()))


bound = I.bound


@pytest.mark.parametrize("news", [[1, 1], [200, 150]])
def test_negative_and_zero_scales(news):
    for ks, scale in ((-0.5, 0.1), (0.0, 0.1), (0.7, -0.2)):
        args = I.attention_case([300, 170], news, 4, 2, 128, 16, BF, "tensor", seed=9)
        args[8] = torch.tensor([ks])
        got = _attend(args, BF, scale)
        want, size, most = I.attention(*args, scale)
        assert ((got.double() - want).abs() <= bound(want, size, most, BF)).all()


@pytest.mark.parametrize("news", [[1, 1], [200, 150]])
@pytest.mark.parametrize("power", [-120, -60, 100])
def test_bf16_queries_of_any_magnitude(power, news):
    # their fp16 forms carry a power of two of the row: scores are the same ones
    args = I.attention_case([300, 170], news, 4, 2, 128, 16, BF, "none", seed=4)
    q = args[0].clone()
    args[0] = (q.double() * 2.0 ** power).to(BF)
    scale = 2.0 ** -power / 16
    got = _attend(args, BF, scale) if scale < 2.0 ** 127 else None
    want, size, most = I.attention(q, *args[1:], 1 / 16)
    assert ((got.double() - want).abs() <= bound(want, size, most, BF)).all()


@pytest.mark.parametrize("d,news", [(64, [1, 1, 2]), (128, [3, 1, 1]), (256, [1, 1, 1]),
                                    (64, [60, 70, 80]), (128, [60, 70, 80]), (256, [150, 100, 140]),
                                    (64, [600, 400, 300]), (128, [700, 400, 290])])
def test_groups_of_nan_and_steps_of_zero(d, news):
    # a group of NaN reaches the rows that see its key only: in V its dims, in K all of them
    lens = [700, 400, 300]
    args = I.attention_case(lens, news, 16 if news[0] > 500 else 4, 2, d, 16, BF, "none", seed=2)
    kg, vg, table = args[3], args[4], args[7]
    hit = [(0, lens[0] - 1, vg), (1, lens[1] - news[1], kg), (2, lens[2] - news[2] // 2 - 1, vg)]
    for b, key, words in hit:
        words[int(table[b, key // 16]), 1, key % 16, 1] = I.NAN_WORD
    kg[table[2, 3], 0] = 64  # a page of zeros
    got = _attend(args, BF, 0.1)
    want, size, most = I.attention(*args, 0.1)
    group = torch.arange(d) // 32 == 1
    for b, key, words in hit:
        for i in range(news[b]):
            o = got[int(args[5][b]) + i]
            sees = lens[b] - news[b] + i >= key
            bad = o.isnan()
            expect = torch.zeros_like(bad)
            if sees:
                expect[bad.shape[0] // 2:] = group if words is vg else True
            assert torch.equal(bad, expect), (b, i)
    ok = ~(got.isnan())
    far = (got.double() - want).abs() <= bound(want, size, most, BF)
    assert far[ok].all()


@pytest.mark.parametrize("news", [[1, 1, 1], [100, 90, 80]])
def test_pages_and_lengths_that_do_not_fit(news):
    lens = [200, 150, 130]
    args = I.attention_case(lens, news, 4, 2, 128, 16, BF, "none", seed=1, width=14)
    want = _attend(args, BF, 0.1)
    total = args[1].shape[0]
    args[7][0, 0] -= total            # from the end: the same page
    args[7][1, 2] = total             # outside: every row that attends to it
    args[6][2] = 14 * 16 + 1          # more than the table has room for
    got = _attend(args, BF, 0.1)
    n = news[0]
    assert torch.equal(got[:n], want[:n])
    assert got[n:].isnan().all()
    args[5][1] = sum(news) + 1        # offsets outside the rows: all of them
    assert _attend(args, BF, 0.1).isnan().all()


def test_a_cache_past_32_bits():
    # pages beyond 2^32 bytes of codes
    page, hkv, d = 64, 8, 128
    nb = (1 << 32) // (page * hkv * d // 2) + 40
    codes = [torch.zeros(nb, page, hkv, d // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    words = [torch.full((nb, hkv, page, d // 32), 64, dtype=torch.int16, device="cuda")
             for _ in range(2)]
    x, y = I.rows(200, hkv, d, FP, 1), I.rows(200, hkv, d, FP, 2)
    x, y = (torch.nan_to_num(t, 0, 1, -1).clamp(-50, 50) for t in (x, y))
    pages = torch.tensor([nb - 1, 3, nb - 20, nb - 7], dtype=torch.int32)
    slots = (pages.long().view(-1, 1) * page + torch.arange(page)).view(-1)[:200]
    i4.reshape_and_cache_int4(x.cuda(), y.cuda(), *codes, *words, slots.cuda())
    key, value = (torch.empty(200, hkv, d, dtype=FP, device="cuda") for _ in range(2))
    cu, table = torch.tensor([0, 200], dtype=torch.int32).cuda(), pages.view(1, -1).cuda()
    i4.gather_cache_int4(*codes, *words, key, value, cu, table)
    for r, got in ((x, key), (y, value)):
        assert torch.equal(got.cpu(), i4.int4_values(*i4.quantise_int4(r)).to(FP))
    for rows in (1, 100):
        q = torch.randn(rows, 16, d, dtype=FP, device="cuda")
        out, want = torch.empty_like(q), torch.empty_like(q)
        args = (torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                torch.tensor([200], dtype=torch.int32, device="cuda"), table, 0.05)
        i4.paged_decode_attention_int4(q, *codes, *words, out, *args)
        i4.paged_attention_int4_reference(q, *codes, *words, want, *args)
        # two roundings to fp16 and one of P, of values below 8 on average
        assert (out.float() - want.float()).abs().max() <= 3 * 2.0 ** -11 * float(value.abs().max())


def _step(st):
    i4.reshape_and_cache_int4(st.key, st.value, st.kc, st.vc, st.kg, st.vg, st.slots, st.ks, st.vs)
    i4.paged_decode_attention_int4(st.q, st.kc, st.vc, st.kg, st.vg, st.out, st.cu, st.used,
                                   st.table, 0.09, st.ks, st.vs)
    i4.gather_cache_int4(st.kc, st.vc, st.kg, st.vg, st.back_k, st.back_v, st.cu_back, st.table,
                         None, st.ks, st.vs)


def _step_state(news, width=80, seed=0):
    g = torch.Generator().manual_seed(seed)
    lens, hq, hkv, d, page = [1200, 300], 8, 2, 128, 16
    args = [_cuda(t) for t in I.attention_case(lens, news, hq, hkv, d, page, BF, "head", seed=seed,
                                               width=width)]
    st = SimpleNamespace(q=args[0], kc=args[1], vc=args[2], kg=args[3], vg=args[4], cu=args[5],
                         used=args[6], table=args[7], ks=args[8], vs=args[9])
    st.table.clamp_(min=0)
    n = sum(news)
    st.key, st.value = (torch.randn(n, hkv, d, generator=g).to(BF).cuda() for _ in range(2))
    st.slots = torch.cat([st.table[b].long().repeat_interleave(page)[m - k:m] * page +
                          torch.arange(m - k, m, device="cuda") % page
                          for b, (m, k) in enumerate(zip(lens, news))])
    st.out = torch.empty_like(st.q)
    st.back_k, st.back_v = (torch.zeros(1500, hkv, d, dtype=BF, device="cuda") for _ in range(2))
    st.cu_back = torch.tensor([0, 1200, 1500], dtype=torch.int32, device="cuda")
    return st


@pytest.mark.parametrize("news", [[1, 1], [3, 1], [300, 200]])
def test_a_step_captured_and_replayed(news):
    st = _step_state(news)
    _step(st)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (another stream than the tensors' own)
        _step(st)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(st)
    for seed in range(3):
        new = _step_state(news, seed=seed + 1)
        for name in ("q", "key", "value", "kc", "vc", "kg", "vg", "used", "table", "slots"):
            getattr(st, name).copy_(getattr(new, name))
        st.ks.copy_(new.ks)
        st.vs.copy_(new.vs)
        graph.replay()
        torch.cuda.synchronize()
        _step(new)
        for name in ("out", "back_k", "back_v", "kc", "kg", "vg"):
            assert torch.equal(getattr(st, name), getattr(new, name)), name
        key, value = (t.cpu() for t in (new.key, new.value))
        rows = i4.int4_values(*i4.quantise_int4(key, new.ks.cpu()), new.ks.cpu()).to(BF)
        assert torch.equal(st.back_k[1200 - news[0]:1200].cpu(), rows[:news[0]])


def test_calls_that_the_kernels_do_not_take_are_composed():
    args = I.attention_case([60], [2], 4, 2, 64, 16, torch.float32, "none")
    want, _, _ = I.attention(*args, 0.1)
    got = _attend(args, torch.float32, 0.1)
    assert (got.double() - want).abs().max() < 1e-4
    with torch.enable_grad():
        q = args[0].to(BF).cuda().requires_grad_()
        out = torch.zeros(2, 4, 64, device="cuda", dtype=BF)
        i4.paged_decode_attention_int4(q, *map(_cuda, args[1:5]), out, *map(_cuda, args[5:8]), 0.1)
        out.float().sum().backward()
        assert q.grad is not None and q.grad.isfinite().all()


class Layer:
    pass


@pytest.mark.parametrize("version", [0, 1])
def test_hooked_forwards_over_4_bit_caches(version):
    g = torch.Generator().manual_seed(1)
    hq, hkv, d, page = 8, 2, 128, 16
    make = vb.make_forward if version else vb.make_forward_v0
    forward = make(vb.ATTENTION_CONFIGS["flashprefill_llama"])
    impl = SimpleNamespace(kv_cache_dtype="int4", scale=0.09)
    layer = Layer()
    layer._k_scale = torch.tensor(0.5, device="cuda")
    kv = torch.zeros(2, 20, page, hkv, i4.int4_row_bytes(d), dtype=torch.uint8, device="cuda")
    prompt = 130
    q, k, v = (torch.randn(prompt + 1, h, d, generator=g).to(BF).cuda() for h in (hq, hkv, hkv))
    table = torch.randperm(20, generator=g)[:10].to(torch.int32).view(1, 10).cuda()
    pos = torch.arange(prompt + 1, device="cuda")
    slots = table[0, pos // page].long() * page + pos % page

    def meta(n, used, slot):
        if version:
            return SimpleNamespace(num_actual_tokens=n, slot_mapping=slot, max_query_len=n,
                                   query_start_loc=torch.tensor([0, n], dtype=torch.int32,
                                                                device="cuda"),
                                   seq_lens=torch.tensor([used], dtype=torch.int32, device="cuda"),
                                   block_table=table)
        part = SimpleNamespace(seq_start_loc=torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                               max_prefill_seq_len=n, block_tables=None if n > 1 else table,
                               seq_lens_tensor=torch.tensor([used], dtype=torch.int32,
                                                            device="cuda"),
                               max_decode_query_len=1)
        return SimpleNamespace(slot_mapping=slot, num_prefill_tokens=n if n > 1 else 0,
                               num_decode_tokens=0 if n > 1 else 1,
                               prefill_metadata=part if n > 1 else None,
                               decode_metadata=None if n > 1 else part)

    out = torch.empty(prompt, hq, d, dtype=BF, device="cuda")
    forward(impl, layer, q[:prompt], k[:prompt], v[:prompt], kv, meta(prompt, prompt, slots[:prompt]),
            output=out)
    one = torch.empty(1, hq, d, dtype=BF, device="cuda")
    forward(impl, layer, q[prompt:], k[prompt:], v[prompt:], kv, meta(1, prompt + 1, slots[prompt:]),
            output=one)
    ks = torch.tensor([0.5])
    hk, hv = (i4.int4_values(*i4.quantise_int4(x.cpu(), s), s).double()
              .repeat_interleave(hq // hkv, 1) for x, s in ((k, ks), (v, None)))
    s = torch.einsum("hd,khd->hk", q[prompt].cpu().double(), hk) * 0.09
    want = torch.einsum("hk,khd->hd", torch.softmax(s, -1), hv)
    assert (one[0].cpu().double() - want).abs().max() <= 2.0 ** -8 * float(want.abs().max()) + 1e-4

"""CPU tests of the 4-bit KV cache: the format's rule, the torch compositions, what the entry
points refuse, the hooked forwards' dispatch, and the registers of the kernels."""

import ctypes
import math
import re
from types import SimpleNamespace

import pytest
import torch

from flashprefill_amd import _lib
from flashprefill_amd import int4_cache as i4
from flashprefill_amd import vllm_backend as vb
from tests import _int4 as I
from tests.test_codegen import HIPCC, _assembly, _registers
from tests.test_codegen import pytestmark as needs_hipcc

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("mode", I.MODES)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_the_rule_of_the_format(d, dtype, mode):
    x = I.rows(300, 3, d, dtype, d)
    g = torch.Generator().manual_seed(d)
    scale = I.scales(mode, 3, g)
    codes, words = i4.quantise_int4(x, scale)
    got = I.values(codes, words, scale)
    assert torch.equal(i4.int4_values(codes, words).double().nan_to_num(7e9),
                       I.values(codes, words, None).nan_to_num(7e9))
    want, step = I.held(x, scale)
    assert torch.equal(got.isnan(), want.isnan())
    # fp32's x (1 / t) may lie on the other side of a tie: by a step, of a few in a million
    off = (got != want) & ~want.isnan()
    t = torch.ones(1, dtype=torch.float64) if scale is None else scale.double().view(1, -1, 1)
    assert off.float().mean() <= (0 if scale is None else 1e-4)
    assert ((got - want).abs()[off] <= 1.001 * (step * t.abs()).expand_as(got)[off]).all()
    # an element within 16384 is off by half a step; by at most 1.5 steps where the step of 4
    # significant bits, rounded down by up to a 17th, leaves the group's largest ones past
    # code 15 (15 x 17 / 16 steps from the smallest, whose own rounding adds half of one)
    fine = x.isfinite() & (x.double() / t).abs().le(16384) & want.isfinite() & (step >= 2.0 ** -14)
    gap = ((want / t - x.double() / t).abs() / step)[fine]
    assert gap.max() <= 1.5001 and (gap > 0.5001).float().mean() < 0.05
    zero = fine & (x == 0)
    assert (want[zero].abs() <= 0.0).float().mean() > 0.5 or not zero.any()


def test_what_groups_hold():
    def held(*x):
        row = torch.tensor(list(x) + [0.0] * (64 - len(x))).view(1, 1, 64)
        return i4.int4_values(*i4.quantise_int4(row))[0, 0]
    assert (held() == 0).all() and (held(-0.0) == 0).all()
    assert held(*[3.0] * 32)[:32].sub(3.0).abs().max() <= 3.0 / 56 * 0.54
    assert held(math.nan)[:32].isnan().all() and (held(math.nan)[32:] == 0).all()
    assert abs(held(math.inf)[0] - 16384) <= 0.5 * 1152 and held(-math.inf)[0] <= -15800
    assert (held(1e-7) == 0).all()  # below 2^-18 of a step
    assert torch.equal(held(*[float(i - 7) for i in range(16)])[:16], torch.arange(16.0) - 7)


@pytest.mark.parametrize("mode", I.MODES)
def test_the_composition_of_attention(mode):
    args = I.attention_case([40, 7, 0], [1, 3, 1], 4, 2, 64, 4, torch.float32, mode)
    out = torch.empty(5, 4, 64)
    i4.paged_decode_attention_int4(*args[:5], out, *args[5:8], 0.25, *args[8:])
    want, size, _ = I.attention(*args, 0.25)
    # fp32 scores below 64, products and sums over 40 keys: a few 2^-19 of sum P |v|
    assert ((out[:4].double() - want[:4]).abs() <= size[:4] * 2.0 ** -16).all()


@pytest.mark.parametrize("mode", I.MODES)
def test_the_compositions_of_write_and_read_back(mode):
    g = torch.Generator().manual_seed(3)
    x, y = I.rows(20, 2, 64, FP, 1), I.rows(20, 2, 64, FP, 2)
    pages = torch.zeros(2, 4, 8, 2, i4.int4_row_bytes(64), dtype=torch.uint8)
    (kc, kg), (vc, vg) = (i4.int4_cache_views(p) for p in pages)
    ks, vs = I.scales(mode, 2, g), I.scales(mode, 2, g)
    table = torch.tensor([[2, 0, 3]])
    slots = torch.tensor([table[0, i // 8] * 8 + i % 8 for i in range(20)])
    slots[7] = -1
    i4.reshape_and_cache_int4_reference(x, y, kc, vc, kg, vg, slots, ks, vs)
    key, value = torch.full((21, 2, 64), 7.0, dtype=FP), torch.full((21, 2, 64), 7.0, dtype=FP)
    i4.gather_cache_int4_reference(kc, vc, kg, vg, key, value, torch.tensor([0, 20]), table, None,
                                   ks, vs)
    for r, got, s in ((x, key, ks), (y, value, vs)):
        want = i4.int4_values(*i4.quantise_int4(r, s), s).to(FP)
        want[7] = 0.0
        assert torch.equal(got[:20].nan_to_num(-9), want.nan_to_num(-9)) and (got[20] == 7).all()


def test_views_of_pages():
    for d in (64, 128, 256):
        pages = torch.zeros(3, 16, 2, i4.int4_row_bytes(d), dtype=torch.uint8)
        codes, groups = i4.int4_cache_views(pages)
        codes.fill_(1)
        groups.fill_(0x0202)
        assert int((pages == 1).sum()) == 3 * 16 * 2 * d // 2
        assert int((pages == 2).sum()) == 3 * 16 * 2 * d // 16 and not (pages == 0).any()
    for bad in (torch.zeros(3, 16, 2, 80, dtype=torch.uint8), torch.zeros(3, 16, 2, 72),
                torch.zeros(16, 2, 72, dtype=torch.uint8),
                torch.zeros(3, 2, 16, 72, dtype=torch.uint8).transpose(1, 2)):
        with pytest.raises(ValueError):
            i4.int4_cache_views(bad)
    with pytest.raises(NotImplementedError):
        i4.int4_row_bytes(96)


def _write_args(**kw):
    x = torch.ones(3, 2, 64, dtype=BF)
    c, w = torch.zeros(4, 16, 2, 32, dtype=torch.uint8), torch.zeros(4, 2, 16, 2, dtype=torch.int16)
    a = dict(key=x, value=x.clone(), key_cache=c, value_cache=c.clone(), key_groups=w,
             value_groups=w.clone(), slot_mapping=torch.arange(3))
    return dict(a, **kw)


BAD = [(dict(key_cache=torch.zeros(4, 16, 2, 32)), NotImplementedError),
       (dict(key_cache=torch.zeros(4, 16, 2, 48, dtype=torch.uint8),
             value_cache=torch.zeros(4, 16, 2, 48, dtype=torch.uint8)), NotImplementedError),
       (dict(value_cache=torch.zeros(4, 8, 2, 32, dtype=torch.uint8)), ValueError),
       (dict(key_groups=torch.zeros(4, 16, 2, 2, dtype=torch.int16)), ValueError),
       (dict(key_groups=torch.zeros(4, 2, 16, 2, dtype=torch.int32)), ValueError),
       (dict(value_groups=torch.zeros(4, 2, 16, 4, dtype=torch.int16)[..., ::2]), ValueError),
       (dict(k_scale=torch.ones(3)), ValueError), (dict(v_scale=torch.ones(1, 2)), ValueError),
       (dict(v_scale=torch.ones(1, dtype=torch.float64)), ValueError),
       (dict(key=torch.ones(3, 2, 64)), NotImplementedError),
       (dict(value=torch.ones(3, 2, 64, dtype=FP)), NotImplementedError),
       (dict(key=torch.ones(3, 2, 32, dtype=BF)), ValueError),
       (dict(key=torch.ones(3, 2, 128, dtype=BF)[..., ::2]), ValueError)]


@pytest.mark.parametrize("kw,error", BAD + [(dict(slot_mapping=torch.arange(4)), ValueError),
                                            (dict(), ValueError)])
def test_writes_that_are_refused(kw, error):
    with pytest.raises(error):  # (the last: the CPU)
        i4.reshape_and_cache_int4(**_write_args(**kw))


@pytest.mark.parametrize("kw,error", BAD + [
    (dict(value=torch.ones(4, 2, 64, dtype=BF)), ValueError),
    (dict(cu_seqlens=torch.tensor([0, 4])), ValueError),
    (dict(cu_seqlens=torch.tensor([0, 3, 2])), ValueError),
    (dict(starts=torch.ones(1)), ValueError), (dict(), ValueError)])
def test_read_backs_that_are_refused(kw, error):
    a = dict(_write_args(), cu_seqlens=torch.tensor([0, 3]),
             block_table=torch.zeros(1, 1, dtype=torch.int32))
    del a["slot_mapping"]
    with pytest.raises(error):
        i4.gather_cache_int4(**dict(a, **kw))


@pytest.mark.parametrize("kw,error", BAD[:9] + [
    (dict(query=torch.ones(1, 2, 64).to(torch.float8_e4m3fn)), NotImplementedError)])
def test_attention_that_is_refused(kw, error):
    a = _write_args()
    for name in ("key", "value", "slot_mapping"):
        del a[name]
    a.update(query=torch.ones(1, 2, 64), out=torch.zeros(1, 2, 64),
             cu_seqlens_q=torch.tensor([0, 1]), seqused_k=torch.tensor([3]),
             block_table=torch.zeros(1, 1, dtype=torch.int32), softmax_scale=0.1)
    with pytest.raises(error):
        i4.paged_decode_attention_int4(**dict(a, **kw))


def _cache(**kw):
    a = _lib.FpKvCacheInt4Args()
    b = a.base
    b.key = b.value = b.key_cache = b.value_cache = b.slot_mapping = 0x10000
    a.k_groups.data = a.v_groups.data = 0x20000
    for g in (a.k_groups, a.v_groups):
        g.stride_block, g.stride_head = 128, 64
    b.k_stride_tok = b.v_stride_tok = 256
    b.k_stride_head = b.v_stride_head = 128
    b.kc_stride_head = b.vc_stride_head = 64
    b.kc_stride_block = b.vc_stride_block = 2048
    b.kc_stride_slot = b.vc_stride_slot = 128
    b.num_tokens, b.num_blocks, b.block_size, b.num_kv_heads, b.head_dim = 5, 4, 16, 2, 128
    for k, v in kw.items():
        if k.startswith("g_"):
            setattr(a.k_groups, k[2:], v)
        elif k.startswith("s_"):
            setattr(a.v_scale, k[2:], v)
        else:
            setattr(b, k, v)
    return a


BAD_ARGS = [(dict(dtype=_lib.FP_DTYPE_F32), _lib.FP_E_UNSUPPORTED),
            (dict(head_dim=96), _lib.FP_E_UNSUPPORTED), (dict(num_kv_heads=0), _lib.FP_E_INVALID_ARG),
            (dict(key=0), _lib.FP_E_INVALID_ARG), (dict(key_cache=0x10008), _lib.FP_E_INVALID_ARG),
            (dict(kc_stride_slot=72), _lib.FP_E_INVALID_ARG), (dict(g_data=0), _lib.FP_E_INVALID_ARG),
            (dict(g_data=0x20004), _lib.FP_E_INVALID_ARG),
            (dict(g_stride_head=66), _lib.FP_E_INVALID_ARG),
            (dict(g_stride_block=-64), _lib.FP_E_INVALID_ARG),
            (dict(s_data=0x10002), _lib.FP_E_INVALID_ARG),
            (dict(s_data=0x10000, s_per_slot=1), _lib.FP_E_UNSUPPORTED),
            (dict(num_tokens=1 << 28), _lib.FP_E_UNSUPPORTED)]


@pytest.mark.parametrize("kw,code", BAD_ARGS + [(dict(slot_mapping=0), _lib.FP_E_INVALID_ARG)])
def test_the_c_write_refuses(kw, code):
    assert _lib.load().fp_kv_cache_write_int4(ctypes.byref(_cache(**kw)), None) == code
    assert _lib.load().fp_kv_cache_write_int4(None, None) == _lib.FP_E_INVALID_ARG


@pytest.mark.parametrize("kw,code", BAD_ARGS)
def test_the_c_read_back_refuses(kw, code):
    a = _lib.FpKvGatherInt4Args()
    a.cache, a.batch, a.table_width, a.cu_seqlens, a.block_table = _cache(**kw), 1, 2, 8, 8
    gather = _lib.load().fp_kv_cache_gather_int4
    assert gather(ctypes.byref(a), None) == code
    a.cache, a.batch = _cache(), 0
    assert gather(ctypes.byref(a), None) == _lib.FP_E_INVALID_ARG
    assert gather(None, None) == _lib.FP_E_INVALID_ARG


def _paged(tokens=4, batch=2, hq=8, hkv=2, d=128, page=16, width=200, **kw):
    a = _lib.FpPagedInt4Args()
    b = a.base
    b.q = b.o = b.key_cache = b.value_cache = b.cu_seqlens = b.seqused = b.block_table = 0x10000
    a.k_groups.data = a.v_groups.data = 0x20000
    b.q_stride_tok = b.o_stride_tok = hq * d
    b.q_stride_head = b.o_stride_head = d
    b.kc_stride_slot = b.vc_stride_slot = hkv * d // 2
    b.kc_stride_block = b.vc_stride_block = page * hkv * d // 2
    b.kc_stride_head = b.vc_stride_head = d // 2
    b.table_stride, b.num_tokens, b.num_blocks = width, tokens, 4
    b.batch, b.table_width, b.block_size = batch, width, page
    b.num_q_heads, b.num_kv_heads, b.head_dim = hq, hkv, d
    for g in (a.k_groups, a.v_groups):
        g.stride_block, g.stride_head = hkv * page * d // 32, page * d // 32
    for k, v in kw.items():
        setattr(a.k_groups if k.startswith("g_") else a.k_scale if k.startswith("s_") else b,
                k[2:] if k[:2] in ("g_", "s_") else k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(d=96), _lib.FP_E_UNSUPPORTED), (dict(kc_stride_slot=72), _lib.FP_E_INVALID_ARG),
    (dict(g_data=0x20008), _lib.FP_E_INVALID_ARG), (dict(g_stride_head=60), _lib.FP_E_INVALID_ARG),
    (dict(page=5, g_stride_head=22), _lib.FP_E_INVALID_ARG), (dict(g_data=0), _lib.FP_E_INVALID_ARG),
    (dict(s_data=0x10000, s_per_slot=1), _lib.FP_E_UNSUPPORTED), (dict(), _lib.FP_E_INVALID_ARG)])
def test_the_c_attention_refuses(kw, code):  # (the last: no workspace)
    lib = _lib.load()
    assert lib.fp_paged_attention_int4(ctypes.byref(_paged(**kw)), None, None) == code
    assert lib.fp_paged_attention_int4(None, None, None) == _lib.FP_E_INVALID_ARG


@pytest.mark.parametrize("kw,want", [
    (dict(width=64), 0),  # room for 1,024 keys: whole segments, no merge
    (dict(tokens=2, batch=2), 2 * 2 * 16 * 2 * 25 * 130 * 4),  # 25 units x 2 segments, 50 groups
    (dict(tokens=64, batch=64, width=8192), 768 * 2 * 16 * 2 * 130 * 4),
    (dict(tokens=64, batch=64, d=256, width=8192), 512 * 2 * 16 * 258 * 4),
    (dict(tokens=64, batch=64, hkv=4, d=64, width=8192), 768 * 2 * 16 * 4 * 66 * 4),
    (dict(tokens=40960, batch=2, width=4096), 0)])  # many rows, enough tiles: no chunks
def test_workspace(kw, want):
    assert _lib.load().fp_paged_int4_workspace_bytes(ctypes.byref(_paged(**kw))) == want


def test_hooked_layers_with_4_bit_caches():
    calls = []
    ops = vb.HookOps(cache_write_int4=lambda *a: calls.append(("write", a)),
                     decode_int4=lambda *a: calls.append(("decode", a)))
    forward = vb.make_forward(vb.ATTENTION_CONFIGS["flashprefill_llama"], ops)
    kv = torch.zeros(2, 4, 16, 2, i4.int4_row_bytes(64), dtype=torch.uint8)
    x = torch.zeros(1, 2, 64, dtype=BF)
    meta = SimpleNamespace(num_actual_tokens=1, slot_mapping=torch.zeros(1, dtype=torch.int64),
                           max_query_len=1, query_start_loc=torch.tensor([0, 1]),
                           seq_lens=torch.tensor([1]), block_table=torch.zeros(1, 1))
    layer = SimpleNamespace(_k_scale=torch.ones(1), _v_scale=None)
    forward(SimpleNamespace(kv_cache_dtype="int4"), layer, x, x, x, kv, meta, output=x.clone())
    (_, w), (_, d) = calls
    assert w[2].shape == (4, 16, 2, 32) and w[4].shape == (4, 2, 16, 2) and w[4].dtype == torch.int16
    assert w[7] is layer._k_scale and w[8] is None
    assert d[3].data_ptr() == w[4].data_ptr() and d[-2] is layer._k_scale
    with pytest.raises(ValueError):
        forward(SimpleNamespace(kv_cache_dtype="int4"), layer, x, x, x, kv.float(), meta,
                output=x.clone())


@needs_hipcc
@pytest.mark.parametrize("source,kernels", [("fp_paged4.hip", 34), ("fp_kvcache4.hip", 12),
                                            ("fp_rotary.hip", 16), ("fp_steps.hip", 4)])
def test_registers(source, kernels):
    """None spills a vector register; few rows leave three waves to a SIMD (two at head_dim
    256), many rows two (one at 256)."""
    found = _registers(_assembly(source))
    assert len(found) == kernels, len(found)
    for name, (regs, spilled) in found.items():
        few = re.match(r"_ZN2fp8k_paged4ILi(\d+)E", name)
        rows = re.match(r"_ZN2fp13k_paged4_rowsILi(\d+)E", name)
        most = {"64": 168, "128": 168, "256": 256}[few.group(1)] if few else \
            {"64": 256, "128": 256, "256": 512}[rows.group(1)] if rows else 128
        assert spilled == 0 and regs <= most, (name, regs, spilled)

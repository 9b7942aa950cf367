"""CPU tests of the 8-bit KV cache: what its entry points refuse, the torch composition of
attention over it, and the hooked forwards' dispatch for layers with an fp8 cache."""

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from tests._kv8 import E4M3, E5M2, MODES, attention, attention_case
from flashprefill_amd import _lib
from flashprefill_amd import vllm_backend as vb

BF = torch.bfloat16


def _tensors(dtype=BF, fmt=E4M3):
    x = torch.ones(3, 2, 64, dtype=dtype)
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.uint8).view(fmt)
    return x, cache, torch.arange(3)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_the_composition_of_attention(mode, fmt):
    args = attention_case([40, 7, 0], [1, 3, 1], 4, 2, 16, 4, torch.float32, fmt, mode)
    out = torch.empty(5, 4, 16)
    vb.paged_decode_attention(*args[:3], out, *args[3:6], 0.25, *args[6:])
    want, size = attention(*args, 0.25)
    # fp32 scores below 16, products and sums over 40 keys: a few 2^-20 of sum P |v|
    assert ((out[:4].double() - want[:4]).abs() <= size[:4] * 2.0 ** -18).all()


def test_scales_that_do_not_fit():
    x, cache, slots = _tensors()
    one = torch.ones(1)
    for bad in (torch.ones(3), torch.ones(2, 1), torch.ones(4, 16, 2), torch.ones(0),
                torch.ones(1, dtype=torch.float64), torch.ones(4, 2, 32)[..., ::2],
                torch.ones(4, 2, 16, 1)):
        for ks, vs in ((bad, one), (one, bad)):
            with pytest.raises(ValueError, match="scale"):
                vb.reshape_and_cache(x, x, cache, cache.clone(), slots, ks, vs)
            with pytest.raises(ValueError, match="scale"):
                vb.paged_decode_attention(x, cache, cache, torch.empty_like(x), torch.arange(4),
                                          torch.ones(3), torch.zeros(3, 1), 0.1, ks, vs)
            with pytest.raises(ValueError, match="scale"):
                vb.gather_cache(cache, cache, x, x.clone(), torch.tensor([0, 3]),
                                torch.zeros(1, 1, dtype=torch.int32), None, ks, vs)
    plain = torch.zeros(4, 16, 2, 64, dtype=BF)
    with pytest.raises(ValueError, match="8-bit"):
        vb.reshape_and_cache(x, x, plain, plain.clone(), slots, one)
    with pytest.raises(ValueError, match="8-bit"):
        vb.gather_cache(plain, plain, x, x.clone(), torch.tensor([0, 3]),
                        torch.zeros(1, 1, dtype=torch.int32), None, one)


def test_types_and_shapes_that_do_not_fit():
    x, cache, slots = _tensors()
    for k, v, kc, vc in ((x.float(), x.float(), cache, cache), (x, x.half(), cache, cache),
                         (x, x, cache, cache.view(torch.uint8).view(E5M2)),
                         (x, x, cache.view(torch.uint8), cache.view(torch.uint8)),
                         (x.half(), x.half(), cache.to(BF), cache.to(BF))):
        with pytest.raises(NotImplementedError):
            vb.reshape_and_cache(k, v, kc, vc, slots)
        with pytest.raises(NotImplementedError):
            vb.gather_cache(kc, vc, k, v, torch.tensor([0, 3]), torch.zeros(1, 1, dtype=torch.int32))
    for k, kc in ((x[:, :1], cache), (x[..., :32], cache), (x[0], cache), (x, cache[0])):
        with pytest.raises(ValueError):
            vb.reshape_and_cache(k, k, kc, kc, slots)
    with pytest.raises(ValueError, match="do not match"):
        vb.reshape_and_cache(x, x, cache, cache, torch.arange(4))
    with pytest.raises(ValueError, match="contiguous"):
        vb.reshape_and_cache(torch.ones(3, 2, 128, dtype=BF)[..., ::2], x, cache, cache, slots)
    with pytest.raises(ValueError, match="one GPU"):
        vb.reshape_and_cache(x, x, cache, cache.clone(), slots)


def test_read_backs_that_do_not_fit():
    x, cache, _ = _tensors()
    table, cu = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 3])

    def call(key=x, cu=cu, table=table, starts=None):
        vb.gather_cache(cache, cache, key, x.clone(), cu, table, starts)

    for kw in (dict(key=x[:2]), dict(cu=cu.view(1, 2)), dict(table=table[0]), dict(table=table[:0]),
               dict(cu=cu.float()), dict(table=table.to(torch.int16)),
               dict(starts=torch.zeros(0, dtype=torch.int32)), dict(starts=torch.zeros(1)),
               dict(cu=torch.tensor([0, 4])), dict(cu=torch.tensor([-1, 3])),
               dict(cu=torch.tensor([0, 3, 2]), table=table.expand(2, 1)),
               dict(cu=torch.zeros(0, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(ValueError, match="one GPU"):
        call()


def _write(**kw):
    a = _lib.FpKvCacheFp8Args()
    b = a.base
    b.key = b.value = b.key_cache = b.value_cache = b.slot_mapping = 0x10000
    b.k_stride_tok = b.v_stride_tok = 256
    b.k_stride_head = b.v_stride_head = b.kc_stride_head = b.vc_stride_head = 128
    b.kc_stride_block = b.vc_stride_block = 4096
    b.kc_stride_slot = b.vc_stride_slot = 256
    b.num_tokens, b.num_blocks, b.block_size, b.num_kv_heads, b.head_dim = 5, 4, 16, 2, 128
    a.format = _lib.FP_CACHE_E4M3
    for k, v in kw.items():
        if k.startswith("ks_"):
            setattr(a.k_scale, k[3:], v)
        else:
            setattr(b if hasattr(b, k) else a, k, v)
    return a


BAD_ROWS = [(dict(dtype=_lib.FP_DTYPE_F32), _lib.FP_E_UNSUPPORTED),
            (dict(head_dim=520), _lib.FP_E_UNSUPPORTED), (dict(head_dim=12), _lib.FP_E_INVALID_ARG),
            (dict(num_kv_heads=0), _lib.FP_E_INVALID_ARG), (dict(block_size=0), _lib.FP_E_INVALID_ARG),
            (dict(num_tokens=-1), _lib.FP_E_INVALID_ARG), (dict(key=0), _lib.FP_E_INVALID_ARG),
            (dict(key=0x10008), _lib.FP_E_INVALID_ARG), (dict(value_cache=0x10004), _lib.FP_E_INVALID_ARG),
            (dict(kc_stride_head=132), _lib.FP_E_INVALID_ARG), (dict(v_stride_tok=-8), _lib.FP_E_INVALID_ARG),
            (dict(num_tokens=1 << 31), _lib.FP_E_UNSUPPORTED),
            (dict(ks_per_slot=1), _lib.FP_E_INVALID_ARG),
            (dict(ks_data=0x10002), _lib.FP_E_INVALID_ARG),
            (dict(ks_data=0x10000, ks_stride_head=-1), _lib.FP_E_INVALID_ARG)]


@pytest.mark.parametrize("kw,rc", BAD_ROWS + [(dict(format=3), _lib.FP_E_UNSUPPORTED),
                                              (dict(format=_lib.FP_CACHE_16BIT), _lib.FP_E_UNSUPPORTED),
                                              (dict(slot_mapping=0), _lib.FP_E_INVALID_ARG),
                                              (dict(num_tokens=0), _lib.FP_OK)])
def test_the_write_checks_its_arguments(kw, rc):
    lib = _lib.load()
    assert lib.fp_kv_cache_write_fp8(ctypes.byref(_write(**kw)), None) == rc
    assert lib.fp_kv_cache_write_fp8(None, None) == _lib.FP_E_INVALID_ARG


@pytest.mark.parametrize("kw,rc", BAD_ROWS + [(dict(format=3), _lib.FP_E_UNSUPPORTED),
                                              (dict(batch=0), _lib.FP_E_INVALID_ARG),
                                              (dict(cu_seqlens=0), _lib.FP_E_INVALID_ARG),
                                              (dict(block_table=0), _lib.FP_E_INVALID_ARG),
                                              (dict(table_width=1 << 27), _lib.FP_E_UNSUPPORTED),
                                              (dict(format=0, value_cache=0x10008), _lib.FP_E_INVALID_ARG),
                                              (dict(num_tokens=0), _lib.FP_OK)])
def test_the_read_back_checks_its_arguments(kw, rc):
    lib, a = _lib.load(), _lib.FpKvGatherArgs()
    w = _write(**{k: v for k, v in kw.items() if hasattr(_write(), k) or
                  hasattr(_write().base, k) or k.startswith("ks_")})
    a.base, a.k_scale, a.format = w.base, w.k_scale, w.format
    a.batch, a.table_width, a.table_stride = 2, 3, 3
    a.cu_seqlens = a.block_table = 0x10000
    for k, v in kw.items():
        if k in ("batch", "cu_seqlens", "block_table", "table_width"):
            setattr(a, k, v)
    assert lib.fp_kv_cache_gather(ctypes.byref(a), None) == rc
    assert lib.fp_kv_cache_gather(None, None) == _lib.FP_E_INVALID_ARG


def test_attention_checks_its_arguments():
    lib = _lib.load()

    def call(**kw):
        a = _lib.FpPagedFp8Args()
        b = a.base
        b.q = b.o = b.key_cache = b.value_cache = b.cu_seqlens = b.seqused = b.block_table = 0x10000
        b.q_stride_tok = b.o_stride_tok = 1024
        b.q_stride_head = b.o_stride_head = b.kc_stride_head = b.vc_stride_head = 128
        b.kc_stride_block = b.vc_stride_block = 4096
        b.kc_stride_slot = b.vc_stride_slot = 256
        b.table_stride, b.num_tokens, b.num_blocks = 3, 2, 4
        b.batch, b.table_width, b.block_size = 2, 3, 16
        b.num_q_heads, b.num_kv_heads, b.head_dim = 8, 2, 128
        a.format = _lib.FP_CACHE_E4M3
        for k, v in kw.items():
            setattr(a.k_scale, k[3:], v) if k.startswith("ks_") else \
                setattr(b if hasattr(b, k) else a, k, v)
        return (lib.fp_paged_attention_fp8(ctypes.byref(a), None, None),
                lib.fp_paged_fp8_workspace_bytes(ctypes.byref(a)))

    for kw, rc in ((dict(format=0), _lib.FP_E_UNSUPPORTED), (dict(head_dim=96), _lib.FP_E_UNSUPPORTED),
                   (dict(kc_stride_head=136), _lib.FP_E_INVALID_ARG),
                   (dict(ks_per_slot=1), _lib.FP_E_INVALID_ARG),
                   (dict(ks_per_slot=1, ks_data=0x10004), _lib.FP_E_INVALID_ARG),
                   (dict(ks_per_slot=1, ks_data=0x10000, ks_stride_block=6), _lib.FP_E_INVALID_ARG),
                   (dict(num_q_heads=7), _lib.FP_E_INVALID_ARG)):
        assert call(**kw) == (rc, 0), kw
    assert call(num_tokens=0) == (_lib.FP_OK, 0)
    assert lib.fp_paged_attention_fp8(None, None, None) == _lib.FP_E_INVALID_ARG


def _hook(name, kv, layer, **kw):
    calls = []
    ops = vb.HookOps(cache_write=lambda *a: calls.append(("cache", a)),
                     prefill=lambda *a: calls.append(("prefill", a)),
                     decode=lambda *a: calls.append(("decode", a)),
                     cache_write_fp8=lambda *a: calls.append(("cache8", a)),
                     decode_fp8=lambda *a: calls.append(("decode8", a)))
    q, k = torch.randn(3, 4, 8), torch.randn(3, 2, 8)
    impl = SimpleNamespace(kv_cache_dtype=name, scale=0.3, **kw)
    one = torch.arange(4, dtype=torch.int32)
    meta = SimpleNamespace(num_actual_tokens=3, query_start_loc=one, max_query_len=1,
                           seq_lens=torch.tensor([5, 9, 2]), block_table=torch.zeros(3, 4),
                           slot_mapping=torch.arange(3), use_cascade=False)
    vb.make_forward(vb.ATTENTION_CONFIGS["flashprefill_llama"], ops)(
        impl, layer, q, k, k, kv, meta, output=torch.empty_like(q))
    v0 = SimpleNamespace(num_prefill_tokens=2, num_decode_tokens=1, slot_mapping=torch.arange(3),
                         prefill_metadata=SimpleNamespace(
                             block_tables=torch.ones(2, 4), query_start_loc=one[:3],
                             seq_lens_tensor=torch.tensor([5, 9])),
                         decode_metadata=SimpleNamespace(
                             max_decode_query_len=1, seq_lens_tensor=torch.tensor([2]),
                             block_tables=torch.zeros(1, 4)))
    vb.make_forward_v0(vb.ATTENTION_CONFIGS["flashprefill_llama"], ops)(
        impl, layer, q, k, k, kv, v0, output=torch.empty_like(q))
    return calls


@pytest.mark.parametrize("name,fmt", [("fp8", E4M3), ("fp8_e4m3", E4M3), ("fp8_e5m2", E5M2)])
@pytest.mark.parametrize("as_bytes", [True, False])
def test_hooked_forwards_of_an_fp8_layer(name, fmt, as_bytes):
    kv = torch.zeros(2, 6, 4, 2, 8, dtype=torch.uint8)
    layer = SimpleNamespace(_k_scale=torch.tensor(0.5), _v_scale=torch.tensor(0.25))
    calls = _hook(name, kv if as_bytes else kv.view(fmt), layer)
    assert [c[0] for c in calls] == ["cache8", "decode8", "cache8", "decode8", "decode8"]
    for what, a in calls:
        kc, vc = a[2:4] if what == "cache8" else a[1:3]
        assert kc.dtype == vc.dtype == fmt and kc.data_ptr() == kv[0].data_ptr()
        assert vc.data_ptr() == kv[1].data_ptr()
        assert a[-2] is layer._k_scale and a[-1] is layer._v_scale
    assert calls[1][1][7] == 0.3 and calls[1][1][3].shape == (3, 4, 8)


def test_hooked_forwards_without_scales_and_of_other_caches():
    kv = torch.zeros(2, 6, 4, 2, 8, dtype=torch.uint8)
    calls = _hook("fp8", kv, SimpleNamespace())
    assert all(a[-2:] == (None, None) for _, a in calls)
    shared = _hook("fp8", kv, None, kv_sharing_target_layer_name="layers.0")
    assert shared[0][0] == "decode8"
    for name, cache in (("fp8", kv.float()), ("fp8_inc", kv), ("fp8_ds_mla", kv),
                        ("fp8_e5m2", kv.view(E4M3))):
        with pytest.raises(NotImplementedError):
            _hook(name, cache, None)
    plain = _hook("auto", kv.to(BF), None)
    assert [c[0] for c in plain] == ["cache", "decode", "cache", "decode", "decode"]
    assert math.isclose(plain[1][1][-1], 0.3)

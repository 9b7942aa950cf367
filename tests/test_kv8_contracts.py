"""CPU tests of what the 8-bit KV cache's operators refuse or leave to torch operations."""

import math
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from tests._kv8 import E4M3, E5M2, MODES, quantise, scales, values
from tests._kv8_paths import path
from flashprefill_amd import vllm_backend as vb

BF = torch.bfloat16


def _step(queries, max_query_len=1):
    return SimpleNamespace(num_actual_tokens=queries, max_query_len=max_query_len,
                           query_start_loc=torch.arange(queries + 1, dtype=torch.int32),
                           seq_lens=torch.full((queries,), 5), slot_mapping=torch.arange(queries),
                           block_table=torch.zeros(queries, 2, dtype=torch.int32), use_cascade=False)


@pytest.mark.parametrize("qdtype", [E4M3, E5M2, torch.float8_e4m3fnuz, torch.uint8])
def test_queries_of_8_bits_are_refused_by_an_8_bit_cache(qdtype):
    """Their codes mean nothing without the layer's query scale."""
    q = torch.ones(2, 4, 8).to(qdtype)
    cache = torch.zeros(6, 4, 2, 8, dtype=torch.uint8).view(E4M3)
    out = torch.full((2, 4, 8), 7.0, dtype=BF)
    args = (q, cache, cache, out, torch.arange(3), torch.tensor([5, 5]), torch.zeros(2, 2).int(), 0.3)
    for fn in (vb.paged_decode_attention, vb.paged_attention_reference):
        with pytest.raises(NotImplementedError, match="query"):
            fn(*args)
    # through the hooked forwards (the cache write, a kernel, stands aside)
    ops = vb.HookOps(cache_write_fp8=lambda *a: None)
    impl = SimpleNamespace(kv_cache_dtype="fp8", scale=0.3)
    layer = SimpleNamespace(_q_scale=torch.tensor(0.05), _k_scale=torch.tensor(0.5),
                            _v_scale=torch.tensor(0.5))
    kv, k = torch.zeros(2, 6, 4, 2, 8, dtype=torch.uint8), torch.ones(2, 2, 8, dtype=BF)
    cfg = vb.ATTENTION_CONFIGS["flashprefill_llama"]
    with pytest.raises(NotImplementedError, match="query"):
        vb.make_forward(cfg, ops)(impl, layer, q, k, k, kv, _step(2), output=out)
    v0 = SimpleNamespace(num_prefill_tokens=0, num_decode_tokens=2, prefill_metadata=None,
                         slot_mapping=torch.arange(2),
                         decode_metadata=SimpleNamespace(
                             max_decode_query_len=1, seq_lens_tensor=torch.tensor([5, 5]),
                             block_tables=torch.zeros(2, 2, dtype=torch.int32)))
    with pytest.raises(NotImplementedError, match="query"):
        vb.make_forward_v0(cfg, ops)(impl, layer, q, k, k, kv, v0, output=out)
    assert (out == 7.0).all()


# ---------------------------------------------------------------------------
# traces, dispatch modes and forward-mode tangents
# ---------------------------------------------------------------------------

def _write_case(fmt, mode, seed=0):
    """Rows with values that a cast can go wrong at, slots of padding, past the cache and
    none, zeroed caches, scales."""
    g = torch.Generator().manual_seed(seed)
    nb, page, hkv, d, n = 5, 6, 3, 24, 22
    k, v = (torch.randn(n, hkv, d, generator=g).to(BF) for _ in range(2))
    k[0], k[1, :, 0], k[2, 0, 1], k[3] = 0.0, math.inf, math.nan, torch.finfo(BF).max
    v[4], v[5, 1], v[6] = -0.0, -math.inf, 2.0 ** -130
    slots = torch.randperm(nb * page, generator=g)[:n]
    slots[7], slots[8], slots[9] = -1, nb * page, -100
    kc, vc = (torch.zeros(nb, page, hkv, d, dtype=torch.uint8).view(fmt) for _ in range(2))
    ks, vs = (scales(mode, nb, page, hkv, g) for _ in range(2))
    return k, v, kc, vc, slots, ks, vs


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("mode", MODES)
def test_the_composition_of_the_write(fmt, mode):
    k, v, kc, vc, slots, ks, vs = _write_case(fmt, mode)
    vb.reshape_and_cache_reference(k, v, kc, vc, slots, ks, vs)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        fixed = torch.ones(1, 1) if s is None else s.view(1, -1) if mode != "slot" else None
        codes, found = quantise(x, fmt, fixed)
        want = torch.zeros(30, 3, 24, dtype=torch.uint8)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < 30:
                want[slot] = codes[t].view(torch.uint8)
                if mode == "slot":
                    assert torch.equal(s[slot // 6, :, slot % 6], found[t])
        assert torch.equal(c.view(torch.uint8).view(30, 3, 24), want)


def test_the_composition_of_a_16_bit_write():
    k, v, kc, vc, slots, _, _ = _write_case(E4M3, "none")
    kc, vc = torch.zeros(kc.shape, dtype=BF), torch.zeros(kc.shape, dtype=BF)
    vb.reshape_and_cache_reference(k, v, kc, vc, slots)
    for x, c in ((k, kc), (v, vc)):
        want = torch.zeros(30, 3, 24, dtype=BF)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < 30:
                want[slot] = x[t]
        assert torch.equal(c.view(30, 3, 24).view(torch.int16), want.view(torch.int16))


def _read_back_case(fmt, mode, seed=0):
    """Sequences of none to many tokens, rows before the first and behind the last, a table
    with pages counted from the end and outside the cache."""
    g = torch.Generator().manual_seed(seed)
    nb, page, hkv, d = 9, 4, 2, 16
    kc, vc = (torch.randn(nb, page, hkv, d, generator=g).to(fmt) for _ in range(2))
    ks, vs = (None, None) if fmt == BF else (scales(mode, nb, page, hkv, g) for _ in range(2))
    cu = torch.tensor([2, 9, 9, 12, 13, 15], dtype=torch.int32)
    table = torch.randint(0, nb, (5, 3), generator=g, dtype=torch.int64)
    table[0, 1], table[2, 0] = -2, nb
    starts = torch.tensor([1, 0, 3, -1, 11])  # the fourth before the first token, the last past the room
    key, value = (torch.full((18, hkv, d), 7.0, dtype=BF) for _ in range(2))
    return kc, vc, key, value, cu, table, starts, ks, vs


def _read_back(cache, scale, rows, cu, table, starts):
    nb, page = cache.shape[:2]
    x, want = values(cache, scale), rows.clone()
    for b in range(cu.numel() - 1):
        for i in range(int(cu[b + 1]) - int(cu[b])):
            t = i + (0 if starts is None else int(starts[b]))
            want[int(cu[b]) + i] = math.nan
            if t >= 0 and (starts is None or starts[b] >= 0) and t < table.shape[1] * page:
                p = int(table[b, t // page])
                if -nb <= p < nb:  # (products of an 8-bit value and a scale in fp32)
                    want[int(cu[b]) + i] = x[p, t % page].float().to(BF)
    return want


@pytest.mark.parametrize("fmt,mode", [(BF, "none")] + [(f, m) for f in (E4M3, E5M2) for m in MODES])
@pytest.mark.parametrize("from_first", [True, False])
def test_the_composition_of_the_read_back(fmt, mode, from_first):
    kc, vc, key, value, cu, table, starts, ks, vs = _read_back_case(fmt, mode)
    starts = None if from_first else starts
    want = [_read_back(c, s, r, cu, table, starts) for c, s, r in ((kc, ks, key), (vc, vs, value))]
    vb.gather_cache_reference(kc, vc, key, value, cu, table, starts, ks, vs)
    for got, w in zip((key, value), want):
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(), w.nan_to_num())
    for bad in ([0, 5, 3], [-1, 4, 9], [0, 4, 19]):  # offsets that do not fit: every row
        vb.gather_cache_reference(kc, vc, key, value, torch.tensor(bad), table, None, ks, vs)
        assert key.isnan().all() and value.isnan().all()
    key.fill_(1.0)  # a table without room
    vb.gather_cache_reference(kc, vc, key, value, torch.tensor([0, 2]), table[:, :0], None, ks, vs)
    assert key[:2].isnan().all() and (key[2:] == 1.0).all()


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_a_trace_holds_the_write_and_the_read_back():
    """Traced over fake tensors, which have no memory: nothing may reach a kernel."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.fx.experimental.symbolic_shapes import ShapeEnv

    env = ShapeEnv(allow_dynamic_output_shape_ops=True)
    with FakeTensorMode(shape_env=env, allow_non_fake_inputs=True):
        x = torch.empty(3, 2, 64, dtype=BF, device="cuda")
        cache = [torch.empty(4, 16, 2, 64, dtype=torch.uint8, device="cuda").view(E4M3)
                 for _ in range(2)]
        sc = [torch.empty(4, 2, 16, device="cuda") for _ in range(2)]
        slots = torch.empty(3, dtype=torch.int64, device="cuda")
        cu, table = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((2,), (1, 4)))

        def step(x, kc, vc, ks, vs, slots, cu, table):
            y, z = torch.zeros_like(x), torch.zeros_like(x)
            vb.reshape_and_cache(x, x, kc, vc, slots, ks, vs)
            vb.gather_cache(kc, vc, y, z, cu, table, None, ks, vs)
            return y, z

        ops = [str(n.target) for n in make_fx(step)(x, *cache, *sc, slots, cu, table).graph.nodes]
        with pytest.raises(ValueError, match="of their own"):
            vb.reshape_and_cache(x, x, cache[0], cache[0], slots, *sc)
        with pytest.raises(ValueError, match="of their own"):
            vb.gather_cache(*cache, x, x, cu, table, None, *sc)
    assert sum("index_put" in o for o in ops) == 4 and sum("copy_" in o for o in ops) == 2


def test_tangents_are_refused():
    # (before anything looks for a GPU)
    k, v, kc, vc, slots, ks, vs = _write_case(E4M3, "head")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(k, torch.ones_like(k))
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.reshape_and_cache(dual, v, kc, vc, slots, ks, vs)
        wide = forward_ad.make_dual(vs, torch.ones_like(vs))
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.gather_cache(kc, vc, k, v, torch.tensor([0, 3]), torch.zeros(1, 9).int(), None, ks, wide)
        # tensors without one are taken as ever (and have to be on a GPU)
        with pytest.raises(ValueError, match="one GPU"):
            vb.reshape_and_cache(k, v, kc, vc, slots, ks, vs)


# ---------------------------------------------------------------------------
# which kernels the GPU tests' calls take
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("news,hq,hkv,d,page,width,want", [
    # one query each: short tables, long ones
    ([1, 1], 8, 2, 128, 16, 57, "whole"), ([1, 1], 8, 2, 128, 16, 64, "whole"),
    ([1, 1], 8, 2, 128, 16, 65, "shared"), ([1, 1, 1], 8, 2, 64, 16, 200, "shared"),
    # many rows
    ([40, 40], 8, 2, 128, 16, 200, "rows merged"), ([40, 40], 8, 2, 64, 16, 200, "rows merged"),
    ([150, 30, 141], 7, 1, 256, 16, 2500, "rows merged"), ([150, 30, 141], 34, 2, 256, 16, 2500, "rows merged"),
    ([130, 70], 8, 2, 256, 16, 1200, "rows merged"), ([700], 8, 2, 256, 16, 1200, "rows merged"),
    # head_dim 256 below 128 rows per sequence, and with so many
    ([150, 30, 141], 5, 5, 256, 16, 2500, "shared"), ([200, 90, 141], 5, 5, 256, 16, 2500, "rows merged"),
])
def test_which_kernels_a_call_takes(news, hq, hkv, d, page, width, want):
    assert path(sum(news), len(news), hq, hkv, d, page, width) == want

"""The 8-bit paged KV cache on the GPU where the call is unusual: under traces and dispatch
modes, in memory of the host, captured where workgroups share the keys."""

import math

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from tests._kv8 import E4M3, E5M2, MODES, attention, attention_case, bound, scales
from tests._kv8_paths import path
from flashprefill_amd import vllm_backend as vb

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


class _Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.ops = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.ops.append(str(func))
        return func(*args, **(kwargs or {}))


def _equal(a, b):
    """Equal values and signs, NaN (of either sign) where the other has NaN."""
    if not a.is_floating_point():
        return torch.equal(a, b)
    a, b = a.float(), b.float()
    nan = a.isnan()
    return torch.equal(nan, b.isnan()) and torch.equal(a[~nan].view(torch.int32),
                                                       b[~nan].view(torch.int32))


def _state(dtype, fmt, mode, page, seed):
    """Rows (among them zeros, infinities, NaN, the type's largest), slots with padding,
    caches and scales: what a call of each operator takes."""
    g = torch.Generator().manual_seed(seed)
    nb, hkv, d, n = 11, 3, 64, 90
    k, v = (torch.randn(n, hkv, d, generator=g).to(dtype) for _ in range(2))
    k[0], k[1, :, 0], k[2, 0, 1], k[3] = 0.0, math.inf, math.nan, torch.finfo(dtype).max
    slots = torch.randperm(nb * page, generator=g)[:n]
    slots[5], slots[6] = -1, nb * page
    c = [torch.zeros(nb, page, hkv, d, dtype=torch.uint8).view(fmt) if fmt in (E4M3, E5M2) else
         torch.zeros(nb, page, hkv, d, dtype=fmt) for _ in range(2)]
    sc = [scales(mode, nb, page, hkv, g) for _ in range(2)]
    cu = torch.tensor([1, 40, 40, 73], dtype=torch.int32)
    table = torch.randint(-2, nb, (3, 5), generator=g, dtype=torch.int32)
    table[1, 0] = nb
    starts = torch.tensor([2, 0, 7], dtype=torch.int32)
    y = [torch.full((90, hkv, d), 7.0, dtype=dtype) for _ in range(2)]
    return [None if t is None else t.to(DEV) for t in (k, v, *c, slots, *sc, cu, table, starts, *y)]


def _step(k, v, kc, vc, slots, ks, vs, cu, table, starts, y, z):
    vb.reshape_and_cache(k, v, kc, vc, slots, ks, vs)
    vb.gather_cache(kc, vc, y, z, cu, table, starts, ks, vs)
    return y, z


def _check_same(mine, other):
    assert all(a is None or _equal(a, b) for a, b in zip(mine, other))


@pytest.mark.parametrize("dtype,fmt,mode", [(t, f, m) for t in (BF, HF) for f in (E4M3, E5M2)
                                            for m in MODES] + [(BF, BF, "none")])
def test_a_dispatch_mode_sees_the_write_and_the_read_back(dtype, fmt, mode):
    for page in (16, 9):
        kernel, seen = (_state(dtype, fmt, mode, page, 3) for _ in range(2))
        _step(*kernel)
        with _Seen() as m:
            _step(*seen)
        assert sum("index_put" in o for o in m.ops) >= 2 and sum("copy_" in o for o in m.ops) >= 2
        _check_same(kernel, seen)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("fmt,mode", [(E4M3, "slot"), (E5M2, "head"), (E4M3, "none"), (BF, "none")])
def test_a_trace_replays_the_write_and_the_read_back(fmt, mode):
    """Both kinds of trace, replayed over other rows, slots and tables."""
    from torch.fx.experimental.proxy_tensor import make_fx

    none = [i for i, t in enumerate(_state(BF, fmt, mode, 16, 4)) if t is None]

    def step(*args):
        args = list(args)
        for i in none:
            args.insert(i, None)
        return _step(*args)

    def given(state):
        return [t for t in state if t is not None]

    traces = [make_fx(step)(*given(_state(BF, fmt, mode, 16, 4)))]
    traces.append(torch.jit.trace(step, tuple(given(_state(BF, fmt, mode, 16, 4))), check_trace=False))
    for seed in (5, 6):
        want = _state(BF, fmt, mode, 16, seed)
        _step(*want)
        for trace in traces:
            mine = _state(BF, fmt, mode, 16, seed)
            with torch.jit.optimized_execution(False):  # (torch's fuser has no 8-bit floats)
                trace(*given(mine))
            _check_same(want, mine)


def test_tangents_are_refused():
    k, v, kc, vc, slots, ks, vs, cu, table, starts, y, z = _state(BF, E4M3, "head", 16, 7)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(ks, torch.ones_like(ks))
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.reshape_and_cache(k, v, kc, vc, slots, dual, vs)
        with pytest.raises(NotImplementedError, match="tangent"):
            vb.gather_cache(kc, vc, y, z, cu, table, starts, dual, vs)
        vb.reshape_and_cache(k, v, kc, vc, slots, ks, vs)
        vb.gather_cache(kc, vc, y, z, cu, table, starts, ks, vs)
    assert (y[0] == 7.0).all() and not (y[1:40] == 7.0).any()


@pytest.mark.parametrize("dtype", [BF, HF])
def test_16_bit_caches_in_pinned_memory_of_the_host(dtype):
    k, v, kc, vc, slots, *_ = _state(dtype, dtype, "none", 16, 8)
    vb.reshape_and_cache(k, v, kc, vc, slots)
    host = [torch.zeros(kc.shape, dtype=dtype, pin_memory=True) for _ in range(2)]
    vb.reshape_and_cache(k, v, *host, slots)
    torch.cuda.synchronize()
    assert _equal(host[0], kc.cpu()) and _equal(host[1], vc.cpu()) and kc.any()
    rows = v.cpu().pin_memory()
    host[1].zero_()
    vb.reshape_and_cache(k, rows, *host, slots)
    torch.cuda.synchronize()
    assert _equal(host[1], vc.cpu())
    # memory that the GPU cannot reach, and 8-bit caches, stay refused
    for c in (torch.zeros(kc.shape, dtype=dtype),
              torch.zeros(kc.shape, dtype=torch.uint8, pin_memory=True).view(E4M3)):
        with pytest.raises(ValueError, match="one GPU"):
            vb.reshape_and_cache(k, v, c, c.clone(), slots)


@pytest.mark.parametrize("news", [1, 40, 130])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("zero", ["softmax", "key"])
def test_a_scale_of_zero_under_scores_near_the_largest(zero, d, news):
    """Products of up to 2^127 times a scale of 0: every visible key counts alike."""
    n, hq, hkv = 700, 8, 2
    args = attention_case([n], [news], hq, hkv, d, 16, BF, E4M3, "tensor", seed=15, width=90)
    q, kc, _, _, _, _, ks, vs = args
    q.zero_()
    q[..., 0] = 2.0 ** 126
    codes = torch.zeros(kc.shape)
    codes[..., 0] = torch.tensor([1.5, -1.5])[torch.randint(0, 2, kc.shape[:3])]
    kc.view(torch.uint8).copy_(codes.to(E4M3).view(torch.uint8))
    ks.fill_(0.0 if zero == "key" else 1.0)
    scale = 0.0 if zero == "softmax" else 0.1
    want, size = attention(*args, scale)
    dev = [t.to(DEV) for t in args]
    out = torch.empty(q.shape, dtype=BF, device=DEV)
    assert vb._paged_kernel_takes(*dev[:3], out, *dev[3:])
    vb.paged_decode_attention(*dev[:3], out, *dev[3:6], scale, *dev[6:])
    # (P is off by 2^127 x 2^-149 in its exponent at most: inside bound's fp32 share)
    off = ((out.cpu().double() - want).abs() / bound(want, size, BF)).max().item()
    assert off <= 1.0


@pytest.mark.parametrize("news,d,width,want", [([1, 1, 1], 128, 200, "shared"), ([4, 1, 2], 64, 200, "shared"),
                                               ([1, 2, 1], 256, 200, "shared"),
                                               ([40, 33, 60], 128, 200, "rows merged"),
                                               ([140, 90, 101], 256, 1200, "rows merged")])
@pytest.mark.parametrize("mode", ["slot", "head"])
def test_capture_and_replay_where_keys_are_shared(news, d, width, want, mode):
    """A graph whose call needs a workspace, replayed over lengths that change which
    workgroups (or chunks) share a row, with the same calls made eagerly in between. Two
    graphs of one pool, so that their workspaces may be one memory."""
    hq, hkv, page = 8, 2, 16
    assert path(sum(news), len(news), hq, hkv, d, page, width) == want
    lens = [3000, 700, 1500]
    args = [t.to(DEV) for t in attention_case(lens, news, hq, hkv, d, page, BF, E4M3, mode, seed=21,
                                              width=width)]
    q, kc, vc, cu, used, table, ks, vs = args
    others = [[3000, 700, 1500], [300, 161, 170], [2900, 150, 130], [201, 699, 1499], [1, 0, 1],
              [2048, 160, 1025]]

    def step(out):
        vb.paged_decode_attention(q, kc, vc, out, cu, used, table, 1 / math.sqrt(d), ks, vs)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(torch.empty_like(q))
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = [torch.zeros_like(q) for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], pool=None if i == 0 else graphs[0].pool()):
            step(outs[i])
    for n in others + others[:2]:
        used.copy_(torch.tensor(n))
        q.normal_()
        mine = torch.zeros_like(q)
        step(mine)
        for i in range(2):
            outs[i].zero_()
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert _equal(outs[i], mine), (n, i)
    assert mine.isfinite().all() and mine.any()


def test_many_rows_of_256_of_one_query_head_each():
    news, width = [200, 90, 141], 2500
    assert path(sum(news), 3, 5, 5, 256, 16, width) == "rows merged"
    for mode in ("head", "slot"):
        args = attention_case([1900, 120, 700], news, 5, 5, 256, 16, BF, E4M3, mode, seed=22,
                              width=width)
        want, size = attention(*args, 1 / 16)
        dev = [t.to(DEV) for t in args]
        out = torch.empty(args[0].shape, dtype=BF, device=DEV)
        assert vb._paged_kernel_takes(*dev[:3], out, *dev[3:])
        vb.paged_decode_attention(*dev[:3], out, *dev[3:6], 1 / 16, *dev[6:])
        off = ((out.cpu().double() - want).abs() / bound(want, size, BF)).max().item()
        assert off <= 1.0

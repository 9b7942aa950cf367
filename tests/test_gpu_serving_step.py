"""GPU test of whole serving steps over a 4-bit cache, captured once and replayed: tables,
rotary positions, write, attention and read-back, each against its plain form on what the
one before it gave, with the requests' histories kept by the host."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4
from flashprefill_amd.rotary import Rotary, apply_rotary
from flashprefill_amd.step_tables import build_step_tables
from tests import _int4 as I
from tests import _rotary as Q
from tests import _steps as S
from tests.test_gpu_rotary import bound as rotary_bound

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("R,N,most,dtype,d,page", [(9, 24, 2, BF, 128, 16), (5, 160, 40, FP, 64, 8),
                                                   (3, 600, 250, BF, 64, 32)])
def test_steps_captured_and_replayed(R, N, most, dtype, d, page):
    g = torch.Generator().manual_seed(N)
    hq, hkv, W, scale = 8, 2, 512 // page, d ** -0.5
    P = R * W // 2  # (pages run out)
    spec = Rotary(d // 2, scaling="bands", factor=8.0, trained_positions=64, theta=1e4)
    freq = spec.on("cuda")
    i32, out16 = dict(dtype=torch.int32, device="cuda"), dict(dtype=dtype, device="cuda")
    lens, new, table = torch.zeros(R, **i32), torch.zeros(R, **i32), torch.full((R, W), -1, **i32)
    free = torch.randperm(P, generator=g).to(**i32)
    num_free = torch.tensor([P], **i32)
    cu, granted = torch.empty(R + 1, **i32), torch.empty(R, **i32)
    pos, slots = (torch.empty(N, dtype=torch.int64, device="cuda") for _ in range(2))
    done = torch.zeros(R, dtype=torch.bool, device="cuda")
    qkv = torch.zeros(N, hq + 2 * hkv, d, **out16)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    caches = [i4.int4_cache_views(torch.full((P, page, hkv, i4.int4_row_bytes(d)), 255,
                                             dtype=torch.uint8, device="cuda")) for _ in range(2)]
    (kc, kg), (vc, vg) = caches
    out = torch.zeros(N, hq, d, **out16)
    starts, at = torch.zeros(R, **i32), torch.zeros(R + 1, **i32)
    back = [torch.zeros(R * W * page, hkv, d, **out16) for _ in range(2)]

    def step():
        build_step_tables(lens, new, table, free, num_free, page, cu, pos, slots, granted,
                          finished=done)
        apply_rotary(q, k, pos, freq, amplitude=spec.amplitude)
        i4.reshape_and_cache_int4(k, v, kc, vc, kg, vg, slots)
        i4.paged_decode_attention_int4(q, kc, vc, kg, vg, out, cu, lens, table, scale)
        i4.gather_cache_int4(kc, vc, kg, vg, *back, at, table, starts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (no tokens: changes nothing)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    books = [[0] * R, None, table.tolist(), free.tolist(), P, page, N, None]
    held = [[torch.zeros(0, hkv, d, dtype=dtype) for _ in range(2)] for _ in range(R)]
    checked = 0
    for i in range(10):
        books[1] = [x if z else 0 for x, z in zip(
            torch.randint(1, most + 1, (R,), generator=g).tolist(),
            torch.randint(0, 4, (R,), generator=g).tolist())]
        books[7] = (torch.rand(R, generator=g) < 0.1).tolist()
        x = torch.randn(qkv.shape, generator=g).to(dtype)
        new.copy_(torch.tensor(books[1]))
        done.copy_(torch.tensor(books[7]))
        qkv.copy_(x)
        want = S.tables(*books)
        at[1:].copy_(torch.tensor(want["seq_lens"]).cumsum(0))
        graph.replay()
        torch.cuda.synchronize()
        for name, t in {"cu": cu, "granted": granted, "positions": pos, "slots": slots,
                        "seq_lens": lens, "num_free": num_free, "table": table}.items():
            assert t.tolist() == want[name], (i, name)
        books[0], books[2], books[3], books[4] = (want["seq_lens"], want["table"],
                                                  want["free_pages"], want["num_free"][0])
        y = qkv.cpu()
        turned = Q.rotated(x[:, :hq + hkv], pos.cpu(), freq.cpu(), False, spec.amplitude, False)
        assert ((y[:, :hq + hkv].double() - turned).abs() <= rotary_bound(
            turned, x[:, :hq + hkv], dtype, spec.amplitude)).all()
        assert torch.equal(y[:, hq + hkv:], x[:, hq + hkv:])
        for r in range(R):
            q0, q1 = want["cu"][r], want["cu"][r + 1]
            if books[7][r]:  # (its pages fit: free_pages has room for all there are)
                held[r] = [t[:0] for t in held[r]]
            if want["granted"][r]:
                held[r] = [torch.cat([t, y[q0:q1, h:h + hkv]])
                           for t, h in zip(held[r], (hq, hq + hkv))]
            n = want["seq_lens"][r]
            assert held[r][0].shape[0] == n
            rows = [i4.int4_values(*i4.quantise_int4(t)) for t in held[r]]
            a = int(at[r])
            for t, b in zip(rows, back):
                assert torch.equal(b[a:a + n].cpu(), t.to(dtype)), (i, r)
            if not want["granted"][r] or q0 == q1:
                continue
            kk, vv = (t.double().repeat_interleave(hq // hkv, 1) for t in rows)
            s = torch.einsum("qhd,khd->hqk", y[q0:q1, :hq].double(), kk) * scale
            size = torch.einsum("qhd,khd->hqk", y[q0:q1, :hq].double().abs(), kk.abs()) * scale
            seen = torch.arange(n).view(1, 1, -1) <= torch.arange(n - (q1 - q0), n).view(1, -1, 1)
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            o = torch.einsum("hqk,khd->qhd", p, vv)
            off = (out[q0:q1].cpu().double() - o).abs()
            assert (off <= I.bound(o, torch.einsum("hqk,khd->qhd", p, vv.abs()),
                                   float(size.max()), dtype)).all(), (i, r)
            checked += 1
    assert checked > R

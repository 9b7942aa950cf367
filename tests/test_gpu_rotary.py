"""GPU tests of rotary positions against 64 bits: layouts, parts of the head, strides and
alignments, in place and not, back again, captured, and in a layer."""

import pytest
import torch

from flashprefill_amd.attention_layer import PrefillAttention, fused_rope_qk
from flashprefill_amd.rotary import Rotary, apply_rotary
from tests import _rotary as Q

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def bound(want, x, dtype, amplitude):
    """Half a spacing of the output, and before it cosine and sine to 2^-23 (the reduced
    angle and the function) with the products' and the sum's roundings: 2^-22 of |x| + |y|,
    both at most the row's largest element."""
    eps = 2.0 ** -8 if dtype == BF else 2.0 ** -11
    most = x.double().abs().amax(-1, keepdim=True) * 2 * amplitude
    return want.abs() * eps * 1.01 + most * 2.0 ** -22 + (0 if dtype == BF else 2.0 ** -25)


CASES = [(1, 1, 1, 64, 64), (5, 4, 2, 128, 128), (33, 8, 1, 128, 64), (70, 7, 3, 256, 256),
         (3000, 4, 1, 64, 32), (9, 3, 2, 80, 40), (9, 3, 2, 100, 52), (12, 5, 5, 66, 22),
         (17, 2, 2, 128, 0), (4, 64, 64, 512, 512), (2, 1, 1, 2, 2), (1100, 28, 4, 128, 24)]


@pytest.mark.parametrize("n,hq,hkv,d,rot", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype,index", [(BF, torch.int64), (FP, torch.int32)])
def test_rotary(n, hq, hkv, d, rot, interleaved, dtype, index):
    f = Rotary(rot, theta=5e5).frequencies()
    q, k, pos = Q.rows(n, hq, d, dtype, 1), Q.rows(n, hkv, d, dtype, 2), Q.positions(n, 3, index)
    for inverse, amplitude in ((False, 1.0), (True, 1.3)):
        wants = [Q.rotated(x, pos, f, interleaved, amplitude, inverse) for x in (q, k)]
        # rows of one projection, in place; and into strided outputs
        qkv = torch.cat([q, k, k], 1).cuda()
        a, b = qkv[:, :hq], qkv[:, hq:hq + hkv]
        kw = dict(interleaved=interleaved, amplitude=amplitude, inverse=inverse)
        out = [torch.full((n + 1, 2 * x.shape[1], d + 6), 9.0, dtype=dtype, device="cuda")
               for x in (q, k)]
        views = [o[:n, ::2, 3:3 + d] for o in out]
        apply_rotary(a, b, pos.cuda(), f.cuda(), q_out=views[0], k_out=views[1], **kw)
        apply_rotary(a, b, pos.cuda(), f.cuda(), **kw)
        for x, y, o, view, want in zip((q, k), (a, b), out, views, wants):
            assert ((y.cpu().double() - want).abs() <= bound(want, x, dtype, amplitude)).all()
            assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
            assert torch.equal(view, y)
            view.fill_(9.0)
            assert (o == 9).all()  # nothing else was written
        assert torch.equal(qkv[:, hq + hkv:].cpu(), k)


def test_whole_heads_by_halves_are_the_fused_kernels():
    # the same angles and formula: equal but for cosines' and sines' last bits
    q, k = Q.rows(300, 8, 128, BF, 1).cuda(), Q.rows(300, 2, 128, BF, 2).cuda()
    pos = Q.positions(300).abs().cuda() % 4096
    a, b = q.clone(), k.clone()
    fused_rope_qk(a, b, pos, 1e6, max_position=4096)
    apply_rotary(q, k, pos, Rotary(128, 1e6).on("cuda"))
    for x, y in ((q, a), (k, b)):
        assert (x != y).float().mean() < 0.01
        assert ((x.double() - y.double()).abs() <= 2.0 ** -7 * y.double().abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_there_and_back(interleaved):
    q, pos = Q.rows(200, 4, 128, FP, 1).cuda(), Q.positions(200).cuda()
    f, out, back = Rotary(96).on("cuda"), torch.empty_like(q), torch.empty_like(q)
    apply_rotary(q, None, pos, f, interleaved=interleaved, q_out=out)
    apply_rotary(out, None, pos, f, interleaved=interleaved, inverse=True, q_out=back)
    most = q.double().abs().amax(-1, keepdim=True)
    # a rounding to fp16 of each of a pair, and the last one
    assert ((back.double() - q.double()).abs() <= 4 * 2.0 ** -11 * most).all()


def test_positions_past_32_bits():
    pos = torch.tensor([2 ** 40 + 1, -(2 ** 35), 0, 2 ** 31])
    f = torch.tensor([1.0, 0.5, 1e-7], dtype=torch.float64)
    x = Q.rows(4, 2, 8, BF)
    y = x.cuda()
    apply_rotary(y, None, pos.cuda(), f.cuda())
    want = Q.rotated(x, pos, f, False, 1.0, False)
    # (an angle of 2^40 is itself off by 2^-13 in 64 bits, on both sides alike)
    assert ((y.cpu().double() - want).abs() <= bound(want, x, BF, 1.0) + 2.0 ** -12).all()


def test_outputs_that_lie_in_an_input():
    x = torch.ones(4, 4, 64, dtype=BF, device="cuda")
    f, pos = Rotary(64).on("cuda"), torch.arange(4, device="cuda")
    with pytest.raises(ValueError, match="memory"):
        apply_rotary(x[:, :2], x[:, 2:], pos, f, q_out=x[:, 2:], k_out=torch.empty_like(x[:, 2:]))
    with pytest.raises(ValueError, match="memory"):
        apply_rotary(x[:3], None, pos[:3], f, q_out=x[1:])
    with pytest.raises(RuntimeError):
        apply_rotary(x, None, pos, f, q_out=x[:, :1].expand(4, 4, 64))
    with pytest.raises(ValueError, match="own"):
        apply_rotary(x, x, pos, f)
    out = torch.empty_like(x)
    with pytest.raises(ValueError, match="own"):
        apply_rotary(x[:, :2], x[:, 2:], pos, f, q_out=out[:, :2], k_out=out[:, :2])
    apply_rotary(x[:0], None, pos[:0], f)


def test_frequencies_on_the_current_device():
    spec = Rotary(64, theta=54321.0)
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            spec.on("cuda")
        x += 1
    f = spec.on("cuda")
    assert spec.on(f.device) is f and f.device.index == torch.cuda.current_device()
    graph.replay()
    torch.cuda.synchronize()
    assert x.item() == 1


def test_capture_and_replay():
    q, pos = Q.rows(40, 4, 128, BF, 1).cuda(), Q.positions(40).cuda()
    f, out = Rotary(64, scaling="yarn", factor=4.0, trained_positions=4096), torch.empty_like(q)
    fd = f.on("cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        apply_rotary(q, None, pos, fd, amplitude=f.amplitude, q_out=out)
    for seed in range(3):
        q.copy_(Q.rows(40, 4, 128, BF, seed + 5))
        pos.copy_(Q.positions(40, seed))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(q)
        apply_rotary(q, None, pos, fd, amplitude=f.amplitude, q_out=want)
        assert torch.equal(out, want)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_a_layer_with_rotary_positions(qk_norm):
    x = torch.randn(700, 256, generator=torch.Generator().manual_seed(0)).to(BF)
    cu = torch.tensor([0, 300, 700], dtype=torch.int32)
    spec = Rotary(64, interleaved=True, scaling="bands", factor=8.0, trained_positions=512)
    args = dict(num_q_heads=4, num_kv_heads=2, head_dim=128, qk_norm=qk_norm, seed=1, dtype=BF)
    layer = PrefillAttention(256, **args, device="cuda", rotary=spec)
    bare = PrefillAttention(256, **args, device="cuda", rotary=Rotary(0))
    q, k, v = layer.project_qkv(x.cuda(), cu.cuda())
    q0, k0, v0 = bare.project_qkv(x.cuda(), cu.cuda())
    pos = torch.cat([torch.arange(300), torch.arange(400)])
    for a, b in ((q, q0), (k, k0)):
        want = Q.rotated(b.cpu(), pos, spec.frequencies(), True, 1.0, False)
        assert ((a.cpu().double() - want).abs() <= bound(want, b.cpu(), BF, 1.0)).all()
    assert torch.equal(v, v0)
    assert layer(x.cuda(), cu.cuda(), 400).isfinite().all()

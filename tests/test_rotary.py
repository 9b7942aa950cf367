"""CPU tests of rotary positions: frequencies against their formulas, the composition
against a rotation pair by pair in 64 bits, and what the entry points refuse."""

import ctypes
import math

import pytest
import torch

from flashprefill_amd import _lib
from flashprefill_amd.attention_layer import PrefillAttention
from flashprefill_amd.rotary import Rotary, apply_rotary, apply_rotary_reference
from tests import _rotary as Q


def test_frequencies_and_linear_scaling():
    f = Rotary(64, theta=5e5).frequencies()
    for i in range(32):
        assert math.isclose(float(f[i]), 5e5 ** (-2 * i / 64), rel_tol=1e-14)
    assert torch.equal(Rotary(64, 5e5, scaling="linear", factor=4.0).frequencies(), f / 4)
    assert Rotary(0).frequencies().numel() == 0 and Rotary(2).frequencies().tolist() == [1.0]


def test_ntk_keeps_the_fastest_and_slows_the_slowest():
    f, s = Rotary(128).frequencies(), Rotary(128, scaling="ntk", factor=8.0).frequencies()
    assert float(s[0]) == 1.0 and math.isclose(float(s[-1]), float(f[-1]) / 8, rel_tol=1e-12)


def test_yarn():
    r = Rotary(128, 1e4, scaling="yarn", factor=16.0, trained_positions=4096)
    f, s = Rotary(128, 1e4).frequencies(), r.frequencies()
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(s[turns > 40], f[turns > 40])
    assert torch.allclose(s[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-12)
    low = math.floor(128 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(1e4)))
    high = math.ceil(128 * math.log(4096 / (2 * math.pi)) / (2 * math.log(1e4)))
    i = (low + high) // 2
    w = (i - low) / (high - low)
    assert math.isclose(float(s[i]), float(f[i]) * (w / 16 + 1 - w), rel_tol=1e-12)
    assert math.isclose(r.amplitude, 0.1 * math.log(16) + 1)
    assert Rotary(128, scaling="yarn", trained_positions=10).amplitude == 1.0
    assert Rotary(128, attention_factor=0.5).amplitude == 0.5


def test_bands():
    r = Rotary(128, 5e5, scaling="bands", factor=8.0, trained_positions=8192)
    f, s = Rotary(128, 5e5).frequencies(), r.frequencies()
    for a, b in zip(f.tolist(), s.tolist()):
        wave = 2 * math.pi / a
        if wave < 8192 / 4:
            assert b == a
        elif wave > 8192:
            assert math.isclose(b, a / 8, rel_tol=1e-12)
        else:
            keep = (8192 / wave - 1) / 3
            assert math.isclose(b, (1 - keep) * a / 8 + keep * a, rel_tol=1e-12)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=-2), dict(scaling="other"),
                                dict(theta=0.0), dict(factor=0.0), dict(scaling="yarn"),
                                dict(scaling="bands"), dict(rotary_dim=2, scaling="ntk"),
                                dict(scaling="yarn", trained_positions=9, theta=1.0),
                                dict(scaling="yarn", trained_positions=9, beta_slow=40.0),
                                dict(scaling="bands", trained_positions=9, low_freq=4.0)])
def test_specs_that_do_not_fit(kw):
    with pytest.raises(ValueError):
        Rotary(**dict(dict(rotary_dim=64), **kw))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_the_composition(interleaved, inverse):
    x, pos, f = Q.rows(9, 3, 40, torch.float32), Q.positions(9), Rotary(24).frequencies()
    y = torch.empty_like(x)
    apply_rotary_reference(x, None, pos, f, interleaved=interleaved, amplitude=1.25,
                           inverse=inverse, q_out=y)
    want = Q.rotated(x, pos, f, interleaved, 1.25, inverse)
    # three roundings of fp32 and those of cosine and sine, of |x| + |y| times 1.25
    assert (y.double() - want).abs().max() <= 6 * 2.0 ** -24 * 2.5 * float(x.abs().max())


def test_a_layer_with_rotary_positions_on_the_cpu():
    x, cu = torch.randn(12, 32), torch.tensor([0, 5, 12], dtype=torch.int32)
    spec = Rotary(16, interleaved=True, scaling="linear", factor=2.0)
    layer = PrefillAttention(32, 4, 2, 32, dtype=torch.float32, qk_norm=True, rotary=spec)
    q, k, v = layer.project_qkv(x, cu)
    plain = PrefillAttention(32, 4, 2, 32, dtype=torch.float32, qk_norm=True, rotary=Rotary(0))
    q0, k0, v0 = plain.project_qkv(x, cu)
    pos = torch.tensor([0, 1, 2, 3, 4, 0, 1, 2, 3, 4, 5, 6])
    for a, b in ((q, q0), (k, k0)):
        assert (a.double() - Q.rotated(b, pos, spec.frequencies(), True, 1.0, False)).abs().max() < 1e-5
    assert torch.equal(v, v0)
    with pytest.raises(ValueError, match="rotary_dim"):
        PrefillAttention(32, 4, 2, 32, rotary=Rotary(64))


def _call(**kw):
    x = torch.ones(4, 2, 64, dtype=torch.bfloat16)
    a = dict(q=x, k=x.clone(), positions=torch.arange(4), frequencies=Rotary(64).frequencies())
    return dict(a, **kw)


@pytest.mark.parametrize("kw,error", [
    (dict(q=torch.ones(4, 2, 64)), NotImplementedError),
    (dict(k=torch.ones(4, 2, 64, dtype=torch.float16)), ValueError),
    (dict(k=torch.ones(3, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=torch.ones(4, 2, 32, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.ones(4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.ones(4, 2, 128, dtype=torch.bfloat16)[..., ::2]), ValueError),
    (dict(q_out=torch.ones(4, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(k=None, k_out=torch.ones(4, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(positions=torch.arange(5)), ValueError), (dict(positions=torch.ones(4)), ValueError),
    (dict(frequencies=torch.ones(32)), ValueError),
    (dict(frequencies=torch.ones(33, dtype=torch.float64)), ValueError),
    (dict(q=torch.ones(4, 2, 64, dtype=torch.bfloat16, requires_grad=True)), RuntimeError),
    (dict(), ValueError)])  # the CPU
def test_what_is_refused(kw, error):
    with pytest.raises(error):
        apply_rotary(**_call(**kw))


def _args(**kw):
    a = _lib.FpRotaryArgs()
    for f in ("q", "k", "q_out", "k_out", "positions", "frequencies"):
        setattr(a, f, 0x10000)
    a.num_tokens, a.num_pairs, a.num_q_heads, a.num_kv_heads, a.head_dim = 4, 32, 4, 2, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=_lib.FP_DTYPE_F32), _lib.FP_E_UNSUPPORTED),
    (dict(head_dim=63), _lib.FP_E_INVALID_ARG), (dict(num_pairs=33), _lib.FP_E_INVALID_ARG),
    (dict(num_tokens=-1), _lib.FP_E_INVALID_ARG), (dict(q=0), _lib.FP_E_INVALID_ARG),
    (dict(k_out=0), _lib.FP_E_INVALID_ARG), (dict(positions=0), _lib.FP_E_INVALID_ARG),
    (dict(frequencies=0), _lib.FP_E_INVALID_ARG), (dict(head_dim=1026), _lib.FP_E_UNSUPPORTED),
    (dict(num_tokens=1 << 24), _lib.FP_E_UNSUPPORTED),
    (dict(num_q_heads=1 << 15, head_dim=66, q_stride_tok=1), _lib.FP_E_UNSUPPORTED)])
def test_the_c_entry_refuses(kw, code):
    assert _lib.load().fp_rotary(ctypes.byref(_args(**kw)), None) == code
    assert _lib.load().fp_rotary(None, None) == _lib.FP_E_INVALID_ARG


def test_frequencies_made_in_a_dispatch_or_inference_mode():
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    spec = Rotary(64, theta=12345.0)
    with FakeTensorMode():
        assert isinstance(spec.on("cpu"), FakeTensor)
    with torch.inference_mode():
        got = spec.on("cpu")
    assert not isinstance(got, FakeTensor) and not got.is_inference()
    assert torch.equal(got, spec.frequencies()) and spec.on(torch.device("cpu")) is got


@pytest.mark.parametrize("own", [False, True])
def test_a_trace_sees_torch_operations(own):
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(q, k, pos, f):
        out = dict(q_out=torch.empty_like(q), k_out=torch.empty_like(k)) if own else {}
        apply_rotary(q, k, pos, f, **out)
        return out.get("q_out", q)

    with FakeTensorMode():
        q, k = (torch.empty(4, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2))
        pos, f = torch.arange(4, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
        ops = [str(n.target) for n in make_fx(step)(q, k, pos, f).graph.nodes]
    assert any("cos" in op for op in ops) and any("copy_" in op for op in ops)

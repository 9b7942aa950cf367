"""CPU tests of the gradients through a layer with rotary positions."""

import math

import pytest
import torch

from flashprefill_amd.attention_layer import PrefillAttention
from flashprefill_amd.rotary import Rotary, rotated
from tests import _rotary as Q

SPECS = [Rotary(32), Rotary(16, interleaved=True, scaling="linear", factor=2.0),
         Rotary(32, scaling="yarn", factor=8.0, trained_positions=64), Rotary(0)]


def _setup(spec, qk_norm):
    g = torch.Generator().manual_seed(5)
    layer = PrefillAttention(24, 4, 2, 32, dtype=torch.float32, qk_norm=qk_norm, rotary=spec,
                             rope_theta=1e4)
    layer.q_norm.data = 1 + 0.2 * torch.randn(32, generator=g)
    layer.k_norm.data = 1 + 0.2 * torch.randn(32, generator=g)
    x = torch.randn(12, 24, generator=g)
    w = [torch.randn(12, h, 32, generator=g) for h in (4, 2, 2)]
    return layer, x, torch.tensor([0, 5, 12], dtype=torch.int32), w


def _loss(layer, x, cu, w):
    return sum((y * z).sum() for y, z in zip(layer.project_qkv(x, cu), w))


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("spec", SPECS, ids=lambda s: f"{s.rotary_dim}-{s.scaling}")
def test_the_gradient_of_a_layer(spec, qk_norm):
    """Against the formula in 64 bits: the weights turned back (their rotation's transpose),
    then the norms' derivative, then the projection's; and against differences."""
    layer, x, cu, w = _setup(spec, qk_norm)
    x.requires_grad_()
    layer.w_qkv.requires_grad_()
    _loss(layer, x, cu, w).backward()
    pos = torch.tensor([0, 1, 2, 3, 4, 0, 1, 2, 3, 4, 5, 6])
    x64, w64 = x.detach().double(), layer.w_qkv.detach().double()
    qkv = (x64 @ w64.t()).view(12, 8, 32)
    g = [Q.rotated(y.double(), pos, spec.frequencies(), spec.interleaved, spec.amplitude, True)
         if i < 2 else y.double() for i, y in enumerate(w)]
    # (dims that do not turn keep their size, the others carry the amplitude)
    if qk_norm:
        for i, (y, norm) in enumerate(((qkv[:, :4], layer.q_norm), (qkv[:, 4:6], layer.k_norm))):
            r = (y.pow(2).mean(-1, keepdim=True) + layer.rms_eps).rsqrt()
            gn = g[i] * norm.detach().double()
            g[i] = r * gn - y * r ** 3 * (gn * y).mean(-1, keepdim=True)
    g = torch.cat(g, 1).view(12, 8 * 32)
    # fp32: factors within 2^-20, sums of at most 256 products within 2^-16 of their sizes, of
    # which the norms' difference is at most 8 times the result's largest
    for got, want, size in ((x.grad, g @ w64, g.abs() @ w64.abs()),
                            (layer.w_qkv.grad, g.t() @ x64, g.t().abs() @ x64.abs())):
        assert ((got.double() - want).abs() <= 2.0 ** -13 * (size + size.max() / 8)).all()
    # differences along a direction: of second order, h^2 of third derivatives that are below
    # 100 |loss|, and 2^-20 of sums of 96 rows' terms over h
    step = torch.randn(12, 24, generator=torch.Generator().manual_seed(1))
    h = 2.0 ** -6
    with torch.no_grad():
        rise = (_loss(layer, x + h * step, cu, w).double() -
                _loss(layer, x - h * step, cu, w).double()) / (2 * h)
    slope = float((x.grad * step).double().sum())
    assert abs(float(rise) - slope) <= 0.02 * float((x.grad * step).double().abs().sum())


def test_whole_heads_by_halves_have_the_gradient_of_the_layer_without_the_option():
    """(theta 1e4: what ``rotary=None`` turns by)"""
    grads = []
    for spec in (Rotary(32, theta=1e4), None):
        layer, x, cu, w = _setup(spec, False)
        x.requires_grad_()
        _loss(layer, x, cu, w).backward()
        grads.append(x.grad.double())
    size = grads[1].abs().max()
    assert (grads[0] - grads[1]).abs().max() <= 2.0 ** -18 * size * math.sqrt(256)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_the_gradient_of_a_rotation(interleaved, inverse):
    """A rotation's derivative turns the other way, by the same amplitude."""
    x, pos, f = Q.rows(9, 3, 40, torch.float32).requires_grad_(), Q.positions(9), \
        Rotary(24).frequencies()
    w = Q.rows(9, 3, 40, torch.float32, 1)
    (rotated(x, pos, f, interleaved=interleaved, amplitude=1.25, inverse=inverse) * w).sum().backward()
    want = Q.rotated(w, pos, f, interleaved, 1.25, not inverse)
    # three roundings of fp32 and those of cosine and sine, of |x| + |y| times 1.25
    assert (x.grad.double() - want).abs().max() <= 6 * 2.0 ** -24 * 2.5 * float(w.abs().max())

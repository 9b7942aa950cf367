"""GPU tests of gradients through a layer with rotary positions: in fp32 those of the CPU
(which are checked there), in 16 bits, where one kernel rotates in place, refused."""

import pytest
import torch

from flashprefill_amd.attention_layer import PrefillAttention
from flashprefill_amd.rotary import Rotary

pytestmark = pytest.mark.gpu
CU = torch.tensor([0, 5, 12], dtype=torch.int32)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_fp32(qk_norm):
    spec = Rotary(16, interleaved=True, scaling="linear", factor=2.0)
    x = torch.randn(12, 24, generator=torch.Generator().manual_seed(1))
    w = torch.randn(12, 8, 32, generator=torch.Generator().manual_seed(2))
    grads = []
    for dev in ("cpu", "cuda"):
        layer = PrefillAttention(24, 4, 2, 32, dtype=torch.float32, qk_norm=qk_norm, rotary=spec,
                                 device=dev)
        y = x.clone().to(dev).requires_grad_()
        (torch.cat(layer.project_qkv(y, CU.to(dev)), 1) * w.to(dev)).sum().backward()
        grads.append(y.grad.cpu().double())
    # sums of 256 products whose factors fp32 holds to 2^-20 or better; sizes up to 8 times
    # the largest sum
    assert (grads[0] - grads[1]).abs().max() <= 2.0 ** -16 * 8 * grads[0].abs().max()


def test_16_bits():
    layer = PrefillAttention(64, 4, 2, 64, rotary=Rotary(64), device="cuda")
    x = torch.randn(12, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        layer.project_qkv(x, CU.cuda())
    with torch.no_grad():
        layer.project_qkv(x, CU.cuda())

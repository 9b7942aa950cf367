"""Rotary positions of any layout: pairs of a head's halves or side by side, part of the
head, and frequencies scaled for contexts longer than the trained one (``fp_rotary``).

``attention_layer.fused_rope_qk`` rotates whole heads by halves from a table of cosines and
norms them first; ``apply_rotary`` needs no table: it forms a token's angles in 64 bits where
it rotates its heads.

The scalings, f_i = theta^(-2 i / r) being the trained frequencies of the r rotated dims, F the
factor and L the trained positions:

* ``linear``: f_i / F (Chen et al. 2023, position interpolation);
* ``ntk``: theta F^(r / (r - 2)) in place of theta, so that the slowest pair turns F times
  slower and the fastest as trained;
* ``yarn`` (Peng et al. 2023): f_i / F where a pair makes less than ``beta_slow`` turns over L
  positions, f_i above ``beta_fast``, a ramp over i between, and cosines and sines times
  0.1 ln F + 1;
* ``bands``: f_i / F for wavelengths above L / ``low_freq``, f_i below L / ``high_freq``, and
  between the two weighted by where the number of turns L f_i / 2 pi lies.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Dict, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from . import vllm_backend as vb

_SCALINGS = ("none", "linear", "ntk", "yarn", "bands")
_ON_DEVICE: Dict[Tuple["Rotary", torch.device], torch.Tensor] = {}


@dataclass(frozen=True)
class Rotary:
    """How positions turn a head's first ``rotary_dim`` dims."""
    rotary_dim: int
    theta: float = 1e4
    interleaved: bool = False
    scaling: str = "none"
    factor: float = 1.0
    trained_positions: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    low_freq: float = 1.0
    high_freq: float = 4.0
    attention_factor: Optional[float] = None

    def __post_init__(self):
        if self.rotary_dim < 0 or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even, got {self.rotary_dim}")
        if self.scaling not in _SCALINGS:
            raise ValueError(f"scaling {self.scaling!r} is none of {_SCALINGS}")
        if self.theta <= 0 or self.factor <= 0:
            raise ValueError("theta and factor must be positive")
        if self.scaling == "ntk" and self.rotary_dim <= 2:
            raise ValueError("ntk scaling needs more than one pair")
        if self.scaling in ("yarn", "bands"):
            if self.trained_positions < 1:
                raise ValueError(f"{self.scaling} scaling needs trained_positions")
            if self.scaling == "yarn" and not (self.theta != 1 and
                                               self.beta_fast >= self.beta_slow > 0):
                raise ValueError("yarn scaling needs theta != 1 and beta_fast >= beta_slow > 0")
            if self.scaling == "bands" and not self.high_freq > self.low_freq > 0:
                raise ValueError("bands scaling needs high_freq > low_freq > 0")

    @property
    def amplitude(self) -> float:
        """The factor of cosines and sines."""
        if self.attention_factor is not None:
            return self.attention_factor
        return 0.1 * math.log(self.factor) + 1.0 if self.scaling == "yarn" and self.factor > 1 \
            else 1.0

    def frequencies(self) -> torch.Tensor:
        """Angles per position of the pairs, fp64 on the CPU."""
        r = self.rotary_dim
        i = torch.arange(r // 2, dtype=torch.float64)
        theta = self.theta * self.factor ** (r / (r - 2)) if self.scaling == "ntk" else self.theta
        f = theta ** (-2 * i / r) if r else i
        if self.scaling == "linear":
            return f / self.factor
        if self.scaling == "yarn":
            low, high = (r * math.log(self.trained_positions / (turns * 2 * math.pi)) /
                         (2 * math.log(theta)) for turns in (self.beta_fast, self.beta_slow))
            low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
            ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
            return f / self.factor * ramp + f * (1 - ramp)
        if self.scaling == "bands":
            turns = self.trained_positions * f / (2 * math.pi)
            keep = ((turns - self.low_freq) / (self.high_freq - self.low_freq)).clamp(0, 1)
            return f / self.factor * (1 - keep) + f * keep
        return f

    def on(self, device) -> torch.Tensor:
        """``frequencies()`` on a device, made once: before a captured graph reads them.
        (A trace or a dispatch mode gets its own, which nothing after it could use.)"""
        if vb._torch_only():
            return self.frequencies().to(device)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        hit = _ON_DEVICE.get((self, device))
        if hit is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"{self} is not on {device} yet: call on() before the capture")
            with torch.inference_mode(False):
                hit = _ON_DEVICE[self, device] = self.frequencies().to(device)
        return hit


def _check_rows(name: str, x: torch.Tensor, out: torch.Tensor, tokens: int, dtype) -> None:
    if x.dim() != 3 or out.shape != x.shape or x.shape[0] != tokens:
        raise ValueError(f"{name} must be ({tokens} tokens, heads, head_dim) and its output "
                         f"alike, got {tuple(x.shape)} and {tuple(out.shape)}")
    if x.dtype != dtype or out.dtype != dtype:
        raise ValueError(f"{name} and its output must be {dtype}, got {x.dtype} and {out.dtype}")
    if (x.shape[2] > 1 and (x.stride(2) != 1 or out.stride(2) != 1)):
        raise ValueError(f"{name} and its output must have a contiguous head dimension")


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                 frequencies: torch.Tensor, *, interleaved: bool = False, amplitude: float = 1.0,
                 inverse: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None) -> None:
    """Rotate q (tokens, Hq, d) and k (tokens, Hkv, d; or None) in bf16 or fp16 on the GPU,
    in place or into ``q_out`` / ``k_out``, on the current stream.

    ``positions`` (tokens,) int32 or int64, of any sign; ``frequencies`` (n,) fp64
    (``Rotary.on``): the first 2 n dims of a head are n pairs, dims i and n + i or,
    ``interleaved``, 2 i and 2 i + 1, which turn by positions[t] * frequencies[i], times
    ``amplitude``; the others stay. ``inverse`` turns back (for ``amplitude`` 1 also the
    gradient's way). Outputs are the inputs themselves or memory of their own.

    Strides of tokens and heads are free; those, head dims and numbers of pairs that are
    multiples of 8 move 16 bytes at a time. No derivative is recorded: inputs that require
    one are refused, forward-mode tangents too. Under a trace or a dispatch mode the rotation
    is made of torch operations."""
    tokens, dev, dtype = q.shape[0], q.device, q.dtype
    if dtype not in vb._DTYPES:
        raise NotImplementedError(f"apply_rotary supports bf16 and fp16, got {dtype}")
    q_out, k_out = q if q_out is None else q_out, k if k_out is None else k_out
    if (k is None) != (k_out is None):
        raise ValueError("k_out without k")
    pairs = [("q", q, q_out)] if k is None else [("q", q, q_out), ("k", k, k_out)]
    for name, x, out in pairs:
        _check_rows(name, x, out, tokens, dtype)
    d, n = q.shape[2], frequencies.numel()
    if k is not None and k.shape[2] != d:
        raise ValueError(f"head dims of q and k differ: {d} and {k.shape[2]}")
    if positions.dim() != 1 or positions.numel() != tokens or positions.dtype not in vb._INDEX:
        raise ValueError(f"positions must be int32 or int64 ({tokens},), got {positions.dtype} "
                         f"{tuple(positions.shape)}")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or 2 * n > d:
        raise ValueError(f"frequencies must be float64 and at most {d // 2}, got "
                         f"{frequencies.dtype} {tuple(frequencies.shape)}")
    tensors = [t for _, x, out in pairs for t in (x, out)]
    if forward_ad._current_level >= 0:
        vb._check_no_tangents(*tensors)
    if not vb._none_requires_grad(*tensors):
        raise RuntimeError("q or k requires a gradient, which apply_rotary does not record: use "
                           "torch.no_grad()")
    for t in (*tensors, positions, frequencies):
        if t.device != dev or dev.type != "cuda":
            raise ValueError("q, k, positions and frequencies must be on one GPU")
    outs = tensors[1::2]
    vb._check_written(*outs)
    torch_only = vb._torch_only()
    if k is not None and q_out.numel() and k_out.numel() and \
            vb._place(q_out, torch_only) == vb._place(k_out, torch_only):
        raise ValueError("the outputs of q and k must be memory of their own")
    stores = None
    for _, x, out in pairs:  # its own input, or no input's memory
        if out is x or (vb._place(out, torch_only) == vb._place(x, torch_only) and
                        out.stride() == x.stride()):
            continue
        if stores is None:
            stores = [y.untyped_storage()._cdata for y in tensors[::2]]
        if out.untyped_storage()._cdata in stores:
            raise ValueError("outputs must be the inputs themselves or memory of their own")
    if torch_only:
        apply_rotary_reference(q, k, positions, frequencies, interleaved=interleaved,
                               amplitude=amplitude, inverse=inverse, q_out=q_out, k_out=k_out)
        return
    positions, frequencies = positions.contiguous(), frequencies.contiguous()
    kk, ko = (q, q_out) if k is None else (k, k_out)
    a = _lib.FpRotaryArgs(
        q.data_ptr(), kk.data_ptr(), q_out.data_ptr(), ko.data_ptr(), *q.stride()[:2],
        *kk.stride()[:2], *q_out.stride()[:2], *ko.stride()[:2], positions.data_ptr(),
        frequencies.data_ptr(), tokens, positions.dtype == torch.int64, n, q.shape[1],
        0 if k is None else k.shape[1], d, vb._DTYPES[dtype], interleaved, inverse, amplitude)
    vb._launch(dev, _lib.load().fp_rotary, ctypes.byref(a))
    torch.autograd.graph.increment_version(outs)


def rotated(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
            interleaved: bool = False, amplitude: float = 1.0, inverse: bool = False
            ) -> torch.Tensor:
    """Rows x (tokens, heads, d) as ``apply_rotary`` turns them, in a tensor of its own, of
    torch operations that record a derivative: angles in 64 bits, cosines and sines and the
    rotation in 32, rounded once."""
    angle = positions.double().view(-1, 1) * frequencies.to(positions.device)
    cos, sin = ((f(angle) * amplitude).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    n = frequencies.numel()
    z = x.float()
    part = z[..., :2 * n]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    u, v = a * cos - b * sin, b * cos + a * sin
    part = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([part, z[..., 2 * n:]], -1).to(x.dtype)


@torch.no_grad()
def apply_rotary_reference(q, k, positions, frequencies, *, interleaved=False, amplitude=1.0,
                           inverse=False, q_out=None, k_out=None) -> None:
    """The torch composition of ``apply_rotary``, in place or into the outputs as there."""
    for x, out in ((q, q_out), (k, k_out)):
        if x is not None:
            (x if out is None else out).copy_(
                rotated(x, positions, frequencies, interleaved=interleaved, amplitude=amplitude,
                        inverse=inverse))

"""Paged KV caches of 4-bit integers: their write, attention over them and their
read-back, the 4-bit forms of ``vllm_backend``'s operators, with HIP kernels behind
``fp_kv_cache_write_int4``, ``fp_paged_attention_int4`` and ``fp_kv_cache_gather_int4``.

A cache of pages of ``block_size`` tokens is two tensors:

* codes, uint8 ``(num_blocks, block_size, Hkv, d / 2)``: byte ``m (d / 32) + j`` of a
  row (m < 16) holds those of dims ``32 j + 2 m`` (low half) and ``32 j + 2 m + 1``;
* group words, int16 ``(num_blocks, Hkv, block_size, d / 32)``: word j of a row serves
  its dims ``32 j .. 32 j + 31``. Its bits 7 .. 14 are those of a fp16 number s with 4
  significant bits, its seven lowest z + 64.

Code c stands for ``s (c + z) t``, t the fixed fp32 scale of the KV head (one value, one
per KV head, or None: 1). A group's step ``s`` and zero point ``z`` follow from its smallest
and largest element: 9/16 of a byte for each element. Elements are off by up to half a step,
about half of a 15th of the group's range (an 8-bit float by up to a 16th of the element); where
the step was rounded down, the group's last ones, which the 16 codes then do not reach, by up
to one and a half. (Of projections' rows one group in six has an element off by more than half a
step, in all 0.6 % of the elements. A step rounded up would reach them and be off by more on
the average.) ``int4_cache_views`` gives both as views of the pages of one tensor of bytes.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from . import vllm_backend as vb

GROUP = 32  # elements that share a word
_MOST = 16384.0  # the largest magnitude that a group holds
_HEAD_DIMS = (64, 128, 256)


def int4_row_bytes(head_dim: int) -> int:
    """Bytes of a cached row: codes and group words."""
    if head_dim not in _HEAD_DIMS:
        raise NotImplementedError(f"4-bit caches: head_dim {head_dim} unsupported "
                                  f"({', '.join(map(str, _HEAD_DIMS))})")
    return head_dim // 2 + head_dim // 16


def int4_cache_views(cache: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and group words in a cache of bytes ``(num_blocks, block_size, Hkv,
    int4_row_bytes(d))`` (uint8), as an engine allocates it for its pages: each page
    holds its codes and, behind them, its group words. The views share its memory."""
    if cache.dtype != torch.uint8 or cache.dim() != 4:
        raise ValueError(f"a 4-bit cache is uint8 (num_blocks, block_size, Hkv, row bytes), got "
                         f"{cache.dtype} {tuple(cache.shape)}")
    nb, bs, hkv, row = cache.shape
    d = row * 16 // 9
    if d not in _HEAD_DIMS or int4_row_bytes(d) != row:
        raise ValueError(f"rows of {row} bytes: int4_row_bytes(head_dim) are "
                         f"{[int4_row_bytes(x) for x in _HEAD_DIMS]}")
    if any(size > 1 and stride != want for size, stride, want in
           zip(cache.shape[1:], cache.stride()[1:], (hkv * row, row, 1))):
        raise ValueError("the pages of a 4-bit cache must be contiguous")
    n = bs * hkv * (d // 2)
    pages = cache.view(nb, bs * hkv * row)
    return (pages[:, :n].view(nb, bs, hkv, d // 2),
            pages[:, n:].view(torch.int16).view(nb, hkv, bs, d // GROUP))


def _check_cache(key_cache, value_cache, key_groups, value_groups, k_scale, v_scale) -> int:
    """Refuse caches, group words and scales that do not fit each other; the head_dim."""
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if t.dtype != torch.uint8:
            raise NotImplementedError(f"{name}: a 4-bit cache is uint8, got {t.dtype}")
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape:
        raise ValueError("caches must be (num_blocks, block_size, num_kv_heads, head_dim / 2)")
    nb, bs, hkv, half = key_cache.shape
    d = 2 * half
    if d not in _HEAD_DIMS:
        raise NotImplementedError(f"4-bit caches: head_dim {d} unsupported "
                                  f"({', '.join(map(str, _HEAD_DIMS))})")
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have contiguous rows")
    for name, g in (("key_groups", key_groups), ("value_groups", value_groups)):
        if g.dtype != torch.int16 or g.shape != (nb, hkv, bs, d // GROUP) or \
                g.device != key_cache.device or g.stride(3) != 1 or \
                (bs > 1 and g.stride(2) != d // GROUP):
            raise ValueError(f"{name} must be int16 (num_blocks, num_kv_heads, block_size, "
                             f"head_dim / 32) = {(nb, hkv, bs, d // GROUP)} on the caches' "
                             f"device, slots contiguous; got {g.dtype} {tuple(g.shape)}")
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is None:
            continue
        if s.dtype != torch.float32:
            raise ValueError(f"{name} must be float32, got {s.dtype}")
        if s.dim() > 1 or s.numel() not in (1, hkv):
            raise ValueError(f"{name} must hold 1 or {hkv} values, got {tuple(s.shape)}")
    return d


def _check_rows(key, value, hkv: int, d: int, what: str) -> None:
    if key.dtype not in vb._DTYPES or value.dtype != key.dtype:
        raise NotImplementedError(f"{what} supports bf16 / fp16 rows, got key {key.dtype}, value "
                                  f"{value.dtype}")
    for name, t in (("key", key), ("value", value)):
        if t.dim() != 3 or t.shape[1:] != (hkv, d):
            raise ValueError(f"{name} {tuple(t.shape)} does not match the cache's "
                             f"{hkv} heads of {d}")
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous head dimension")


def _groups(g: torch.Tensor) -> _lib.FpKvGroups:
    return _lib.FpKvGroups(g.data_ptr(), *g.stride()[:2])


def _cache_args(key, value, key_cache, value_cache, key_groups, value_groups, slots, n, d,
                k_scale, v_scale):
    """``fp_kv_cache_int4_args``, and the tensors whose memory they name."""
    nb, bs, hkv, _ = key_cache.shape
    base = _lib.FpKvCacheArgs(key.data_ptr(), value.data_ptr(), *key.stride()[:2],
                              *value.stride()[:2], key_cache.data_ptr(), value_cache.data_ptr(),
                              *key_cache.stride()[:3], *value_cache.stride()[:3], slots, n, nb,
                              bs, hkv, d, vb._DTYPES[key.dtype])
    (ks, k_keep), (vs, v_keep) = (vb._scale_args(s, key.device) for s in (k_scale, v_scale))
    return _lib.FpKvCacheInt4Args(base, _groups(key_groups), _groups(value_groups), ks, vs), \
        (k_keep, v_keep)


def reshape_and_cache_int4(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                           value_cache: torch.Tensor, key_groups: torch.Tensor,
                           value_groups: torch.Tensor, slot_mapping: torch.Tensor,
                           k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None) -> None:
    """Write key / value (tokens, Hkv, d) in bf16 or fp16 into 4-bit paged caches at
    ``slot_mapping``, as ``reshape_and_cache`` does into others: one slot per token, the
    mapping's length is the number of tokens written, negative slots (and those past the
    cache) are skipped.

    With x' = x / t (t: the fixed scale) within +-16384, infinities too, and lo and hi a group's smallest and largest x', every rounding to
    nearest even:

    * s = max((hi - lo) / 15, hi / 56, -lo / 56) to 4 significant bits (below 2^-14 to a
      multiple of 2^-17, of which 0 stands for a group of zeros);
    * z = lo / s, within -64 .. 63, and c = x' / s - z, within 0 .. 15.

    A NaN makes its group NaN. Slots named by two tokens hold either row, or parts of
    both. No derivative is recorded (forward-mode tangents are refused). Under a trace or
    a dispatch mode the write is made of torch operations, with the same results."""
    d = _check_cache(key_cache, value_cache, key_groups, value_groups, k_scale, v_scale)
    _check_rows(key, value, key_cache.shape[2], d, "4-bit kv-cache write")
    n = slot_mapping.numel()
    if key.shape[0] < n or value.shape[0] < n:
        raise ValueError(f"key {tuple(key.shape)} / value {tuple(value.shape)} have fewer rows "
                         f"than the {n} slots")
    dev, written = key.device, [key_cache, value_cache, key_groups, value_groups]
    if forward_ad._current_level >= 0:
        vb._check_no_tangents(key, value, *written, k_scale, v_scale)
    for t in (key, value, key_cache, value_cache):
        if not t.is_cuda or t.device != dev:
            raise ValueError("key, value and the caches must be on one GPU")
    vb._check_written(*written)
    torch_only = vb._torch_only()
    if n and len({vb._place(t, torch_only) for t in written}) < 4:
        raise ValueError("the caches and the group words must be memory of their own")
    if torch_only:
        reshape_and_cache_int4_reference(key, value, *written, slot_mapping, k_scale, v_scale)
        return
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    a, keep = _cache_args(key, value, *written, slots.data_ptr(), n, d, k_scale, v_scale)
    vb._launch(dev, _lib.load().fp_kv_cache_write_int4, ctypes.byref(a))
    torch.autograd.graph.increment_version(written)


def quantise_int4(x: torch.Tensor, scale: Optional[torch.Tensor] = None
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Code bytes and group words of rows x (tokens, Hkv, d): ``reshape_and_cache_int4``'s
    rule as torch operations."""
    n, h, d = x.shape
    x = x.float()
    if scale is not None:
        x = x / scale.to(x.device).view(1, -1, 1)
    x = x.view(n, h, d // GROUP, GROUP).clamp(-_MOST, _MOST)
    lo, hi = x.amin(-1), x.amax(-1)  # (NaN where there is one)
    # (tensors, by which torch divides: by numbers it multiplies with their reciprocals)
    want = torch.maximum((hi - lo) / lo.new_full((), 15.0),
                         torch.maximum(hi, -lo) / lo.new_full((), 56.0))
    m = want.view(torch.int32)
    m = (m + 0x7ffff + ((m >> 20) & 1)) >> 20 << 20
    s = torch.where(want < 2.0 ** -14, torch.round(want * 2.0 ** 17) * 2.0 ** -17,
                    m.view(torch.float32)).abs()  # (a group of -0: 0)
    nan = want.isnan()
    none = (s == 0) | nan
    some = torch.where(none, torch.ones_like(s), s)
    z = torch.round(lo / some).clamp(-64, 63).masked_fill(none, 0.0)
    c = (torch.round(x / some.unsqueeze(-1)) - z.unsqueeze(-1)).clamp(0, 15)
    c = c.masked_fill(none.unsqueeze(-1), 0.0).to(torch.uint8)
    bits = s.masked_fill(nan, 0.0).to(torch.float16).view(torch.int16)
    word = (bits | (z.to(torch.int16) + 64)).masked_fill(nan, 0x7f80)
    c = c.view(n, h, d // GROUP, 16, 2)
    byte = c[..., 0] | c[..., 1] << 4
    return byte.transpose(-1, -2).reshape(n, h, d // 2), word


def int4_values(codes: torch.Tensor, groups: torch.Tensor,
                scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The fp32 values (..., Hkv, d) of code bytes (..., Hkv, d / 2) and group words
    (..., Hkv, d / 32)."""
    *lead, half = codes.shape
    b = codes.unflatten(-1, (16, half // 16)).transpose(-1, -2)  # (..., d / 32, 16)
    c = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()
    s = (groups & 0x7f80).contiguous().view(torch.float16).float()
    x = ((c + ((groups & 127) - 64).float().unsqueeze(-1)) * s.unsqueeze(-1)).flatten(-2)
    return x if scale is None else x * scale.to(x.device).view(-1, 1)


@torch.no_grad()
def reshape_and_cache_int4_reference(key, value, key_cache, value_cache, key_groups, value_groups,
                                     slot_mapping, k_scale=None, v_scale=None) -> None:
    """The torch composition of ``reshape_and_cache_int4``, what a trace or a dispatch
    mode sees of it."""
    nb, bs = key_cache.shape[:2]
    slots = slot_mapping.reshape(-1).long().to(key_cache.device)
    rows = ((slots >= 0) & (slots < nb * bs)).nonzero().view(-1)
    page, at = slots[rows] // bs, slots[rows] % bs
    for x, cache, groups, scale in ((key, key_cache, key_groups, k_scale),
                                    (value, value_cache, value_groups, v_scale)):
        cache[page, at], groups[page, :, at] = quantise_int4(x[rows], scale)


def gather_cache_int4(key_cache: torch.Tensor, value_cache: torch.Tensor,
                      key_groups: torch.Tensor, value_groups: torch.Tensor, key: torch.Tensor,
                      value: torch.Tensor, cu_seqlens: torch.Tensor, block_table: torch.Tensor,
                      starts: Optional[torch.Tensor] = None,
                      k_scale: Optional[torch.Tensor] = None,
                      v_scale: Optional[torch.Tensor] = None) -> None:
    """Read 4-bit paged caches back into packed bf16 or fp16 rows, which are written:
    ``gather_cache`` (its rows, sequences and checks on the device) with
    ``s (c + z) t`` in fp32, rounded once."""
    d = _check_cache(key_cache, value_cache, key_groups, value_groups, k_scale, v_scale)
    _check_rows(key, value, key_cache.shape[2], d, "4-bit kv-cache read-back")
    if value.shape != key.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} differ")
    B, dev = vb._check_sequences(cu_seqlens, block_table, starts, key.shape[0]), key.device
    if forward_ad._current_level >= 0:
        vb._check_no_tangents(key, value, key_cache, value_cache, k_scale, v_scale)
    for t in (key, value, key_cache, value_cache):
        if not t.is_cuda or t.device != dev:
            raise ValueError("key, value and the caches must be on one GPU")
    vb._check_written(key, value)
    torch_only = vb._torch_only()
    if key.numel() and vb._place(key, torch_only) == vb._place(value, torch_only):
        raise ValueError("key and value must be memory of their own")
    if B == 0:
        return
    if torch_only:
        gather_cache_int4_reference(key_cache, value_cache, key_groups, value_groups, key, value,
                                    cu_seqlens, block_table, starts, k_scale, v_scale)
        return
    sequences, keep = vb._sequence_args(cu_seqlens, block_table, starts, dev)
    cache, scales = _cache_args(key, value, key_cache, value_cache, key_groups, value_groups, 0,
                                key.shape[0], d, k_scale, v_scale)
    a = _lib.FpKvGatherInt4Args(cache, *sequences)
    vb._launch(dev, _lib.load().fp_kv_cache_gather_int4, ctypes.byref(a))
    torch.autograd.graph.increment_version([key, value])


@torch.no_grad()
def gather_cache_int4_reference(key_cache, value_cache, key_groups, value_groups, key, value,
                                cu_seqlens, block_table, starts=None, k_scale=None,
                                v_scale=None) -> None:
    """The torch composition of ``gather_cache_int4``, what a trace or a dispatch mode
    sees of it."""
    if key.numel() == 0:
        return
    page, at, fits, written = vb._cached_places(key.device, key.shape[0], key_cache.shape,
                                                cu_seqlens, block_table, starts)
    for y, cache, groups, scale in ((key, key_cache, key_groups, k_scale),
                                    (value, value_cache, value_groups, v_scale)):
        x = int4_values(cache[page, at], groups[page, :, at], scale).to(y.dtype)
        x = x.masked_fill(~fits.view(-1, 1, 1), math.nan)
        y.copy_(torch.where(written.view(-1, 1, 1), x, y))


def paged_decode_attention_int4(query: torch.Tensor, key_cache: torch.Tensor,
                                value_cache: torch.Tensor, key_groups: torch.Tensor,
                                value_groups: torch.Tensor, out: torch.Tensor,
                                cu_seqlens_q: torch.Tensor, seqused_k: torch.Tensor,
                                block_table: torch.Tensor, softmax_scale: float,
                                k_scale: Optional[torch.Tensor] = None,
                                v_scale: Optional[torch.Tensor] = None) -> None:
    """Attention over 4-bit paged caches: ``paged_decode_attention`` (its rows, lengths
    and checks on the device) over the values that the caches hold, none of which is
    rounded on the way. bf16 / fp16 queries and outputs on the GPU take the HIP kernels
    behind ``fp_paged_attention_int4``; calls that those do not take (the CPU, fp32,
    layouts that they cannot read in 16-byte pieces, inputs that require gradients) the
    torch composition."""
    d = _check_cache(key_cache, value_cache, key_groups, value_groups, k_scale, v_scale)
    if query.element_size() < 2:
        raise NotImplementedError(f"a query of {query.dtype} over a 4-bit cache: its codes have a "
                                  f"scale of their own, which this operator does not take")
    caches = key_cache, value_cache, key_groups, value_groups
    if not _kernel_takes(query, *caches, out, cu_seqlens_q, seqused_k, block_table, k_scale,
                         v_scale, d):
        paged_attention_int4_reference(query, *caches, out, cu_seqlens_q, seqused_k, block_table,
                                       softmax_scale, k_scale, v_scale)
        return
    dev, lib = query.device, _lib.load()
    base, keep = vb._paged_args(query, key_cache, value_cache, out, cu_seqlens_q, seqused_k,
                                block_table, softmax_scale, d)
    (ks, k_keep), (vs, v_keep) = (vb._scale_args(s, dev) for s in (k_scale, v_scale))
    call = _lib.FpPagedInt4Args(base, _groups(key_groups), _groups(value_groups), ks, vs)
    vb._attend(dev, call, lib.fp_paged_int4_workspace_bytes, lib.fp_paged_attention_int4, out)


def _kernel_takes(query, key_cache, value_cache, key_groups, value_groups, out, cu, used, table,
                  k_scale, v_scale, d: int) -> bool:
    nb, bs, hkv, _ = key_cache.shape
    if not vb._call_fits(query, out, (nb, bs, hkv, d), cu, used, table):
        return False
    if key_cache.device != query.device or value_cache.device != query.device:
        return False
    for t in (query, key_cache, value_cache, out):
        if not vb._rows_ok(t, True):
            return False
    words = 8 if bs % 16 == 0 else d // GROUP
    for g in (key_groups, value_groups):
        if g.data_ptr() % (2 * words) or (nb > 1 and (g.stride(0) % words or g.stride(0) < 0)) or \
                (hkv > 1 and (g.stride(1) % words or g.stride(1) < 0)):
            return False
    if key_cache.stride(1) >= 1 << 24 or value_cache.stride(1) >= 1 << 24:
        return False
    return vb._none_requires_grad(query, out, k_scale, v_scale)


def paged_attention_int4_reference(query, key_cache, value_cache, key_groups, value_groups, out,
                                   cu_seqlens_q, seqused_k, block_table, softmax_scale,
                                   k_scale=None, v_scale=None) -> None:
    """The torch composition of ``paged_decode_attention_int4`` in fp32, a sequence at a
    time: the path of the calls that the kernels do not take."""
    vb._attend_composed(
        query, out, cu_seqlens_q, seqused_k, block_table, softmax_scale, key_cache.shape[1],
        lambda blocks: (int4_values(key_cache[blocks], key_groups[blocks].transpose(1, 2), k_scale),
                        int4_values(value_cache[blocks], value_groups[blocks].transpose(1, 2),
                                    v_scale)))

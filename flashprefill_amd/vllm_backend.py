"""vLLM attention-backend hook: FlashPrefill for prefill steps.

Two forwards, one per reference patch:

* ``make_forward`` / ``apply_patch``: vLLM's v1 engine
  (``patches/patch_loader_vllm_0_12_0.py:57-253``), described below;
* ``make_forward_v0`` / ``apply_patch_v0``: the v0 engine's backend
  (``patches/patch_loader_vllm_0_10_0.py:55-376``), whose metadata splits a
  batch into prefill tokens first and decode tokens after them.

The v1 forward mirrors what the 0.12 patch does to
``FlashAttentionImpl.forward``:

* write the step's key / value rows into the paged KV cache
  (``reshape_and_cache_flash``, :140-149) -- here the HIP kernel behind
  ``fp_kv_cache_write``;
* ``is_prefill = max_query_len > 1`` (:169): prefill batches go to
  ``flash_prefill_varlen_func`` over the step's own packed q / k / v with the
  per-model selection config (:186-200);
* decode batches (one query per sequence) go to a paged decode attention over
  the cache (:201-225, vLLM's ``flash_attn_varlen_func``);
* a profiling run (``attn_metadata is None``) zero-fills the output (:95-97),
  encoder attention and cascade attention are delegated unchanged (:104-114,
  :226-252), fused output quantisation is rejected (:90-93);
* an fp8 ``kv_cache_dtype`` (:151-166) keeps the cache in 8-bit floats with the
  layer's ``_k_scale`` / ``_v_scale``: written by the HIP kernel behind
  ``fp_kv_cache_write_fp8``, attended by ``fp_paged_attention_fp8``. The query
  stays in 16 bits: one that the layer has quantised is refused.

vLLM is not a dependency: the forward only touches the attributes of the
impl object and the metadata that the reference's forward reads, and the two
vLLM operations it cannot provide itself (decode over the paged cache, and
the encoder / cascade paths) are injected. ``apply_patch`` installs the
forward on vLLM's ``FlashAttentionImpl`` when vLLM is importable, or on any
class passed to it (the tests use stand-ins).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Any, Callable, Dict, Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .flashprefill_varlen_func import flash_prefill_varlen_func

# Per-model selection configs of the reference patch
# (patches/patch_loader_vllm_0_12_0.py:13-40): block 128, sink 2, window 4,
# last 2 q-blocks dense; alpha per model family.
ATTENTION_CONFIGS: Dict[str, Dict[str, Any]] = {
    "flashprefill_llama": {"block_size": 128, "attention_sink": 2, "window_size": 4,
                           "alpha": 0.18, "last_n_full_block": 2},
    "flashprefill_qwen2": {"block_size": 128, "attention_sink": 2, "window_size": 4,
                           "alpha": 0.08, "last_n_full_block": 2},
    "flashprefill_qwen3moe": {"block_size": 128, "attention_sink": 2, "window_size": 4,
                              "alpha": 0.12, "last_n_full_block": 2},
}
DEFAULT_CONFIG = "flashprefill_qwen2"  # the reference patch's choice (:43)

_DTYPES = {torch.bfloat16: _lib.FP_DTYPE_BF16, torch.float16: _lib.FP_DTYPE_F16}


# 8-bit cache types and their names in vLLM's kv_cache_dtype
_FORMATS = {torch.float8_e4m3fn: _lib.FP_CACHE_E4M3, torch.float8_e5m2: _lib.FP_CACHE_E5M2}
_FP8_NAMES = {"fp8": torch.float8_e4m3fn, "fp8_e4m3": torch.float8_e4m3fn,
              "fp8_e5m2": torch.float8_e5m2}


def _check_scales(cache: torch.Tensor, k_scale, v_scale) -> None:
    """Refuse scales that are not of one of the forms that ``reshape_and_cache``
    describes, or that come with a 16-bit cache."""
    if k_scale is None and v_scale is None:
        return
    nb, bs, hkv = cache.shape[:3]
    for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
        if s is None:
            continue
        if cache.dtype not in _FORMATS:
            raise ValueError(f"{name}: scales belong to 8-bit caches, this one is {cache.dtype}")
        if s.dtype != torch.float32:
            raise ValueError(f"{name} must be float32, got {s.dtype}")
        if s.dim() == 3:
            if s.shape != (nb, hkv, bs) or s.device != cache.device or \
                    (bs > 1 and s.stride(2) != 1):
                raise ValueError(f"{name}: one scale per slot is (num_blocks, num_kv_heads, "
                                 f"block_size) = {(nb, hkv, bs)} on the cache's device, slots "
                                 f"contiguous; got {tuple(s.shape)} on {s.device}")
        elif s.dim() > 1 or s.numel() not in (1, hkv):
            raise ValueError(f"{name} must hold 1 or {hkv} values, or one per slot "
                             f"{(nb, hkv, bs)}; got {tuple(s.shape)}")


def _slot_scale_strides(scale: torch.Tensor) -> tuple:
    """Strides of scales per slot between pages and between heads, 0 where there is one
    (torch may give such a dimension any stride)."""
    nb, hkv, _ = scale.shape
    return scale.stride(0) if nb > 1 else 0, scale.stride(1) if hkv > 1 else 0


def _scale_args(scale: Optional[torch.Tensor], device) -> tuple:
    """``fp_kv_scales`` of a checked scale, and the tensor whose memory it names."""
    if scale is None:
        return _lib.FpKvScales(), None
    if scale.dim() == 3:
        return _lib.FpKvScales(scale.data_ptr(), *_slot_scale_strides(scale), 1), scale
    if scale.device != device or not scale.is_contiguous():
        scale = scale.to(device).contiguous()
    return _lib.FpKvScales(scale.data_ptr(), 0, 1 if scale.numel() > 1 else 0, 0), scale


def _launch(device: torch.device, fn, *args) -> None:
    """``fn(*args, stream)`` with ``device`` current, on torch's current stream there."""
    if torch.cuda.current_device() == device.index:
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))
        return
    with torch.cuda.device(device):
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))


def _check_rows(key, value, key_cache, value_cache, what: str) -> None:
    """Types, layout and sizes that the cache's write and read-back share."""
    if key.dtype not in _DTYPES or value.dtype != key.dtype or \
            value_cache.dtype != key_cache.dtype or \
            (key_cache.dtype != key.dtype and key_cache.dtype not in _FORMATS):
        raise NotImplementedError(
            f"{what} supports bf16 / fp16 rows and caches of their dtype, float8_e4m3fn or "
            f"float8_e5m2, got key {key.dtype}, value {value.dtype}, caches {key_cache.dtype}, "
            f"{value_cache.dtype}")
    for name, t in (("key", key), ("value", value), ("key_cache", key_cache),
                    ("value_cache", value_cache)):
        if t.stride(-1) != 1:
            raise ValueError(f"{name} must have a contiguous head dimension")
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape:
        raise ValueError("caches must be (num_blocks, block_size, num_kv_heads, head_dim)")
    if key.dim() != 3 or value.dim() != 3 or key.shape[1:] != key_cache.shape[2:] or \
            value.shape[1:] != key_cache.shape[2:]:
        raise ValueError(f"key {tuple(key.shape)} / value {tuple(value.shape)} do not match the "
                         f"cache {tuple(key_cache.shape)}")


def _check_written(*tensors) -> None:
    """Refuse what torch's own in-place operations refuse, or would record: several
    elements in one place, inference tensors outside inference mode, and tensors that
    require a gradient (the kernels have none)."""
    for t in tensors:
        if 0 in t.stride() and any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
            raise RuntimeError("a tensor to be written has several elements in one memory "
                               "location: clone() it first")
        if t.is_inference() and not torch.is_inference_mode_enabled():
            raise RuntimeError("an inference tensor cannot be written outside inference mode")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("a tensor to be written requires a gradient: use torch.no_grad()")


_tracing_state, _dispatch_modes = torch._C._get_tracing_state, torch._C._len_torch_dispatch_stack


def _torch_only() -> bool:
    """Whether a trace or a dispatch mode is on: they see torch operations, not kernels."""
    return _dispatch_modes() > 0 or _tracing_state() is not None


def _check_no_tangents(*tensors) -> None:
    """Refuse forward-mode tangents, which the kernels would drop."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("a tensor has a forward-mode tangent: the cache's write and "
                                      "read-back have no derivative")


def _place(t: torch.Tensor, torch_only: bool):
    """Where a tensor begins. (Those without memory, as in a trace over fake tensors, have
    a storage of their own all the same.)"""
    return (t.untyped_storage()._cdata, t.storage_offset()) if torch_only else t.data_ptr()


def _cache_args(key, value, key_cache, value_cache, slots: int, n: int) -> _lib.FpKvCacheArgs:
    nb, bs, hkv, d = key_cache.shape
    return _lib.FpKvCacheArgs(key.data_ptr(), value.data_ptr(), *key.stride()[:2],
                              *value.stride()[:2], key_cache.data_ptr(), value_cache.data_ptr(),
                              *key_cache.stride()[:3], *value_cache.stride()[:3], slots, n, nb,
                              bs, hkv, d, _DTYPES[key.dtype])


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                      value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                      k_scale: Optional[torch.Tensor] = None,
                      v_scale: Optional[torch.Tensor] = None) -> None:
    """Write key / value (tokens, Hkv, d) into the paged caches
    (num_blocks, block_size, Hkv, d) at ``slot_mapping`` (int64, one slot per
    token; the mapping's length is the number of tokens written, negative
    slots are padding and skipped), on the current stream.

    Caches of key's dtype hold the rows as they are, and may lie in pinned memory of
    the host. Caches of float8_e4m3fn or float8_e5m2 hold ``x / scale`` rounded to
    nearest even, what lies beyond the format's largest finite value (infinities too)
    as that value, NaN as NaN. The fp32 scales are

    * fixed, and read: one value, or one per KV head (None: 1);
    * one per slot and KV head, ``(num_blocks, Hkv, block_size)``: found from each
      row, its largest finite magnitude over the format's largest finite value (1
      for a row of zeros), and written beside it.

    Slots named by two tokens hold either row, or parts of both. No derivative is
    recorded (forward-mode tangents are refused by 8-bit caches). Under a trace or a
    dispatch mode the write is made of torch operations, with the same results."""
    _check_rows(key, value, key_cache, value_cache, "kv-cache write")
    _check_scales(key_cache, k_scale, v_scale)
    n = slot_mapping.numel()
    if key.shape[0] < n or value.shape[0] < n:
        raise ValueError(f"key {tuple(key.shape)} / value {tuple(value.shape)} do not match the "
                         f"cache {tuple(key_cache.shape)} and {n} slots")
    dev, eight = key.device, key_cache.dtype in _FORMATS
    if eight and forward_ad._current_level >= 0:
        _check_no_tangents(key, value, key_cache, value_cache, k_scale, v_scale)
    for t in (key, value, key_cache, value_cache):
        if t.is_cuda and t.device == dev:
            continue
        # (pinned memory of the host the GPU reads and writes in place)
        if t is key or t.is_cuda or eight or not t.is_pinned():
            raise ValueError("key, value and the caches must be on one GPU")
    torch_only = _torch_only()
    if eight:
        written = [key_cache, value_cache]
        written += [s for s in (k_scale, v_scale) if s is not None and s.dim() == 3]
        _check_written(*written)
        if n and len({_place(t, torch_only) for t in written}) < len(written):
            raise ValueError("the caches and the scales to be written must be memory of their own")
    if torch_only:
        reshape_and_cache_reference(key, value, key_cache, value_cache, slot_mapping, k_scale,
                                    v_scale)
        return
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    lib = _lib.load()
    base = _cache_args(key, value, key_cache, value_cache, slots.data_ptr(), n)
    if not eight:
        _launch(dev, lib.fp_kv_cache_write, ctypes.byref(base))
        return
    (ks, k_keep), (vs, v_keep) = _scale_args(k_scale, dev), _scale_args(v_scale, dev)
    _launch(dev, lib.fp_kv_cache_write_fp8,
            ctypes.byref(_lib.FpKvCacheFp8Args(base, ks, vs, _FORMATS[key_cache.dtype])))
    torch.autograd.graph.increment_version(written)


@torch.no_grad()
def reshape_and_cache_reference(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                                value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                                k_scale: Optional[torch.Tensor] = None,
                                v_scale: Optional[torch.Tensor] = None) -> None:
    """The torch composition of ``reshape_and_cache``, what a trace or a dispatch mode
    sees of it."""
    bs = key_cache.shape[1]
    for x, cache, scale in ((key, key_cache, k_scale), (value, value_cache, v_scale)):
        dev = cache.device
        slots = slot_mapping.reshape(-1).long().to(dev)
        rows = ((slots >= 0) & (slots < cache.shape[0] * bs)).nonzero().view(-1)
        page, at = slots[rows] // bs, slots[rows] % bs
        x = x.to(dev)[rows]
        if cache.dtype not in _FORMATS:
            cache[page, at] = x
            continue
        x, top = x.float(), torch.finfo(cache.dtype).max
        s = None
        if scale is not None and scale.dim() == 3:
            # (a tensor, by which torch divides: a number's reciprocal it would multiply by)
            s = x.abs().masked_fill(~x.isfinite(), 0.0).amax(-1) / x.new_full((), top)
            s = torch.where(s > 0, s, torch.ones_like(s))
            scale[page, :, at] = s
        elif scale is not None:
            s = scale.to(dev).view(1, -1)
        if s is not None:
            x = x / s.unsqueeze(-1)
        cache[page, at] = x.clamp(-top, top).to(cache.dtype)


def gather_cache(key_cache: torch.Tensor, value_cache: torch.Tensor, key: torch.Tensor,
                 value: torch.Tensor, cu_seqlens: torch.Tensor, block_table: torch.Tensor,
                 starts: Optional[torch.Tensor] = None, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None) -> None:
    """Read the paged caches back, the inverse of ``reshape_and_cache``: row
    ``cu_seqlens[b] + i`` of key / value (tokens, Hkv, d; written) becomes cached
    token ``starts[b] + i`` (``starts`` None: token i) of sequence b, whose pages
    are ``block_table[b]``, for every row up to ``cu_seqlens[b + 1] - 1``; rows of
    no sequence are left as they are. 8-bit caches give ``c * scale`` (scales as
    ``reshape_and_cache`` takes them) in fp32, rounded once to key's dtype;
    16-bit ones are copied.

    No host synchronisation: what only the device sees is checked there. Offsets
    that descend or leave the rows make every row NaN, tokens before the first or
    past the room of the table, and pages outside the cache (a number below 0
    counts from the end, as in an index), their own rows. No derivative is
    recorded (forward-mode tangents are refused). Under a trace or a dispatch mode the
    read-back is made of torch operations, with the same results."""
    _check_rows(key, value, key_cache, value_cache, "kv-cache read-back")
    _check_scales(key_cache, k_scale, v_scale)
    if value.shape != key.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} differ")
    if cu_seqlens.dim() != 1 or block_table.dim() != 2 or \
            (starts is not None and starts.dim() != 1):
        raise ValueError("cu_seqlens and starts must have one dimension, block_table two")
    B, dev = cu_seqlens.numel() - 1, key.device
    if B < 0 or block_table.shape[0] < B or (starts is not None and starts.numel() < B):
        raise ValueError(f"block_table {tuple(block_table.shape)} or starts do not match "
                         f"{B} sequences")
    for name, t in (("cu_seqlens", cu_seqlens), ("block_table", block_table), ("starts", starts)):
        if t is not None and t.dtype not in _INDEX:
            raise ValueError(f"{name} must be int32 or int64, got {t.dtype}")
    if forward_ad._current_level >= 0:
        _check_no_tangents(key, value, key_cache, value_cache, k_scale, v_scale)
    if not cu_seqlens.is_cuda:  # known without a synchronisation
        at = cu_seqlens.tolist()
        if at[0] < 0 or at[-1] > key.shape[0] or any(x > y for x, y in zip(at, at[1:])):
            raise ValueError(f"cu_seqlens {at} do not ascend within {key.shape[0]} rows")
    for t in (key, value, key_cache, value_cache):
        if not t.is_cuda or t.device != dev:
            raise ValueError("key, value and the caches must be on one GPU")
    _check_written(key, value)
    torch_only = _torch_only()
    if key.numel() and _place(key, torch_only) == _place(value, torch_only):
        raise ValueError("key and value must be memory of their own")
    if B == 0:
        return
    if torch_only:
        gather_cache_reference(key_cache, value_cache, key, value, cu_seqlens, block_table, starts,
                               k_scale, v_scale)
        return
    cu, table = cu_seqlens.to(dev).contiguous(), block_table.to(dev)
    if table.stride(1) != 1:
        table = table.contiguous()
    if starts is not None:
        starts = starts.to(dev).contiguous()
    (ks, k_keep), (vs, v_keep) = _scale_args(k_scale, dev), _scale_args(v_scale, dev)
    a = _lib.FpKvGatherArgs(
        _cache_args(key, value, key_cache, value_cache, 0, key.shape[0]), ks, vs,
        _FORMATS.get(key_cache.dtype, _lib.FP_CACHE_16BIT), B, table.shape[1],
        cu.dtype == torch.int64, table.dtype == torch.int64,
        starts is not None and starts.dtype == torch.int64, cu.data_ptr(), table.data_ptr(),
        None if starts is None else starts.data_ptr(), table.stride(0))
    _launch(dev, _lib.load().fp_kv_cache_gather, ctypes.byref(a))
    torch.autograd.graph.increment_version([key, value])


@torch.no_grad()
def gather_cache_reference(key_cache: torch.Tensor, value_cache: torch.Tensor, key: torch.Tensor,
                           value: torch.Tensor, cu_seqlens: torch.Tensor, block_table: torch.Tensor,
                           starts: Optional[torch.Tensor] = None,
                           k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None) -> None:
    """The torch composition of ``gather_cache``, what a trace or a dispatch mode sees
    of it."""
    dev, n, B = key.device, key.shape[0], cu_seqlens.numel() - 1
    nb, bs = key_cache.shape[:2]
    if key.numel() == 0:
        return
    if nb < 1 or bs < 1:
        raise ValueError("the caches have no pages")
    room = block_table.shape[1] * bs
    cu, row = cu_seqlens.long().to(dev), torch.arange(n, device=dev)
    off = (cu[0] < 0) | (cu[-1] > n) | (cu[1:] < cu[:-1]).any()
    b = torch.bucketize(row, cu, right=True) - 1
    written = (b >= 0) & (b < B)
    b = torch.where(written, b, 0)
    at = row - cu[b]
    fits, written = written & ~off, written | off
    if starts is not None:
        first = starts.long().to(dev)[b]
        fits = fits & (first >= 0) & (first < room)
        at = at + torch.where(fits, first, 0)
    fits = fits & (at >= 0) & (at < room)
    at = torch.where(fits, at, 0)
    if room > 0:
        page, at = block_table.long().to(dev)[b, at // bs], at % bs
        page = torch.where(page < 0, page + nb, page)
        fits = fits & (page >= 0) & (page < nb)
        page = torch.where(fits, page, 0)
    else:
        page = at
    for y, cache, scale in ((key, key_cache, k_scale), (value, value_cache, v_scale)):
        x = cache[page, at]
        if cache.dtype in _FORMATS:
            x = x.float()
            if scale is not None:
                s = scale[page, :, at] if scale.dim() == 3 else scale.to(dev).view(1, -1)
                x = x * s.unsqueeze(-1)
            x = x.to(y.dtype)
        x = x.masked_fill(~fits.view(-1, 1, 1), math.nan)
        y.copy_(torch.where(written.view(-1, 1, 1), x, y))


def paged_decode_attention(query: torch.Tensor, key_cache: torch.Tensor,
                           value_cache: torch.Tensor, out: torch.Tensor,
                           cu_seqlens_q: torch.Tensor, seqused_k: torch.Tensor,
                           block_table: torch.Tensor, softmax_scale: float,
                           k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None) -> None:
    """Attention over the paged cache (the role of vLLM's
    ``flash_attn_varlen_func`` with a block table in the reference's decode
    branch): every query row of sequence b attends causally to the first
    ``seqused_k[b]`` cached tokens, the last query sitting at position
    ``seqused_k[b] - 1``; fp32 softmax and sums. The default when no vLLM
    decode op is injected, not part of the prefill path.

    bf16 / fp16 tensors on the GPU (head_dim 64, 128 or 256) take the HIP
    kernels behind ``fp_paged_attention``: no host synchronisation, so what
    only the device sees is checked there (a sequence with more cached tokens
    than its table row has room for, or rows that attend to a page outside the
    cache, get NaN; offsets that descend or leave the query rows make every
    row NaN). Every other call (CPU, fp32, other head dims or layouts, offsets
    or lengths on the host that do not fit, inputs that require gradients)
    takes the torch composition.

    Caches of float8_e4m3fn or float8_e5m2 stand for their values times
    ``k_scale`` / ``v_scale``, which are as ``reshape_and_cache`` takes them; query
    and out stay in 16 bits (a query of 8 bits is refused), and no cached value is
    rounded on the way (``fp_paged_attention_fp8``)."""
    _check_scales(key_cache, k_scale, v_scale)
    if _paged_kernel_takes(query, key_cache, value_cache, out, cu_seqlens_q, seqused_k,
                           block_table, k_scale, v_scale):
        _paged_attention_kernel(query, key_cache, value_cache, out, cu_seqlens_q, seqused_k,
                                block_table, softmax_scale, k_scale, v_scale)
    else:
        paged_attention_reference(query, key_cache, value_cache, out, cu_seqlens_q, seqused_k,
                                  block_table, softmax_scale, k_scale, v_scale)


_INDEX = (torch.int32, torch.int64)


def _rows_ok(t: torch.Tensor, any_stride_of_one: bool) -> bool:
    step = 16 // t.element_size()
    *rest, last = t.stride()
    if last != 1 or t.data_ptr() % 16:
        return False
    for i, s in enumerate(rest):
        if (s % step or s < 0) and not (any_stride_of_one and t.shape[i] == 1):
            return False
    return True


def _paged_kernel_takes(query, key_cache, value_cache, out, cu, used, table, k_scale=None,
                        v_scale=None) -> bool:
    """Whether the HIP kernels take this call as it is: 16-bit tensors of one
    type on one GPU (or caches of one 8-bit type with scales that the kernels can
    read in 16-byte pieces), head_dim 64 / 128 / 256, 16-byte aligned rows, int32
    / int64 metadata of matching shapes, no derivative, functional transform,
    trace or dispatch mode to carry along (they see only torch operations)."""
    if not query.is_cuda or query.dtype not in _DTYPES:
        return False
    if forward_ad._current_level >= 0 or _torch_only() or \
            torch._C._functorch.peek_interpreter_stack() is not None:
        return False
    dev, dt = query.device, query.dtype
    if query.dim() != 3 or out.dim() != 3 or key_cache.dim() != 4 or \
            value_cache.shape != key_cache.shape:
        return False
    nb, bs, hkv, d = key_cache.shape
    T, hq, dq = query.shape
    if d not in (64, 128, 256) or dq != d or nb < 1 or bs < 1 or hkv < 1 or hq < 1 or hq % hkv or \
            out.shape[0] < T or out.shape[1:] != query.shape[1:]:
        return False
    cdt = key_cache.dtype
    if cdt != dt and cdt not in _FORMATS:
        return False
    for t, want in ((query, dt), (key_cache, cdt), (value_cache, cdt), (out, dt)):
        if t.dtype != want or t.device != dev or not _rows_ok(t, cdt != dt):
            return False
    for s in (k_scale, v_scale):
        if s is not None and s.dim() == 3 and bs % 16 == 0 and \
                (s.data_ptr() % 16 or any(st % 4 for st in _slot_scale_strides(s))):
            return False
    # torch refuses to write these, and so does the composition
    if (0 in out.stride() and any(n > 1 and st == 0 for n, st in zip(out.shape, out.stride()))) or \
            (out.is_inference() and not torch.is_inference_mode_enabled()):
        return False
    if key_cache.stride(1) >= 1 << 24 or value_cache.stride(1) >= 1 << 24:
        return False
    if cu.dim() != 1 or used.dim() != 1 or table.dim() != 2 or cu.numel() < 2:
        return False
    B = cu.numel() - 1
    if used.numel() < B or table.shape[0] < B or cu.dtype not in _INDEX or \
            used.dtype not in _INDEX or table.dtype not in _INDEX:
        return False
    if table.shape[1] * bs >= 1 << 30 or T * hq >= 1 << 30:
        return False
    if not cu.is_cuda:  # known without a synchronisation: refused there
        at = cu.tolist()
        if at[0] < 0 or at[-1] > T or any(x > y for x, y in zip(at, at[1:])):
            return False
    if not used.is_cuda and any(n > table.shape[1] * bs for n in used[:B].tolist()):
        return False
    if not torch.is_grad_enabled():
        return True
    for t in (query, key_cache, value_cache, out, k_scale, v_scale):
        if t is not None and t.requires_grad:
            return False
    return True


def _paged_attention_kernel(query, key_cache, value_cache, out, cu, used, table, scale,
                            k_scale=None, v_scale=None) -> None:
    dev = query.device
    nb, bs, hkv, d = key_cache.shape
    T, hq = query.shape[:2]
    cu, used = cu.to(dev).contiguous(), used.to(dev).contiguous()
    table = table.to(dev)
    if table.stride(1) != 1:
        table = table.contiguous()
    lib = _lib.load()
    call = _lib.FpPagedArgs(
        query.data_ptr(), *query.stride()[:2], out.data_ptr(), *out.stride()[:2],
        key_cache.data_ptr(), value_cache.data_ptr(), *key_cache.stride()[:3],
        *value_cache.stride()[:3], cu.data_ptr(), used.data_ptr(), table.data_ptr(),
        table.stride(0), T, nb, cu.numel() - 1, table.shape[1], bs, hq, hkv, d,
        _DTYPES[query.dtype], cu.dtype == torch.int64, used.dtype == torch.int64,
        table.dtype == torch.int64, float(scale))
    ws_bytes, launch = lib.fp_paged_workspace_bytes, lib.fp_paged_attention
    if key_cache.dtype in _FORMATS:
        (ks, k_keep), (vs, v_keep) = _scale_args(k_scale, dev), _scale_args(v_scale, dev)
        call = _lib.FpPagedFp8Args(call, ks, vs, _FORMATS[key_cache.dtype])
        ws_bytes, launch = lib.fp_paged_fp8_workspace_bytes, lib.fp_paged_attention_fp8
    # A buffer of this call's own: threads that share a stream may interleave
    # their launches, and a shared one would be written between the chunks and
    # their merge. The caching allocator hands it on in stream order.
    n = ws_bytes(ctypes.byref(call))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _launch(dev, launch, ctypes.byref(call), None if ws is None else ws.data_ptr())
    # a graph that saved `out` finds it changed, as after any in-place operation
    torch.autograd.graph.increment_version(out)


def paged_attention_reference(query: torch.Tensor, key_cache: torch.Tensor,
                              value_cache: torch.Tensor, out: torch.Tensor,
                              cu_seqlens_q: torch.Tensor, seqused_k: torch.Tensor,
                              block_table: torch.Tensor, softmax_scale: float,
                              k_scale: Optional[torch.Tensor] = None,
                              v_scale: Optional[torch.Tensor] = None) -> None:
    """The torch composition of ``paged_decode_attention`` in fp32 (one small
    gather per sequence): the kernels' reference, and the path of the calls
    they do not take."""
    if key_cache.dtype in _FORMATS and query.element_size() < 2:
        raise NotImplementedError(f"a query of {query.dtype} over an 8-bit cache: its codes have a "
                                  f"scale of their own, which this operation does not take")
    cu = cu_seqlens_q.tolist()
    used = seqused_k.tolist()
    _, bs, hkv, d = key_cache.shape
    hq = query.shape[1]
    g = hq // hkv
    for b in range(len(cu) - 1):
        q0, q1 = cu[b], cu[b + 1]
        nq, nk = q1 - q0, int(used[b])
        if nq == 0:
            continue
        nblk = (nk + bs - 1) // bs
        blocks = block_table[b, :nblk].long()
        k = _pages_fp32(key_cache, blocks, k_scale).reshape(nblk * bs, hkv, d)[:nk]
        v = _pages_fp32(value_cache, blocks, v_scale).reshape(nblk * bs, hkv, d)[:nk]
        q = query[q0:q1].float()  # (nq, hq, d)
        k = k.repeat_interleave(g, dim=1).permute(1, 2, 0).contiguous()  # (hq, d, nk)
        v = v.repeat_interleave(g, dim=1).permute(1, 0, 2).contiguous()  # (hq, nk, d)
        s = torch.matmul(q.permute(1, 0, 2).contiguous(), k) * softmax_scale  # (hq, nq, nk)
        qpos = torch.arange(nk - nq, nk, device=query.device).view(1, nq, 1)
        kpos = torch.arange(nk, device=query.device).view(1, 1, nk)
        s = s.masked_fill(kpos > qpos, float("-inf"))
        o = torch.matmul(torch.softmax(s, dim=-1), v)  # (hq, nq, d)
        out[q0:q1] = o.permute(1, 0, 2).to(out.dtype)


def _pages_fp32(cache: torch.Tensor, blocks: torch.Tensor,
                scale: Optional[torch.Tensor]) -> torch.Tensor:
    """The pages' values in fp32, (blocks, block_size, Hkv, d)."""
    x = cache[blocks].float()
    if scale is None:
        return x
    if scale.dim() == 3:
        return x * scale[blocks].transpose(1, 2).unsqueeze(-1)
    return x * scale.to(x.device).view(-1, 1)


@dataclass
class HookOps:
    """The operations the hooked forward calls; the defaults are this
    package's (KV-cache write kernel, FlashPrefill, paged attention).
    ``encoder`` and ``cascade`` take the impl and the reference's arguments
    and default to raising: they stay vLLM's. ``cache_write_fp8`` and
    ``decode_fp8`` serve layers with an fp8 cache: the operations above with the
    scales as two more arguments."""
    cache_write: Callable[..., None] = reshape_and_cache
    prefill: Callable[..., None] = flash_prefill_varlen_func
    decode: Callable[..., None] = paged_decode_attention
    encoder: Optional[Callable[..., torch.Tensor]] = None
    cascade: Optional[Callable[..., torch.Tensor]] = None
    cache_write_fp8: Callable[..., None] = reshape_and_cache
    decode_fp8: Callable[..., None] = paged_decode_attention


def _cache_ops(impl, layer, ops: HookOps, key_cache, value_cache):
    """The layer's caches, its cache write and its attention over them: those of
    ``ops``, or for an fp8 ``kv_cache_dtype`` the 8-bit forms with the layer's
    ``_k_scale`` / ``_v_scale`` (1 where it has none) over the caches, which vLLM
    allocates as bytes, in their type."""
    name = str(getattr(impl, "kv_cache_dtype", "auto"))
    if not name.startswith("fp8"):
        return key_cache, value_cache, ops.cache_write, ops.decode
    dtype = _FP8_NAMES.get(name)
    if dtype is None or key_cache.dtype not in (torch.uint8, dtype):
        raise NotImplementedError(f"kv_cache_dtype {name} with a cache of {key_cache.dtype} is not "
                                  f"supported by this hook (8-bit caches: {sorted(_FP8_NAMES)})")
    scales = getattr(layer, "_k_scale", None), getattr(layer, "_v_scale", None)

    def write(key, value, kc, vc, slots):
        ops.cache_write_fp8(key, value, kc, vc, slots, *scales)

    def decode(q, kc, vc, out, cu, used, table, scale):
        ops.decode_fp8(q, kc, vc, out, cu, used, table, scale, *scales)

    return key_cache.view(dtype), value_cache.view(dtype), write, decode


def _is_encoder(attn_type) -> bool:
    """vLLM's AttentionType.ENCODER / ENCODER_ONLY ("encoder", "encoder_only";
    an enum member's name works too)."""
    name = str(getattr(attn_type, "value", attn_type)).lower().rsplit(".", 1)[-1]
    return name in ("encoder", "encoder_only")


def make_forward(cfg: Dict[str, Any], ops: Optional[HookOps] = None):
    """The FlashAttentionImpl.forward replacement, closed over the selection
    config ``cfg`` (one of ATTENTION_CONFIGS' values)."""
    ops = ops or HookOps()

    def flash_prefill_forward(self, layer, query, key, value, kv_cache, attn_metadata,
                              output=None, output_scale=None, output_block_scale=None):
        if output is None:
            raise ValueError("Output tensor must be provided.")
        if output_scale is not None or output_block_scale is not None:
            raise NotImplementedError("fused output quantization is not supported")
        if attn_metadata is None:  # profiling run
            return output.fill_(0)
        n = attn_metadata.num_actual_tokens
        if _is_encoder(getattr(self, "attn_type", "decoder")):
            if ops.encoder is None:
                raise NotImplementedError("encoder attention is left to vLLM's backend")
            return ops.encoder(self, query[:n], key[:n], value[:n], output[:n], attn_metadata,
                               layer)
        key_cache, value_cache, cache_write, decode = _cache_ops(self, layer, ops,
                                                                 *kv_cache.unbind(0))
        if getattr(self, "kv_sharing_target_layer_name", None) is None and key is not None \
                and value is not None:
            cache_write(key, value, key_cache, value_cache, attn_metadata.slot_mapping)
        if getattr(attn_metadata, "use_cascade", False):
            if ops.cascade is None:
                raise NotImplementedError("cascade attention is left to vLLM's backend")
            return ops.cascade(self, query[:n], key_cache, value_cache, output[:n],
                               attn_metadata, layer)
        if getattr(self, "dcp_world_size", 1) > 1:
            raise NotImplementedError("decode context parallelism is left to vLLM's backend")
        cu_seqlens_q = attn_metadata.query_start_loc
        if attn_metadata.max_query_len > 1:  # prefill
            ops.prefill(query[:n], key[:n], value[:n], output[:n], cu_seqlens_q,
                        attn_metadata.max_query_len, cfg["alpha"], cfg["block_size"],
                        cfg["attention_sink"], cfg["window_size"], cfg["last_n_full_block"])
        else:
            decode(query[:n], key_cache, value_cache, output[:n], cu_seqlens_q,
                   attn_metadata.seq_lens, attn_metadata.block_table,
                   getattr(self, "scale", 1.0 / math.sqrt(query.shape[-1])))
        return output

    return flash_prefill_forward


def apply_patch(impl_cls=None, config: str = DEFAULT_CONFIG, ops: Optional[HookOps] = None):
    """Replace ``impl_cls.forward`` (default: vLLM's v1 FlashAttentionImpl)
    with the FlashPrefill forward for ``config``; returns the original forward.
    The reference's per-rank Triton cache directory (:49-54) has no
    counterpart: nothing is compiled at run time here."""
    if impl_cls is None:
        import vllm.v1.attention.backends.flash_attn as fa_backend  # noqa: WPS433
        impl_cls = fa_backend.FlashAttentionImpl
    cfg = ATTENTION_CONFIGS[config]
    if ops is None:
        ops = HookOps()
        try:  # inside vLLM, decode uses vLLM's own paged attention op
            from vllm.attention.utils.fa_utils import flash_attn_varlen_func as vllm_fa

            def vllm_decode(q, kc, vc, out, cu, seqused_k, block_table, scale):
                vllm_fa(q=q, k=kc, v=vc, out=out, cu_seqlens_q=cu, max_seqlen_q=1,
                        seqused_k=seqused_k, max_seqlen_k=int(seqused_k.max()),
                        softmax_scale=scale, causal=True, block_table=block_table)
            ops.decode = vllm_decode
        except ImportError:
            pass
    original = impl_cls.forward
    impl_cls.forward = make_forward(cfg, ops)
    return original


# ---------------------------------------------------------------------------
# vLLM v0 engine (patches/patch_loader_vllm_0_10_0.py)
# ---------------------------------------------------------------------------

def _is_decoder(attn_type) -> bool:
    name = str(getattr(attn_type, "value", attn_type)).lower().rsplit(".", 1)[-1]
    return name == "decoder"


def make_forward_v0(cfg: Dict[str, Any], ops: Optional[HookOps] = None):
    """The v0 engine's FlashAttentionImpl.forward replacement
    (patches/patch_loader_vllm_0_10_0.py:78-376), closed over ``cfg``:

    * the step's key / value rows go into the paged cache at ``slot_mapping``
      when the cache is allocated (:139-172), an fp8 cache with the layer's scales;
    * the batch's first ``num_prefill_tokens`` query rows are prefill, the
      ``num_decode_tokens`` after them decode (:186-195);
    * prefill without block tables (or with an empty cache) is FlashPrefill
      over the step's own rows, cu_seqlens = ``seq_start_loc`` and
      max_seq_len = ``max_prefill_seq_len`` (:197-246); prefill with block
      tables (prefix caching) is paged attention over the cache, queries
      ending at ``seq_lens_tensor`` (:270-295), ``ops.decode``'s operation;
    * decode is paged attention over the cache: varlen with
      ``query_start_loc`` when ``max_decode_query_len > 1`` (:313-339), one
      query per sequence otherwise (:340-368).

    Attention types other than decoder go to ``ops.encoder``, cache write
    included (the reference writes encoder-decoder layers through
    ``cross_slot_mapping`` and then runs them through the same causal
    FlashPrefill call, which only suits decoder layers); fused output
    quantisation is rejected (:108-111)."""
    ops = ops or HookOps()

    def flash_prefill_forward_v0(self, layer, query, key, value, kv_cache, attn_metadata,
                                 output=None, output_scale=None):
        if output is None:
            raise ValueError("Output tensor must be provided.")
        if output_scale is not None:
            raise NotImplementedError("fused output quantization is not supported")
        attn_type = getattr(self, "attn_type", "decoder")
        if not _is_decoder(attn_type):
            if ops.encoder is None:
                raise NotImplementedError("encoder and encoder-decoder attention are left to "
                                          "vLLM's backend")
            return ops.encoder(self, query, key, value, output, attn_metadata, layer)
        scale = getattr(self, "scale", 1.0 / math.sqrt(query.shape[-1]))
        key_cache = value_cache = None
        decode = ops.decode
        if kv_cache.numel() > 0:
            key_cache, value_cache, cache_write, decode = _cache_ops(self, layer, ops,
                                                                     kv_cache[0], kv_cache[1])
            if key is not None and value is not None:
                cache_write(key, value, key_cache, value_cache,
                            attn_metadata.slot_mapping.flatten())
        n_pre = attn_metadata.num_prefill_tokens
        n_dec = attn_metadata.num_decode_tokens
        prefill_meta = attn_metadata.prefill_metadata
        if prefill_meta is not None:
            tables = getattr(prefill_meta, "block_tables", None)
            if kv_cache.numel() == 0 or tables is None or tables.numel() == 0:
                ops.prefill(query[:n_pre], key[:n_pre], value[:n_pre], output[:n_pre],
                            prefill_meta.seq_start_loc, prefill_meta.max_prefill_seq_len,
                            cfg["alpha"], cfg["block_size"], cfg["attention_sink"],
                            cfg["window_size"], cfg["last_n_full_block"])
            else:  # prefix caching: the new queries end each cached sequence
                decode(query[:n_pre], key_cache, value_cache, output[:n_pre],
                       prefill_meta.query_start_loc, prefill_meta.seq_lens_tensor, tables, scale)
        decode_meta = attn_metadata.decode_metadata
        if decode_meta is not None:
            dq = query[n_pre:n_pre + n_dec]
            dout = output[n_pre:n_pre + n_dec]
            if (decode_meta.max_decode_query_len or 1) > 1:
                cu = decode_meta.query_start_loc
            else:  # one query per sequence
                cu = torch.arange(decode_meta.seq_lens_tensor.numel() + 1, dtype=torch.int32,
                                  device=query.device)
            decode(dq, key_cache, value_cache, dout, cu, decode_meta.seq_lens_tensor,
                   decode_meta.block_tables, scale)
        return output

    return flash_prefill_forward_v0


def apply_patch_v0(impl_cls=None, config: str = DEFAULT_CONFIG, ops: Optional[HookOps] = None):
    """Replace ``impl_cls.forward`` (default: the v0 engine's
    FlashAttentionImpl, imported from either module path the reference tries,
    patch_loader_vllm_0_10_0.py:57-61) with the v0 FlashPrefill forward for
    ``config``; returns the original forward."""
    if impl_cls is None:
        try:
            import vllm.attention.backends.flash_attn as fa_backend  # noqa: WPS433
        except ImportError:
            import vllm.model_executor.layers.attention.backends.flash_attn as fa_backend  # noqa
        impl_cls = fa_backend.FlashAttentionImpl
    if ops is None:
        ops = HookOps()
        try:  # inside vLLM, paged attention is vLLM's own op (patch :19-20, :270-368)
            from vllm.vllm_flash_attn import flash_attn_varlen_func as vllm_fa

            def vllm_paged(q, kc, vc, out, cu, seqused_k, block_table, scale):
                max_q = int((cu[1:] - cu[:-1]).max())
                vllm_fa(q=q, k=kc, v=vc, out=out, cu_seqlens_q=cu, max_seqlen_q=max_q,
                        seqused_k=seqused_k, max_seqlen_k=int(seqused_k.max()),
                        softmax_scale=scale, causal=True, block_table=block_table)
            ops.decode = vllm_paged
        except ImportError:
            pass
    original = impl_cls.forward
    impl_cls.forward = make_forward_v0(ATTENTION_CONFIGS[config], ops)
    return original

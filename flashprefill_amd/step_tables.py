"""Tables of a serving step over a paged KV cache, built on the GPU from the requests'
lengths (``fp_build_step_tables``): pages given back and taken, the block table, the slots
that ``reshape_and_cache`` writes, the offsets and lengths that ``paged_decode_attention``
reads and the positions that ``apply_rotary`` turns by. The host needs no length, so a
captured step admits, extends and ends requests by writing two small tensors."""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from . import vllm_backend as vb


def build_step_tables(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                      free_pages: torch.Tensor, num_free: torch.Tensor, block_size: int,
                      cu_seqlens: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                      granted: torch.Tensor, *, finished: Optional[torch.Tensor] = None,
                      seq_lens_out: Optional[torch.Tensor] = None,
                      num_free_out: Optional[torch.Tensor] = None) -> None:
    """Make a step's tables on the current stream, without a host synchronisation.

    Row r of ``block_table`` (R, W) holds a request of ``seq_lens[r]`` cached tokens in its
    first ``ceil(seq_lens[r] / block_size)`` pages, and is to get ``new_lens[r]`` more.
    ``free_pages[:num_free]`` are the cache's free pages. All of these are int32 on one
    GPU; ``num_free`` has one entry.

    * ``finished`` (R,; bool or uint8): rows whose request has ended. Their pages go behind
      the free ones in the order of the rows, their length becomes 0; new tokens start
      another request there. (A row whose pages would not fit ``free_pages`` stays, and is
      granted nothing.)
    * Written: ``cu_seqlens`` (R + 1,) int32, where the rows' tokens begin, clamped to the
      room for tokens N; ``granted`` (R,) int32, 1 where the tokens got their places, i.e.
      they fit N and the table's width, and either need no new page or belong to the first
      rows that do whose needs the free pages serve together; ``block_table``, the pages taken behind the
      row's own, from the free ones' end on; ``positions`` and ``slots`` (N,) int64: each
      token's position, and its slot ``page * block_size + position % block_size``, or -1
      for rows that were granted nothing. Behind the last token they are 0 and -1 (padding).
    * ``seq_lens_out`` and ``num_free_out`` (by default ``seq_lens`` and ``num_free``): the
      lengths with the granted tokens, and the free pages left.

    With outputs of their own the call may be made again with other ``new_lens``. Rows with
    a negative length, or one past the table's width, are granted nothing. Under a trace or a
    dispatch mode the tables are made of torch operations."""
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be (requests, width), got {tuple(block_table.shape)}")
    R, W = block_table.shape
    seq_lens_out = seq_lens if seq_lens_out is None else seq_lens_out
    num_free_out = num_free if num_free_out is None else num_free_out
    dev, N = block_table.device, positions.numel()
    for name, t, size, dtype in (
            ("seq_lens", seq_lens, R, torch.int32), ("new_lens", new_lens, R, torch.int32),
            ("num_free", num_free, 1, torch.int32), ("cu_seqlens", cu_seqlens, R + 1, torch.int32),
            ("granted", granted, R, torch.int32), ("seq_lens_out", seq_lens_out, R, torch.int32),
            ("num_free_out", num_free_out, 1, torch.int32),
            ("free_pages", free_pages, None, torch.int32),
            ("positions", positions, N, torch.int64), ("slots", slots, N, torch.int64)):
        if t.dtype != dtype or t.dim() != 1 or (size is not None and t.numel() != size):
            raise ValueError(f"{name} must be {dtype} with {'any number of' if size is None else size}"
                             f" entries, got {t.dtype} {tuple(t.shape)}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if not t.is_cuda or t.device != dev:
            raise ValueError("all tensors must be on one GPU")
    if block_table.dtype != torch.int32 or (W > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 with contiguous rows, got {block_table.dtype}, "
                         f"strides {block_table.stride()}")
    if finished is not None:
        if finished.dtype not in (torch.bool, torch.uint8) or finished.shape != (R,) or \
                finished.device != dev or not finished.is_contiguous():
            raise ValueError(f"finished must be contiguous bool or uint8 ({R},) on {dev}, got "
                             f"{finished.dtype} {tuple(finished.shape)}")
    if block_size < 1:
        raise ValueError(f"block_size must be positive, got {block_size}")
    written = [block_table, free_pages, cu_seqlens, positions, slots, granted, seq_lens_out,
               num_free_out]
    vb._check_written(block_table)
    for t in written:  # (the others are contiguous, and of integers)
        if t.is_inference():
            vb._check_written(t)
    torch_only = vb._torch_only()
    named = [new_lens, *written]
    if finished is not None:
        named.append(finished)
    if seq_lens is not seq_lens_out and \
            vb._place(seq_lens, torch_only) != vb._place(seq_lens_out, torch_only):
        named.append(seq_lens)
    if num_free is not num_free_out and \
            vb._place(num_free, torch_only) != vb._place(num_free_out, torch_only):
        named.append(num_free)
    places = [vb._place(t, True) if torch_only else t.data_ptr() for t in named if t.numel()]
    if len(set(places)) < len(places):
        raise ValueError("the tensors must be memory of their own (but seq_lens_out and "
                         "num_free_out may be seq_lens and num_free)")
    if torch_only:
        build_step_tables_reference(seq_lens, new_lens, block_table, free_pages, num_free,
                                    block_size, cu_seqlens, positions, slots, granted,
                                    finished=finished, seq_lens_out=seq_lens_out,
                                    num_free_out=num_free_out)
        return
    lib = _lib.load()
    a = _lib.FpStepsArgs(
        seq_lens.data_ptr(), new_lens.data_ptr(),
        None if finished is None else finished.data_ptr(), block_table.data_ptr(),
        block_table.stride(0) if R > 1 else W, free_pages.data_ptr(), num_free.data_ptr(),
        seq_lens_out.data_ptr(), num_free_out.data_ptr(), cu_seqlens.data_ptr(),
        positions.data_ptr(), slots.data_ptr(), granted.data_ptr(), N, R, W, free_pages.numel(),
        block_size)
    n = lib.fp_steps_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    vb._launch(dev, lib.fp_build_step_tables, ctypes.byref(a), None if ws is None else ws.data_ptr())
    torch.autograd.graph.increment_version(written)


@torch.no_grad()
def build_step_tables_reference(seq_lens, new_lens, block_table, free_pages, num_free, block_size,
                                cu_seqlens, positions, slots, granted, *, finished=None,
                                seq_lens_out=None, num_free_out=None) -> None:
    """The torch composition of ``build_step_tables``, what a trace or a dispatch mode sees
    of it."""
    (R, W), P, N, dev = block_table.shape, free_pages.numel(), slots.numel(), block_table.device
    length, add = seq_lens.long(), new_lens.long()
    free = num_free.long().clamp(0, P)
    done = torch.zeros(R, dtype=torch.bool, device=dev) if finished is None else finished.bool()
    column = torch.arange(W, device=dev)
    ok = (length >= 0) & (length <= W * block_size)

    def pages(n):
        return (n + block_size - 1) // block_size

    back = torch.where(done & ok, pages(length), 0)
    behind = back.cumsum(0)
    ends = done & ok & ((back == 0) | (behind <= P - free))
    back = torch.where(ends, back, 0)
    moved = column < back.view(-1, 1)
    at = free + (behind - back).view(-1, 1) + column
    free_pages[at[moved]] = block_table[moved]
    free = free + back.sum()
    length = torch.where(ends, 0, length)
    n = add.clamp(min=0)
    end = n.cumsum(0)
    fits = ok & (add >= 0) & (done == ends) & (end <= N) & (length + n <= W * block_size)
    held = torch.where(ok, pages(length), 0)
    need = torch.where(fits, pages(length + n) - held, 0)
    upto = need.cumsum(0)
    yes = fits & ((need == 0) | (upto <= free))
    need = torch.where(yes, need, 0)
    moved = (column >= held.view(-1, 1)) & (column < (held + need).view(-1, 1))
    at = free - 1 - (upto - need).view(-1, 1) - (column - held.view(-1, 1))
    block_table[moved] = free_pages[at[moved]]
    (num_free if num_free_out is None else num_free_out).copy_(free - need.sum())
    (seq_lens if seq_lens_out is None else seq_lens_out).copy_(torch.where(yes, length + n, length))
    granted.copy_(yes)
    cu_seqlens[:1] = 0
    cu_seqlens[1:] = end.clamp(max=N)
    row = torch.arange(N, device=dev)
    r = torch.bucketize(row, cu_seqlens.long(), right=True) - 1
    inside = r < R
    if R == 0 or W == 0:
        positions.zero_()
        slots.fill_(-1)
        if R == 0:
            return
    r = r.clamp(max=R - 1)
    position = torch.where(inside, length[r] + row - (end - n)[r], 0)
    positions.copy_(position)
    if W == 0:
        return
    placed = inside & yes[r]
    at = torch.where(placed, position, 0)
    slot = block_table[r, at // block_size].long() * block_size + at % block_size
    slots.copy_(torch.where(placed, slot, -1))

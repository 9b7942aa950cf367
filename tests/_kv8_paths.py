"""Which kernels a call of attention over an 8-bit cache takes, as its workspace tells."""

import ctypes

from flashprefill_amd import _lib


def workspace(tokens, batch, hq, hkv, d, page, width):
    """Bytes of the call's workspace (no memory is touched: addresses are made up)."""
    a = _lib.FpPagedFp8Args()
    b = a.base
    b.q = b.o = b.key_cache = b.value_cache = b.cu_seqlens = b.seqused = b.block_table = 0x10000
    b.q_stride_tok = b.o_stride_tok = hq * d
    b.kc_stride_slot = b.vc_stride_slot = hkv * d
    b.kc_stride_block = b.vc_stride_block = page * hkv * d
    b.q_stride_head = b.o_stride_head = b.kc_stride_head = b.vc_stride_head = d
    b.table_stride, b.num_tokens, b.num_blocks = width, tokens, 4
    b.batch, b.table_width, b.block_size = batch, width, page
    b.num_q_heads, b.num_kv_heads, b.head_dim = hq, hkv, d
    a.format = _lib.FP_CACHE_E4M3
    return _lib.load().fp_paged_fp8_workspace_bytes(ctypes.byref(a))


def path(tokens, batch, hq, hkv, d, page, width):
    """"rows" (the many-row kernel, one chunk), "rows merged" (several chunks), "shared"
    (few rows, workgroups that share the keys) or "whole" (a segment per workgroup)."""
    n = workspace(tokens, batch, hq, hkv, d, page, width)
    g, room = hq // hkv, width * page
    pair = 2 if d == 64 and hkv % 2 == 0 else 1
    tiles = min(tokens * ((g + 15) // 16), tokens * g // 16 + batch)
    groups = min(512, max(1, tiles * (hkv // pair)) * max(1, -(-room // 128)))
    shared = groups * 2 * 16 * pair * (d + 2) * 4
    if n == 0:
        many = tokens * g >= 32 * batch if d <= 128 else tokens * g >= 128 * batch and room > 1024
        return "rows" if many else "whole"
    # (partials of chunks: rows x chunks, which no case here has equal to the above)
    return "shared" if n == shared else "rows merged"

"""CPU tests of what the 8-bit KV cache's operators refuse or leave to torch operations."""

from types import SimpleNamespace

import pytest
import torch

from tests._kv8 import E4M3, E5M2
from flashprefill_amd import vllm_backend as vb

BF = torch.bfloat16


def _step(queries, max_query_len=1):
    return SimpleNamespace(num_actual_tokens=queries, max_query_len=max_query_len,
                           query_start_loc=torch.arange(queries + 1, dtype=torch.int32),
                           seq_lens=torch.full((queries,), 5), slot_mapping=torch.arange(queries),
                           block_table=torch.zeros(queries, 2, dtype=torch.int32), use_cascade=False)


@pytest.mark.parametrize("qdtype", [E4M3, E5M2, torch.float8_e4m3fnuz, torch.uint8])
def test_queries_of_8_bits_are_refused_by_an_8_bit_cache(qdtype):
    """Their codes mean nothing without the layer's query scale."""
    q = torch.ones(2, 4, 8).to(qdtype)
    cache = torch.zeros(6, 4, 2, 8, dtype=torch.uint8).view(E4M3)
    out = torch.full((2, 4, 8), 7.0, dtype=BF)
    args = (q, cache, cache, out, torch.arange(3), torch.tensor([5, 5]), torch.zeros(2, 2).int(), 0.3)
    for fn in (vb.paged_decode_attention, vb.paged_attention_reference):
        with pytest.raises(NotImplementedError, match="query"):
            fn(*args)
    # through the hooked forwards (the cache write, a kernel, stands aside)
    ops = vb.HookOps(cache_write_fp8=lambda *a: None)
    impl = SimpleNamespace(kv_cache_dtype="fp8", scale=0.3)
    layer = SimpleNamespace(_q_scale=torch.tensor(0.05), _k_scale=torch.tensor(0.5),
                            _v_scale=torch.tensor(0.5))
    kv, k = torch.zeros(2, 6, 4, 2, 8, dtype=torch.uint8), torch.ones(2, 2, 8, dtype=BF)
    cfg = vb.ATTENTION_CONFIGS["flashprefill_llama"]
    with pytest.raises(NotImplementedError, match="query"):
        vb.make_forward(cfg, ops)(impl, layer, q, k, k, kv, _step(2), output=out)
    v0 = SimpleNamespace(num_prefill_tokens=0, num_decode_tokens=2, prefill_metadata=None,
                         slot_mapping=torch.arange(2),
                         decode_metadata=SimpleNamespace(
                             max_decode_query_len=1, seq_lens_tensor=torch.tensor([5, 5]),
                             block_tables=torch.zeros(2, 2, dtype=torch.int32)))
    with pytest.raises(NotImplementedError, match="query"):
        vb.make_forward_v0(cfg, ops)(impl, layer, q, k, k, kv, v0, output=out)
    assert (out == 7.0).all()

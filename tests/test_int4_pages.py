"""CPU tests of 4-bit pages whose dimensions of one entry have strides of their own."""

import pytest
import torch

from flashprefill_amd import int4_cache as i4


@pytest.mark.parametrize("hkv,page", [(1, 16), (2, 1), (1, 1)])
def test_pages_of_one_head_or_one_slot(hkv, page):
    row = i4.int4_row_bytes(64)
    store = torch.zeros(3 * page * hkv * row, dtype=torch.uint8)
    want = i4.int4_cache_views(store.view(3, page, hkv, row))
    strides = (page * hkv * row, 7 if page == 1 else hkv * row, 5 if hkv == 1 else row, 1)
    for a, b in zip(i4.int4_cache_views(store.as_strided((3, page, hkv, row), strides)), want):
        assert a.shape == b.shape and a.data_ptr() == b.data_ptr()
        a.fill_(1)
        assert (b == 1).all()
    with pytest.raises(ValueError, match="contiguous"):
        i4.int4_cache_views(torch.zeros(3, 2 * page + 2, hkv, row, dtype=torch.uint8)[:, ::2])

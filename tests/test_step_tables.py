"""CPU tests of a serving step's tables: the torch composition against plain Python, and
what the entry points refuse."""

import ctypes

import pytest
import torch

from flashprefill_amd import _lib
from flashprefill_amd.step_tables import build_step_tables, build_step_tables_reference
from tests import _steps as S


@pytest.mark.parametrize("kw", S.CASES, ids=str)
@pytest.mark.parametrize("finished", [True, False])
def test_the_composition(kw, finished):
    args = S.case(seed=kw["R"], **kw)
    want = S.tables(*args[:-1], args[-1] if finished else None)
    for alias in (False, True):
        assert S.call(build_step_tables_reference, args, "cpu", alias, finished) == want


def test_the_composition_of_lengths_that_cannot_be():
    args = S.bad_lengths(S.case(seed=3, R=60, W=20, page=8, room=300, spare=60))
    assert S.call(build_step_tables_reference, args, "cpu") == S.tables(*args)
    assert S.call(build_step_tables_reference, [[], [], [], [3, 1], 2, 8, 4, []], "cpu")["slots"] \
        == [-1] * 4


def _tensors(R=3, W=4, N=8):
    i32 = dict(dtype=torch.int32)
    return dict(seq_lens=torch.zeros(R, **i32), new_lens=torch.ones(R, **i32),
                block_table=torch.zeros(R, W, **i32), free_pages=torch.arange(9, **i32),
                num_free=torch.tensor([9], **i32), block_size=16,
                cu_seqlens=torch.zeros(R + 1, **i32), positions=torch.zeros(N, dtype=torch.int64),
                slots=torch.zeros(N, dtype=torch.int64), granted=torch.zeros(R, **i32))


@pytest.mark.parametrize("bad", [
    dict(seq_lens=torch.zeros(2, dtype=torch.int32)), dict(seq_lens=torch.zeros(3)),
    dict(new_lens=torch.zeros(3, dtype=torch.int64)), dict(block_table=torch.zeros(3, 4)),
    dict(block_table=torch.zeros(12, dtype=torch.int32)),
    dict(block_table=torch.zeros(3, 8, dtype=torch.int32)[:, ::2]),
    dict(num_free=torch.zeros(2, dtype=torch.int32)),
    dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)),
    dict(slots=torch.zeros(7, dtype=torch.int64)), dict(positions=torch.zeros(8, dtype=torch.int32)),
    dict(granted=torch.zeros(6, dtype=torch.int32)[::2]), dict(finished=torch.zeros(2, dtype=torch.bool)),
    dict(finished=torch.zeros(3)), dict(), dict(seq_lens_out=torch.zeros(4, dtype=torch.int32))])
def test_what_is_refused(bad):
    with pytest.raises(ValueError):  # (none of them at last: the CPU)
        build_step_tables(**dict(_tensors(), **bad))


def _args(**kw):
    a = _lib.FpStepsArgs()
    for f in ("seq_lens", "new_lens", "block_table", "free_pages", "num_free", "seq_lens_out",
              "num_free_out", "cu_seqlens", "positions", "slots", "granted"):
        setattr(a, f, 0x10000)
    a.table_stride, a.num_tokens, a.requests, a.table_width, a.num_pages, a.block_size = \
        9000, 9000, 3, 4, 9, 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(requests=-1), _lib.FP_E_INVALID_ARG), (dict(block_size=0), _lib.FP_E_INVALID_ARG),
    (dict(num_tokens=-1), _lib.FP_E_INVALID_ARG), (dict(num_free=0), _lib.FP_E_INVALID_ARG),
    (dict(slots=0), _lib.FP_E_INVALID_ARG), (dict(block_table=0), _lib.FP_E_INVALID_ARG),
    (dict(num_tokens=1 << 31), _lib.FP_E_UNSUPPORTED),
    (dict(table_width=1 << 28), _lib.FP_E_UNSUPPORTED),
    (dict(requests=1 << 20, table_width=1 << 12), _lib.FP_E_UNSUPPORTED),
    (dict(), _lib.FP_E_INVALID_ARG)])
def test_the_c_entry_refuses(kw, code):
    lib = _lib.load()
    assert lib.fp_build_step_tables(ctypes.byref(_args(**kw)), None, None) == code
    assert lib.fp_build_step_tables(None, None, None) == _lib.FP_E_INVALID_ARG


def test_workspace():
    size = _lib.load().fp_steps_workspace_bytes
    assert size(ctypes.byref(_args())) == 16 + 12 * 3
    assert size(ctypes.byref(_args(num_tokens=8192))) == 0
    assert size(ctypes.byref(_args(num_tokens=1, requests=1025))) == 16 + 12 * 1025
    assert size(ctypes.byref(_args(block_size=0))) == 0

"""GPU tests of steps of few tokens in which long requests end: tens of thousands of pages come
back, in rows of every length, against plain Python."""

import pytest
import torch

from flashprefill_amd.step_tables import build_step_tables
from tests import _steps as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [
    dict(R=24, W=6000, page=4, room=200, spare=100, end=0.9),
    dict(R=1000, W=300, page=2, room=3000, spare=500, end=0.6),
    dict(R=5, W=40000, page=1, room=64, spare=0, end=0.95, most_new=5),
    dict(R=300, W=400, page=16, room=8000, spare=9, end=0.9, pool=20000)], ids=str)
def test_many_pages_come_back(kw):
    args = S.case(seed=kw["R"], **kw)
    want = S.tables(*args)
    back = sum(-(-n // kw["page"]) for n, d in zip(args[0], args[-1]) if d)
    assert back > 16384
    for alias in (False, True):
        got = S.call(build_step_tables, args, "cuda", alias)
        for k in want:
            assert got[k] == want[k], k


@pytest.mark.parametrize("pages", [16383, 16384, 16385, 17407, 17408, 17409, 32768])
def test_one_row_of_pages(pages):
    """Rows that end at, before and after what a wave moves at a time, beside short ones."""
    g = torch.Generator().manual_seed(pages)
    lens = [3, pages - 10, 0, 5, 9]
    perm = torch.randperm(pages + 20, generator=g).tolist()
    table, at = [], 0
    for n in lens:
        table.append(perm[at:at + n] + [-1] * (pages - n))
        at += n
    free = perm[at:] + [-9] * at
    args = [lens, [1, 2, 1, 1, 1], table, free, len(perm) - at, 1, 8,
            [True, True, True, True, False]]
    want = S.tables(*args)
    got = S.call(build_step_tables, args, "cuda")
    for k in want:
        assert got[k] == want[k], k

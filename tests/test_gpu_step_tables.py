"""GPU tests of a serving step's tables against plain Python: one launch and several,
captured and replayed, and a server's steps one after the other."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from flashprefill_amd.step_tables import build_step_tables
from tests import _steps as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", S.CASES, ids=str)
@pytest.mark.parametrize("finished", [True, False])
def test_tables(kw, finished):
    args = S.case(seed=kw["R"], **kw)
    want = S.tables(*args[:-1], args[-1] if finished else None)
    for alias in (False, True):
        got = S.call(build_step_tables, args, "cuda", alias, finished)
        for k in want:
            assert got[k] == want[k], k


@pytest.mark.parametrize("room", [300, 9000])
def test_lengths_that_cannot_be(room):
    args = S.bad_lengths(S.case(seed=3, R=60, W=20, page=8, room=room, spare=60))
    assert S.call(build_step_tables, args, "cuda") == S.tables(*args)
    args[4] = 10 ** 6  # more free pages than there is room for
    assert S.call(build_step_tables, args, "cuda") == S.tables(*args)
    none = S.call(build_step_tables, [[], [], [], [3, 1], 2, 8, room, []], "cuda")
    assert none["slots"] == [-1] * room and none["cu"] == [0] and none["num_free"] == [2]


def test_slots_past_32_bits():
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.full((1, 4), -1, **i32)
    slots = torch.empty(70, dtype=torch.int64, device="cuda")
    positions = torch.empty_like(slots)
    build_step_tables(torch.zeros(1, **i32), torch.tensor([70], **i32), table,
                      torch.tensor([2 ** 31 - 1, 2 ** 30], **i32), torch.tensor([2], **i32), 64,
                      torch.empty(2, **i32), positions, slots, torch.empty(1, **i32))
    assert slots.tolist() == [2 ** 30 * 64 + i for i in range(64)] + \
        [(2 ** 31 - 1) * 64 + i for i in range(6)]


class Seen(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_a_dispatch_mode_sees_torch_operations():
    args = S.case(seed=1, R=20, W=9, page=8, room=100, spare=30)
    with Seen():
        got = S.call(build_step_tables, args, "cuda")
    assert got == S.tables(*args)


@pytest.mark.parametrize("R,N", [(40, 400), (1500, 9000)])
def test_a_servers_steps_captured_and_replayed(R, N):
    # one graph makes every step's tables in place; the host keeps its own books
    page, W = 8, 12
    g = torch.Generator().manual_seed(R)
    P = R * 5
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, new, table = torch.zeros(R, **i32), torch.zeros(R, **i32), torch.full((R, W), -1, **i32)
    free = torch.randperm(P, generator=g).to(**i32)
    num_free, cu, granted = torch.tensor([P], **i32), torch.empty(R + 1, **i32), torch.empty(R, **i32)
    pos, slots = (torch.empty(N, dtype=torch.int64, device="cuda") for _ in range(2))
    done = torch.zeros(R, dtype=torch.bool, device="cuda")

    def step():
        build_step_tables(lens, new, table, free, num_free, page, cu, pos, slots, granted,
                          finished=done)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # (no tokens yet: changes nothing)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    books = [[0] * R, None, table.tolist(), free.tolist(), P, page, N, None]
    for i in range(12):
        share = N // R + 1 if i % 3 else 4 * page
        books[1] = [x if z else 0 for x, z in zip(
            torch.randint(0, 2 * share, (R,), generator=g).tolist(),
            torch.randint(0, 3, (R,), generator=g).tolist())]
        books[7] = (torch.rand(R, generator=g) < 0.15).tolist()
        new.copy_(torch.tensor(books[1]))
        done.copy_(torch.tensor(books[7]))
        graph.replay()
        want = S.tables(*books)
        got = {"cu": cu, "granted": granted, "positions": pos, "slots": slots, "seq_lens": lens,
               "num_free": num_free, "table": table, "free_pages": free}
        for k, v in got.items():
            assert v.tolist() == want[k], (i, k)
        books[0], books[2], books[3], books[4] = (want["seq_lens"], want["table"],
                                                  want["free_pages"], want["num_free"][0])
        owned = [p for r in range(R) for p in want["table"][r][:-(-want["seq_lens"][r] // page)]]
        owned += want["free_pages"][:want["num_free"][0]]
        assert sorted(owned) == list(range(P))  # every page has one owner
        torch.cuda.synchronize()

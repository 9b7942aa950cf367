"""A serving step's tables as plain Python, request by request."""

import torch


def tables(seq_lens, new_lens, table, free_pages, num_free, page, room, finished=None):
    """What ``build_step_tables`` writes, from lists (table: rows of page numbers): a dict of
    lists; N = room."""
    R, W, P = len(seq_lens), len(table[0]) if table else 0, len(free_pages)
    table, free_pages = [list(r) for r in table], list(free_pages)
    finished = finished or [False] * R
    lens, free = list(seq_lens), min(max(num_free, 0), P)
    ok = [0 <= n <= W * page for n in lens]
    stays, top, full = [False] * R, free, False
    for r in range(R):
        if not finished[r] or not ok[r]:
            stays[r] = bool(finished[r])
            continue
        held = -(-lens[r] // page)
        if held and (full or top + held > P):
            stays[r] = full = True
            continue
        free_pages[top:top + held] = table[r][:held]
        top, lens[r] = top + held, 0
    out = {"cu": [0], "granted": [], "positions": [], "slots": []}
    at, short = 0, False
    for r in range(R):
        n = max(new_lens[r], 0)
        fits = ok[r] and new_lens[r] >= 0 and not stays[r] and at + n <= room and \
            lens[r] + n <= W * page
        need = -(-(lens[r] + n) // page) - -(-lens[r] // page) if fits else 0
        yes = fits and (need == 0 or (not short and need <= top))
        short = short or (fits and not yes)
        if yes:
            held = -(-lens[r] // page)
            for j in range(need):
                top -= 1
                table[r][held + j] = free_pages[top]
        for i in range(n):
            if at + i < room:
                p = lens[r] + i
                out["positions"].append(p)
                out["slots"].append(table[r][p // page] * page + p % page if yes else -1)
        at += n
        out["cu"].append(min(at, room))
        out["granted"].append(int(yes))
        lens[r] += n if yes else 0
    pad = room - len(out["positions"])
    out["positions"] += [0] * pad
    out["slots"] += [-1] * pad
    return dict(out, seq_lens=lens, num_free=[top], table=table, free_pages=free_pages)


def case(R, W, page, room, spare, seed, end=0.2, most_new=None, pool=None):
    """Arguments of ``tables`` with consistent pages, requests of every size among them."""
    g = torch.Generator().manual_seed(seed)

    def ints(lo, hi, n):
        return torch.randint(lo, hi, (n,), generator=g).tolist()

    lens = [n if z else 0 for n, z in zip(ints(0, max(1, W * page * 2 // 3), R), ints(0, 4, R))]
    new = [x if z == 0 else min(x, 1) for x, z in
           zip(ints(0, (most_new or 3 * page) + 1, R), ints(0, 3, R))]
    held = [-(-n // page) for n in lens]
    P = sum(held) + spare
    perm = torch.randperm(P, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(perm[at:at + h] + [-7] * (W - h))
        at += h
    free = perm[at:] + [-9] * (P - spare)
    done = [x < end for x in torch.rand(R, generator=g).tolist()]
    return [lens, new, table, free[:P if pool is None else pool], spare, page, room, done]


def call(fn, args, device, alias=False, use_finished=True):
    """``fn`` (build_step_tables or its composition) on tensors of ``args``: the dict of
    ``tables``."""
    lens, new, table, free, num_free, page, room, done = args

    def t(x, dtype=torch.int32):
        return torch.tensor(x, dtype=dtype, device=device)

    R = len(lens)
    tab = t(table).view(R, -1) if R else t([]).view(0, 4)
    lens, new, free, num_free = t(lens), t(new), t(free), t([num_free])
    out = {"cu": t([-5] * (R + 1)), "granted": t([-5] * R), "positions": t([-5] * room, torch.int64),
           "slots": t([-5] * room, torch.int64)}
    lo, no = (lens, num_free) if alias else (torch.full_like(lens, -5), torch.full_like(num_free, -5))
    fn(lens, new, tab, free, num_free, page, out["cu"], out["positions"], out["slots"],
       out["granted"], finished=t(done, torch.bool) if use_finished else None,
       **({} if alias else {"seq_lens_out": lo, "num_free_out": no}))
    out = {k: v.tolist() for k, v in out.items()}
    return dict(out, seq_lens=lo.tolist(), num_free=no.tolist(), table=tab.tolist(),
                free_pages=free.tolist())


# requests, width, page, tokens, spare pages, then others by name
CASES = [dict(R=1, W=4, page=16, room=20, spare=3), dict(R=7, W=5, page=4, room=40, spare=6),
         dict(R=64, W=30, page=16, room=700, spare=40), dict(R=64, W=30, page=1, room=90, spare=25),
         dict(R=300, W=9, page=24, room=9000, spare=2000, most_new=60),
         dict(R=1024, W=6, page=8, room=3000, spare=700),
         dict(R=1025, W=6, page=8, room=20000, spare=4000),
         dict(R=2500, W=12, page=5, room=9000, spare=500, end=0.5),
         dict(R=40, W=700, page=16, room=60000, spare=900, most_new=5000),
         dict(R=33, W=8, page=16, room=300, spare=0), dict(R=20, W=8, page=16, room=0, spare=9),
         dict(R=50, W=8, page=16, room=500, spare=20, end=0.6, pool=160)]


def bad_lengths(args):
    """The same with lengths that cannot be: negative ones and some past the table."""
    lens, new, table = list(args[0]), list(args[1]), args[2]
    for r in range(0, len(lens), 5):
        lens[r] = -1 - r if r % 2 else len(table[0]) * args[5] + 1 + r
    for r in range(2, len(lens), 7):
        new[r] = -3
    return [lens, new, *args[2:]]

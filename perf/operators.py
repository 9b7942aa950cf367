"""The 8-bit KV cache's operators as performance cases, with their plain forms.

Three kinds of case, all of the serving hook's paged cache held as 8-bit floats
(e4m3 or e5m2) with scales:

* ``write``: ``reshape_and_cache`` of a step's key / value rows, which come as
  views of one QKV projection, into the slots of the pages; ``attend``:
  ``paged_decode_attention`` over the pages, decode steps (one query per
  sequence), several queries each, and prefill whose prefix is cached;
  ``gather``: ``gather_cache``, the cached tokens of each sequence read back as
  16-bit rows.

``scales``: "tensor" (one fp32 value), "head" (one per KV head), both fixed by a
calibration, or "slot" (one per token and head, found as the row is written).

``own`` chooses between the plain form (elementary torch operations in 32 bits)
and the framework's entry points. ``listed()`` names the fixed cases,
``draw(rng)`` gives further ones, ``prepare`` makes what a program holds before
the call, ``run`` is one pass, ``work`` the bytes and operations that it cannot
do without, ``exact`` the same outputs in 64 bits.
"""

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# format: type, largest finite value
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0), "e5m2": (torch.float8_e5m2, 57344.0)}


def _case(kind, name, lens, hq, hkv, d, dtype="bf16", fmt="e4m3", scales="tensor", page=16, new=0,
          starts=False):
    case = {"kind": kind, "lens": ",".join(str(int(n)) for n in lens), "new": new, "hq": hq,
            "hkv": hkv, "d": d, "dtype": dtype, "fmt": fmt, "scales": scales, "page": page,
            "starts": starts}
    if name:
        case["name"] = name
    return case


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def listed():
    return [
        # the new tokens of a decode step of 32 running requests: a launch, little data
        _case("write", "write_decode_32", [1] * 32, 32, 8, 128),
        # a serving step of ragged prompts, scales found per token and head
        _case("write", "write_ragged_prompts", [9001, 4408, 1023, 129, 1], 28, 4, 128,
              scales="slot"),
        # one long-context prompt, calibrated scales per head
        _case("write", "write_prompt_128k", [131072], 32, 8, 128, scales="head"),
        # decode of one short chat: latency of the call
        _case("attend", "decode_one_short", [333], 32, 8, 128, new=1),
        # a decode step of 32 running requests of mixed context lengths
        _case("attend", "decode_32", [(211 + 977 * i * i) % 15000 + 300 for i in range(32)],
              32, 8, 128, new=1),
        # decode of one long request: too few sequences to fill the card by themselves
        _case("attend", "decode_one_long", [65000], 32, 8, 128, scales="slot", new=1),
        # wide heads in fp16, the format with more exponent bits, larger pages
        _case("attend", "decode_wide_fp16", [(137 + 701 * i * i) % 6000 + 77 for i in range(16)],
              16, 4, 256, dtype="fp16", fmt="e5m2", scales="head", page=64, new=1),
        # several queries per sequence (drafted tokens to be verified), head_dim 64
        _case("attend", "verify_4_of_16", [(411 + 1377 * i * i) % 9000 + 40 for i in range(16)],
              32, 8, 64, scales="slot", new=4),
        # prompts whose prefix is cached: the new tokens attend over the pages
        _case("attend", "prefix_prefill", [6144, 2500, 1111], 28, 4, 128, scales="slot", new=500),
        # long new parts over a cached prefix
        _case("attend", "prefix_prefill_long", [6144, 5000, 4321, 4096], 32, 8, 128, new=2048),
        # a few cached prefixes read back, from the middle on
        _case("gather", "read_back_ragged", [700, 65, 1, 2311], 28, 4, 128, scales="slot",
              starts=True),
        # every running request's cache read back
        _case("gather", "read_back_32", [(211 + 977 * i * i) % 15000 + 300 for i in range(32)],
              32, 8, 128, scales="head"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "gather"])
    hq, hkv = rng.choice([(32, 8), (28, 4), (32, 4), (8, 2), (16, 1), (8, 8)])
    d = rng.choice([64, 128, 128, 256])
    more = {"dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "fmt": rng.choice(["e4m3", "e4m3", "e5m2"]),
            "scales": rng.choice(["tensor", "head", "slot"]),
            "page": rng.choice([16, 16, 24, 32, 64, 128])}
    # what the widest heads of a case cost beside 8 of 128
    share = max(1, hkv * d // 1024)
    n = _log_uniform(rng, 1, 32)
    if kind == "attend":
        pick = rng.random()
        if pick < 0.55:
            new, top = 1, 15000 // share
        elif pick < 0.75:
            new, top = rng.randint(2, 8), 9000 // share
        else:
            n, top = min(n, 3), 5000
            new = _log_uniform(rng, 9, 700 // share)
        lens = [new + _log_uniform(rng, 1, top) for _ in range(n)]
        return _case(kind, None, lens, hq, hkv, d, new=new, **more)
    if kind == "write":
        lens = [_log_uniform(rng, 1, 100000 // share // n) for _ in range(n)]
    else:
        lens = [_log_uniform(rng, 1, 15000 // share) for _ in range(n)]
        more["starts"] = rng.random() < 0.5
    return _case(kind, None, lens, hq, hkv, d, **more)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _rows(n, heads, d, dtype, g):
    """Rows as projections give them: every token of its own size, and a few
    channels of each head several times as large as the others."""
    x = torch.randn(n, heads, d, generator=g, device="cuda", dtype=dtype)
    x *= torch.exp(0.5 * torch.randn(n, 1, 1, generator=g, device="cuda")).to(dtype)
    wide = (torch.rand(1, heads, d, generator=g, device="cuda") < 0.05).to(dtype)
    return x.mul_(1 + 4 * wide)


def _pages(lens, page, g):
    """Shuffled pages: how many, and the block table (unused entries 0)."""
    need = [(n + page - 1) // page for n in lens]
    perm = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return sum(need), table


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _filled(case, total, g):
    """A cache of `total` pages in use and its scales."""
    fmt, top = FORMATS[case["fmt"]]
    hkv, d, page = case["hkv"], case["d"], case["page"]
    x = _rows(total * page, hkv, d, DTYPES[case["dtype"]], g)
    size = x.abs().amax(-1)  # (tokens, heads)
    if case["scales"] == "slot":
        scale = size.float() / top
        kept = scale.view(total, page, hkv).transpose(1, 2).contiguous()
    else:
        scale = (size.amax(0) if case["scales"] == "head" else size.amax().view(1)).float() / top
        kept, scale = scale, scale.view(1, -1)
    step = max(1, (1 << 28) // (hkv * d))
    cache = torch.cat([(c.float() / (scale[i * step:(i + 1) * step] if scale.shape[0] > 1 else scale
                                     ).unsqueeze(-1)).clamp_(-top, top).to(fmt)
                       for i, c in enumerate(x.split(step))])
    return cache.view(total, page, hkv, d), kept


def prepare(case, seed):
    kind, lens, new, page = case["kind"], _lens(case), case["new"], case["page"]
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    fmt, top = FORMATS[case["fmt"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(1234577 * (seed + 1))
    st = SimpleNamespace(kind=kind, top=top, page=page, new=new, slot=case["scales"] == "slot")
    if kind == "write":
        n = sum(lens)
        qkv = _rows(n, hq + 2 * hkv, d, dtype, g)
        st.key, st.value = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        # the prompts' tokens lie one after the other in shuffled pages, with room
        # left in the cache; a serving engine pads the mapping with slots of -1
        total, table = _pages([m + 20 for m in lens], page, g)
        st.slots = torch.cat([table[b].long().repeat_interleave(page)[:m + page][m % 7:][:m] * page
                              + (torch.arange(m, device="cuda") + m % 7) % page
                              for b, m in enumerate(lens)])
        st.slots[torch.arange(n, device="cuda") % 97 == 96] = -1
        st.key_cache = torch.zeros(total, page, hkv, d, dtype=torch.uint8, device="cuda").view(fmt)
        st.value_cache = torch.zeros_like(st.key_cache)
        if st.slot:
            st.k_scale = torch.zeros(total, hkv, page, device="cuda")
            st.v_scale = torch.zeros(total, hkv, page, device="cuda")
        else:  # calibrated on other rows: a few of these lie beyond the range
            dims = (0, 2) if case["scales"] == "head" else (0, 1, 2)
            st.k_scale = st.key[::5].abs().amax(dims).float().view(-1) / top
            st.v_scale = st.value[::5].abs().amax(dims).float().view(-1) / top
        return st
    total, st.table = _pages(lens, page, g)
    st.key_cache, st.k_scale = _filled(case, total, g)
    st.value_cache, st.v_scale = _filled(case, total, g)
    if kind == "attend":
        n = len(lens) * new
        st.query = torch.randn(n, hq, d, generator=g, device="cuda", dtype=dtype)
        st.out = torch.empty_like(st.query)
        st.cu = torch.arange(0, n + 1, new, dtype=torch.int32, device="cuda")
        st.used = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st.scale = 1 / math.sqrt(d)
        return st
    first = [n // 3 if case["starts"] else 0 for n in lens]
    st.starts = torch.tensor(first, dtype=torch.int32, device="cuda") if case["starts"] else None
    st.cu = _offsets([n - m for n, m in zip(lens, first)])
    # as many rows as a server's buffer has; those behind the last sequence stay
    st.key = torch.ones(sum(lens) - sum(first) + 3, hkv, d, device="cuda", dtype=dtype)
    st.value = torch.ones_like(st.key)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    if st.kind == "write":
        _own_write(st) if own else _plain_write(st)
        out = {"key_cache": st.key_cache, "value_cache": st.value_cache}
        if st.slot:
            out.update(k_scale=st.k_scale, v_scale=st.v_scale)
        return out
    if st.kind == "attend":
        return _own_attend(st) if own else _plain_attend(st)
    _own_gather(st) if own else _plain_gather(st)
    return {"key": st.key, "value": st.value}


def _own_write(st):
    from flashprefill_amd.vllm_backend import reshape_and_cache

    reshape_and_cache(st.key, st.value, st.key_cache, st.value_cache, st.slots,
                      k_scale=st.k_scale, v_scale=st.v_scale)


def _own_attend(st):
    from flashprefill_amd.vllm_backend import paged_decode_attention

    paged_decode_attention(st.query, st.key_cache, st.value_cache, st.out, st.cu, st.used,
                           st.table, st.scale, k_scale=st.k_scale, v_scale=st.v_scale)
    return st.out


def _own_gather(st):
    from flashprefill_amd.vllm_backend import gather_cache

    gather_cache(st.key_cache, st.value_cache, st.key, st.value, st.cu, st.table,
                 starts=st.starts, k_scale=st.k_scale, v_scale=st.v_scale)


def _put(x, cache, scale, page, at, top, slot):
    """Rows x (tokens, heads, d) as 8-bit values at (page, at)."""
    x = x.float()
    if slot:
        size = x.abs().masked_fill(~x.isfinite(), 0.0).amax(-1) / top
        s = torch.where(size > 0, size, torch.ones_like(size))
        scale[page, :, at] = s
    else:
        s = scale.view(1, -1)
    codes = (x / s.unsqueeze(-1)).clamp(-top, top).to(cache.dtype)
    cache.view(torch.uint8)[page, at] = codes.view(torch.uint8)


def _plain_write(st):
    rows = (st.slots >= 0).nonzero().view(-1)
    slots = st.slots[rows]
    page, at = slots // st.page, slots % st.page
    _put(st.key[rows], st.key_cache, st.k_scale, page, at, st.top, st.slot)
    _put(st.value[rows], st.value_cache, st.v_scale, page, at, st.top, st.slot)


def _values(cache, scale, pages, slot):
    """The pages' values in fp32: (*pages.shape, page, heads, d)."""
    x = cache.view(torch.uint8)[pages].view(cache.dtype).float()
    return x * (scale[pages].transpose(-1, -2) if slot else scale).unsqueeze(-1)


def _plain_attend(st):
    B, new = st.used.numel(), st.new
    T, hq, d = st.query.shape
    hkv = st.key_cache.shape[2]
    pages = st.table.long()
    # (B, heads, keys, d)
    k = _values(st.key_cache, st.k_scale, pages, st.slot).flatten(1, 2).transpose(1, 2)
    v = _values(st.value_cache, st.v_scale, pages, st.slot).flatten(1, 2).transpose(1, 2)
    # (B, heads, queries of the head x new, d)
    q = st.query.float().view(B, new, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, hkv, hq // hkv * new, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * st.scale
    key = torch.arange(k.shape[2], device=q.device)
    last = st.used.view(B, 1) - new + torch.arange(new, device=q.device)  # (B, new)
    hidden = (key > last.unsqueeze(-1)).view(B, 1, 1, new, -1)
    s = s.view(B, hkv, hq // hkv, new, -1).masked_fill_(hidden, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True)).flatten(2, 3)
    o = torch.matmul(p, v.contiguous()) / p.sum(-1, keepdim=True)
    o = o.view(B, hkv, hq // hkv, new, d).permute(0, 3, 1, 2, 4).reshape(T, hq, d)
    st.out.copy_(o)
    return st.out


def _plain_gather(st):
    cu = st.cu.long()
    n = torch.arange(st.key.shape[0], device=cu.device)
    b = torch.bucketize(n, cu, right=True) - 1
    rows = (b < cu.numel() - 1).nonzero().view(-1)
    b = b[rows]
    token = rows - cu[b] + (st.starts.long()[b] if st.starts is not None else 0)
    page, at = st.table[b, token // st.page].long(), token % st.page
    for x, cache, scale in ((st.key, st.key_cache, st.k_scale),
                            (st.value, st.value_cache, st.v_scale)):
        y = cache.view(torch.uint8)[page, at].view(cache.dtype).float()
        y = y * (scale[page, :, at] if st.slot else scale).unsqueeze(-1)
        x[rows] = y.to(x.dtype)


# ---------------------------------------------------------------------------
# work and 64-bit results
# ---------------------------------------------------------------------------

def work(case):
    lens, new, d, hq, hkv = _lens(case), case["new"], case["d"], case["hq"], case["hkv"]
    n, slot = sum(lens), case["scales"] == "slot"
    token = 2 * hkv * (d + (4 if slot else 0))  # a token's K and V in the cache, scales included
    pages = sum((m + case["page"] - 1) // case["page"] for m in lens)
    if case["kind"] == "write":
        n -= n // 97
        return {"bytes": n * (4 * hkv * d + token + 8), "flops": 4 * n * hkv * d}
    if case["kind"] == "attend":
        T = len(lens) * new
        seen = sum(new * m - new * (new - 1) // 2 for m in lens)
        return {"bytes": n * token + 4 * pages + 4 * T * hq * d + 8 * len(lens),
                "flops": 4 * seen * hq * d}
    if case["starts"]:
        n = sum(m - m // 3 for m in lens)
    return {"bytes": n * (4 * hkv * d + token) + 4 * pages, "flops": 2 * n * hkv * d}


def exact(case, seed):
    st = prepare(case, seed)
    lens, page, hkv, d = _lens(case), case["page"], case["hkv"], case["d"]
    if case["kind"] == "write":
        out = {}
        at = [(t, s) for t, s in enumerate(st.slots.tolist()) if s >= 0]
        tokens, slots = (torch.tensor(x, device="cuda") for x in zip(*at)) if at else (None, None)
        for name, x, cache in (("key_cache", st.key, st.key_cache),
                               ("value_cache", st.value, st.value_cache)):
            flat = torch.zeros(cache.shape[0] * page, hkv, d, dtype=torch.float64, device="cuda")
            fixed = st.k_scale if name == "key_cache" else st.v_scale
            found = torch.zeros(cache.shape[0] * page, hkv, dtype=torch.float64, device="cuda")
            if at:
                y = x[tokens].double()
                s = y.abs().amax(-1) / st.top if st.slot else fixed.double().view(1, -1)
                found[slots] = s.expand(len(at), hkv)
                flat[slots] = torch.clamp(y / s.unsqueeze(-1), -st.top, st.top)
            out[name] = flat.view(cache.shape)
            if st.slot:
                out["k_scale" if name == "key_cache" else "v_scale"] = found.view(
                    -1, page, hkv).transpose(1, 2).contiguous()
        return out

    def tokens_of(b, cache, scale, lo, hi):
        """Tokens lo .. hi - 1 of sequence b: (tokens, heads, d)."""
        t = torch.arange(lo, hi, device="cuda")
        p, o = st.table[b][t // page].long(), t % page
        x = cache.view(torch.uint8)[p, o].view(cache.dtype).to(torch.float64)
        return x * (scale[p, :, o] if st.slot else scale.view(1, -1)).double().unsqueeze(-1)

    if case["kind"] == "gather":
        key, value = (torch.ones(x.shape, dtype=torch.float64, device="cuda")
                      for x in (st.key, st.value))
        cu = st.cu.tolist()
        for b in range(len(lens)):
            lo = int(st.starts[b]) if st.starts is not None else 0
            hi = lo + cu[b + 1] - cu[b]
            key[cu[b]:cu[b + 1]] = tokens_of(b, st.key_cache, st.k_scale, lo, hi)
            value[cu[b]:cu[b + 1]] = tokens_of(b, st.value_cache, st.v_scale, lo, hi)
        return {"key": key, "value": value}

    new, group = case["new"], case["hq"] // hkv
    out = torch.empty(st.query.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k = tokens_of(b, st.key_cache, st.k_scale, 0, n)
        v = tokens_of(b, st.value_cache, st.v_scale, 0, n)
        after = torch.ones(new, n, dtype=torch.bool, device="cuda").triu(n - new + 1)
        for h in range(case["hq"]):
            q = st.query[b * new:(b + 1) * new, h].double()
            s = (q @ k[:, h // group].t().contiguous()) * st.scale
            s[after] = -math.inf
            out[b * new:(b + 1) * new, h] = torch.softmax(s, -1) @ v[:, h // group].contiguous()
    return out

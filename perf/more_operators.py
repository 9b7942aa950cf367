"""A serving step over a 4-bit KV cache as performance cases, with the plain forms.

Four kinds of case, in the order in which a step of a serving engine makes the calls:

* ``tables``: ``build_step_tables``: the finished requests' pages go back to the
  free ones, the step's tokens get pages from there, and every token its slot and
  its position;
* ``rotate``: ``apply_rotary``: queries and keys, views of one QKV projection, are
  rotated into buffers of their own;
* ``store``: ``reshape_and_cache_int4``, then ``gather_cache_int4`` of the same
  tokens: keys and values as the cache holds them, e.g. handed on as a prefix;
  ``gather``: ``gather_cache_int4`` alone, cached tokens of each sequence as 16-bit
  rows;
* ``attend``: ``paged_decode_attention_int4`` over the pages: decode steps, several
  queries each, and prefill whose prefix is cached.

The 4-bit cache holds groups of 32 consecutive elements of a row. Element x is the
code c (0 .. 15) that stands for s (c + z) t: the group's step s, 4 significant bits
and fp16's exponents, and its zero point z (-64 .. 63) are one 16-bit word, the fp16
bits of s with z + 64 in the seven lowest. t is a fixed fp32 scale of the KV head, or
1. Byte m (d / 32) + j of a row (m < 16) holds dims 32 j + 2 m (low half) and
32 j + 2 m + 1.

``own`` chooses between the plain form (elementary torch operations in 32 bits; 64
for the angles) and the framework's entry points. ``listed()`` names the fixed cases,
``draw(rng)`` gives further ones, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``work`` the bytes and operations that it cannot do
without, ``exact`` the same outputs in 64 bits.
"""

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GROUP = 32  # elements that share a step and a zero point
MOST = 57344.0  # the largest magnitude that a group holds
WIDEST = 56.0  # steps from zero to a group's largest magnitude, about


def _cache_case(kind, name, lens, hq, hkv, d, dtype="bf16", scales="none", page=16, new=0,
                starts=False):
    case = {"kind": kind, "lens": ",".join(str(int(n)) for n in lens), "new": new, "hq": hq,
            "hkv": hkv, "d": d, "dtype": dtype, "scales": scales, "page": page, "starts": starts}
    if name:
        case["name"] = name
    return case


def _rotate_case(name, tokens, hq, hkv, d, rot, dtype="bf16", interleaved=False, theta=1e6,
                 factor=1.0, inverse=False):
    case = {"kind": "rotate", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "dtype": dtype, "interleaved": interleaved, "theta": theta, "factor": factor,
            "inverse": inverse}
    if name:
        case["name"] = name
    return case


def _tables_case(name, requests, tokens, longest, page, prompts, scarce=False):
    case = {"kind": "tables", "requests": requests, "tokens": tokens, "longest": longest,
            "page": page, "prompts": prompts, "scarce": scarce}
    if name:
        case["name"] = name
    return case


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def listed():
    return [
        # a decode step of 256 running requests, a few of them ending: latency of the call
        _tables_case("tables_decode_256", 256, 256, 15000, 16, 0),
        # a step that admits long prompts beside running requests, pages running short
        _tables_case("tables_prompts", 1000, 400000, 131072, 16, 24, scarce=True),
        # the new tokens of 32 running requests, far positions scaled for a long context
        _rotate_case("rotate_decode_32", 32, 32, 8, 128, 128, factor=4.0),
        # a long prompt, pairs side by side, half of each head rotated
        _rotate_case("rotate_prompt_64k", 65536, 28, 4, 128, 64, dtype="fp16", interleaved=True,
                     theta=1e4),
        # the new tokens of a decode step of 32 running requests: launches, little data
        _cache_case("store", "store_decode_32", [1] * 32, 32, 8, 128),
        # one long-context prompt, with calibrated scales per head
        _cache_case("store", "store_prompt_128k", [131072], 32, 8, 128, scales="head"),
        # a few cached prefixes read back, from the middle on
        _cache_case("gather", "read_back_ragged", [700, 65, 1, 2311], 28, 4, 128, starts=True),
        # every running request's cache read back
        _cache_case("gather", "read_back_32",
                    [(211 + 977 * i * i) % 15000 + 300 for i in range(32)], 32, 8, 128),
        # decode of one short chat: latency of the call
        _cache_case("attend", "decode_one_short", [333], 32, 8, 128, new=1),
        # a decode step of 32 running requests of mixed context lengths
        _cache_case("attend", "decode_32",
                    [(211 + 977 * i * i) % 15000 + 300 for i in range(32)], 32, 8, 128, new=1),
        # one rank's heads of a long request, few KV heads, drafted tokens to be verified
        _cache_case("attend", "verify_4_of_128k", [131000], 8, 2, 64, dtype="fp16",
                    scales="head", page=64, new=4),
        # long new parts over a cached prefix
        _cache_case("attend", "prefix_prefill_long", [6144, 5000, 4321, 4096], 32, 8, 128,
                    new=2048),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "rotate", "store", "gather", "attend", "attend", "attend"])
    if kind == "tables":
        requests = _log_uniform(rng, 1, 1000)
        prompts = rng.choice([0, rng.randint(0, min(requests, 24))])
        tokens = requests + (_log_uniform(rng, 1, 390000) if prompts else rng.randint(0, 100))
        return _tables_case(None, requests, tokens, _log_uniform(rng, 20, 131072),
                            rng.choice([16, 16, 24, 64, 128]), prompts, rng.random() < 0.4)
    hq, hkv = rng.choice([(32, 8), (28, 4), (32, 4), (8, 2), (16, 1), (8, 8)])
    d = rng.choice([64, 128, 128, 256])
    # what the widest heads of a case cost beside 8 of 128
    share = max(1, hkv * d // 1024)
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "rotate":
        rows = (hq + hkv) * d // 4096 + 1
        return _rotate_case(None, _log_uniform(rng, 1, 60000 // rows), hq, hkv, d,
                            rng.choice([d, d, d // 2, d // 4, 8 * rng.randint(1, d // 8)]), dtype,
                            rng.random() < 0.5, rng.choice([1e4, 5e5, 1e6]),
                            rng.choice([1.0, 4.0, 8.0]), rng.random() < 0.2)
    more = {"dtype": dtype, "scales": rng.choice(["none", "none", "tensor", "head"]),
            "page": rng.choice([16, 16, 24, 32, 64, 128])}
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
        return _cache_case(kind, None, lens, hq, hkv, d, new=new, **more)
    if kind == "store":
        lens = [_log_uniform(rng, 1, 100000 // share // n) for _ in range(n)]
    else:
        lens = [_log_uniform(rng, 1, 15000 // share) for _ in range(n)]
        more["starts"] = rng.random() < 0.5
    return _cache_case(kind, None, lens, hq, hkv, d, **more)


# ---------------------------------------------------------------------------
# the 4-bit format
# ---------------------------------------------------------------------------

def _words(step, zero):
    """Group words of steps (fp32, 4 significant bits) and zero points."""
    bits = step.to(torch.float16).view(torch.int16)
    return torch.where(step.isnan(), 0x7F80, bits.to(torch.int32) | (zero.int() + 64)).to(torch.int16)


def _quantise(x, t):
    """Rows x (tokens, heads, d) as (code bytes, group words). t: fp32, (1 | heads), or
    None."""
    n, h, d = x.shape
    x = x.float()
    if t is not None:
        x = x / t.view(1, -1, 1)
    x = x.view(n, h, d // GROUP, GROUP).clamp(-MOST, MOST)
    lo, hi = x.amin(-1), x.amax(-1)  # (NaN where there is one)
    # (tensors, by which torch divides: by numbers it multiplies with their reciprocals)
    want = torch.maximum((hi - lo) / lo.new_full((), 15.0),
                         torch.maximum(hi, -lo) / lo.new_full((), WIDEST))
    # to 4 significant bits, ties to even; below fp16's normal range multiples of 2^-17
    m = want.view(torch.int32)
    m = (m + 0x7FFFF + ((m >> 20) & 1)) >> 20 << 20
    step = torch.where(want < 2.0 ** -14, torch.round(want * 2.0 ** 17) * 2.0 ** -17,
                       m.view(torch.float32))
    step = torch.where(want.isnan(), want, step)
    some = torch.where(step == 0, torch.ones_like(step), step)
    zero = torch.round(lo / some).clamp(-64, 63)
    zero = torch.where((step == 0) | step.isnan(), torch.zeros_like(zero), zero)
    code = (torch.round(x / some.unsqueeze(-1)) - zero.unsqueeze(-1)).clamp(0, 15)
    code = torch.where((step == 0).unsqueeze(-1) | x.isnan() | step.isnan().unsqueeze(-1),
                       torch.zeros_like(code), code).to(torch.uint8)
    # pairs of dims to bytes, byte (m, j) of the pair 2 m, 2 m + 1 of group j
    pair = code.view(n, h, d // GROUP, 16, 2)
    byte = pair[..., 0] | pair[..., 1] << 4
    return byte.transpose(-1, -2).reshape(n, h, d // 2), _words(step, zero)


def _values(byte, word, t):
    """The fp32 values of code bytes (..., heads, d / 2) and group words (..., heads,
    d / 32)."""
    *lead, half = byte.shape
    b = byte.view(*lead, 16, half // 16).transpose(-1, -2)  # (..., d / 32, 16)
    code = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()
    word = word.to(torch.int32)
    step = (word & 0x7F80).to(torch.int16).view(torch.float16).float()
    x = (code + ((word & 127) - 64).float().unsqueeze(-1)) * step.unsqueeze(-1)
    x = x.flatten(-2)
    return x if t is None else x * t.view(-1, 1)


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


def _fixed(case, g):
    """A fixed scale: none, one, or one per KV head, as a calibration finds them."""
    if case["scales"] == "none":
        return None
    n = case["hkv"] if case["scales"] == "head" else 1
    return torch.exp(0.3 * torch.randn(n, generator=g, device="cuda") - 1.0)


def _filled(case, total, t, g):
    """A cache of `total` pages in use: code bytes and group words."""
    hkv, d, page = case["hkv"], case["d"], case["page"]
    x = _rows(total * page, hkv, d, DTYPES[case["dtype"]], g)
    parts = [_quantise(c, t) for c in x.split(max(1, (1 << 27) // (hkv * d)))]
    byte, word = (torch.cat(y) for y in zip(*parts))
    return (byte.view(total, page, hkv, d // 2),
            word.view(total, page, hkv, d // GROUP).transpose(1, 2).contiguous())


def _frequencies(case):
    """Angles per position of the pairs, in 64 bits: theta^(-2 i / rot), and for a long
    context those that turn slowly over the 8,192 trained positions divided by the
    factor, with a ramp between (YaRN, Peng et al. 2023)."""
    rot, theta, factor = case["rot"], case["theta"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = theta ** (-2 * i / rot)
    if factor > 1:
        low, high = (rot * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))
                     for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    return f


def _prepare_rotate(case, g):
    n, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
    qkv = torch.randn(n, hq + 2 * hkv, d, generator=g, device="cuda", dtype=DTYPES[case["dtype"]])
    st = SimpleNamespace(kind="rotate", interleaved=case["interleaved"], inverse=case["inverse"])
    st.q, st.k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    st.q_out, st.k_out = torch.empty_like(st.q), torch.empty_like(st.k)
    st.positions = torch.randint(0, 131072, (n,), generator=g, device="cuda")
    if n > 1024:  # a prompt behind a cached prefix
        st.positions = torch.arange(n, device="cuda") + st.positions[0]
    st.frequencies = _frequencies(case).cuda()
    st.amplitude = 0.1 * math.log(case["factor"]) + 1.0
    return st


def _prepare_tables(case, g):
    R, page, longest, prompts = case["requests"], case["page"], case["longest"], case["prompts"]
    st = SimpleNamespace(kind="tables", page=page)

    def shuffled(values):
        at = torch.randperm(R, generator=g, device="cuda")
        return torch.tensor(values, dtype=torch.int64, device="cuda")[at]

    # lengths of every size, and rows in which nothing runs yet
    lens = [0 if i % 20 == 19 else int(longest ** ((i + 0.5) / R)) for i in range(R)]
    # a token each, and the prompts' shares of the step's tokens
    new = [1 + 2 * (i + 1) * (case["tokens"] - R) // (prompts * (prompts + 1)) if i < prompts else 1
           for i in range(R)]
    used = sum((n + page - 1) // page for n in lens)
    spare = sum((n + page - 1) // page + 1 for n in new) // (2 if case["scarce"] else 1) + 3
    st.width = (max(lens) + max(new)) // page + 2
    lens, new = shuffled(lens), shuffled(new)
    # requests that have ended; in the rows of some others begin
    st.finished = torch.rand(R, generator=g, device="cuda") < 0.05
    new[st.finished & (torch.rand(R, generator=g, device="cuda") < 0.5)] = 0
    st.seq_lens, st.new_lens = lens.to(torch.int32), new.to(torch.int32)
    held = (lens + page - 1) // page
    perm = torch.randperm(used + spare, generator=g, device="cuda").to(torch.int32)
    st.block_table = torch.full((R, st.width), -1, dtype=torch.int32, device="cuda")
    st.block_table[torch.arange(st.width, device="cuda") < held.view(-1, 1)] = perm[:used]
    st.free_pages = torch.full((used + spare,), -1, dtype=torch.int32, device="cuda")
    st.free_pages[:spare] = perm[used:]
    st.num_free = torch.tensor([spare], dtype=torch.int32, device="cuda")
    # as many rows as a captured graph's buffers have
    n = case["tokens"] + 5
    st.cu = torch.empty(R + 1, dtype=torch.int32, device="cuda")
    st.positions, st.slots = (torch.empty(n, dtype=torch.int64, device="cuda") for _ in range(2))
    st.granted = torch.empty(R, dtype=torch.int32, device="cuda")
    st.seq_lens_out, st.num_free_out = torch.empty_like(st.seq_lens), torch.empty_like(st.num_free)
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1234577 * (seed + 1))
    kind = case["kind"]
    if kind == "rotate":
        return _prepare_rotate(case, g)
    if kind == "tables":
        return _prepare_tables(case, g)
    lens, new, page = _lens(case), case["new"], case["page"]
    hq, hkv, d, dtype = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    st = SimpleNamespace(kind=kind, page=page, new=new, starts=None)
    st.k_scale, st.v_scale = _fixed(case, g), _fixed(case, g)
    if kind == "store":
        n = sum(lens)
        qkv = _rows(n, hq + 2 * hkv, d, dtype, g)
        st.key, st.value = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        # the tokens of a sequence of m lie one after the other in shuffled pages, behind
        # m % 7 cached ones and with room left; a serving engine pads the mapping with
        # slots of -1
        total, st.table = _pages([m + 20 for m in lens], page, g)
        st.starts = torch.tensor([m % 7 for m in lens], dtype=torch.int32, device="cuda")
        st.cu = _offsets(lens)
        b = torch.repeat_interleave(torch.arange(len(lens), device="cuda"),
                                    torch.tensor(lens, device="cuda"), output_size=n)
        token = torch.arange(n, device="cuda") - st.cu.long()[b] + st.starts.long()[b]
        st.slots = st.table[b, token // page].long() * page + token % page
        st.slots[torch.arange(n, device="cuda") % 97 == 96] = -1
        st.key_cache = torch.zeros(total, page, hkv, d // 2, dtype=torch.uint8, device="cuda")
        st.key_groups = torch.zeros(total, hkv, page, d // GROUP, dtype=torch.int16, device="cuda")
        st.value_cache, st.value_groups = (torch.zeros_like(x) for x in (st.key_cache,
                                                                         st.key_groups))
        st.key_out, st.value_out = (torch.ones(n, hkv, d, device="cuda", dtype=dtype)
                                    for _ in range(2))
        return st
    total, st.table = _pages(lens, page, g)
    st.key_cache, st.key_groups = _filled(case, total, st.k_scale, g)
    st.value_cache, st.value_groups = _filled(case, total, st.v_scale, g)
    if kind == "attend":
        n = len(lens) * new
        st.query = torch.randn(n, hq, d, generator=g, device="cuda", dtype=dtype)
        st.out = torch.empty_like(st.query)
        st.cu = torch.arange(0, n + 1, new, dtype=torch.int32, device="cuda")
        st.used = torch.tensor(lens, dtype=torch.int32, device="cuda")
        st.scale = 1 / math.sqrt(d)
        return st
    first = [n // 3 if case["starts"] else 0 for n in lens]
    if case["starts"]:
        st.starts = torch.tensor(first, dtype=torch.int32, device="cuda")
    st.cu = _offsets([n - m for n, m in zip(lens, first)])
    # as many rows as a server's buffer has; those behind the last sequence stay
    n = sum(lens) - sum(first) + 3
    st.key_out, st.value_out = (torch.ones(n, hkv, d, device="cuda", dtype=dtype)
                                for _ in range(2))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    if st.kind == "tables":
        _own_tables(st) if own else _plain_tables(st)
        return {"seq_lens": st.seq_lens_out, "num_free": st.num_free_out, "cu_seqlens": st.cu,
                "positions": st.positions, "slots": st.slots, "granted": st.granted,
                "block_table": st.block_table, "free_pages": st.free_pages}
    if st.kind == "rotate":
        _own_rotate(st) if own else _plain_rotate(st)
        return {"q": st.q_out, "k": st.k_out}
    if st.kind == "attend":
        _own_attend(st) if own else _plain_attend(st)
        return st.out
    if st.kind == "store":
        _own_store(st) if own else _plain_store(st)
    _own_gather(st) if own else _plain_gather(st)
    return {"key": st.key_out, "value": st.value_out}


def _own_tables(st):
    from flashprefill_amd.step_tables import build_step_tables

    build_step_tables(st.seq_lens, st.new_lens, st.block_table, st.free_pages, st.num_free,
                      st.page, st.cu, st.positions, st.slots, st.granted, finished=st.finished,
                      seq_lens_out=st.seq_lens_out, num_free_out=st.num_free_out)


def _own_rotate(st):
    from flashprefill_amd.rotary import apply_rotary

    apply_rotary(st.q, st.k, st.positions, st.frequencies, interleaved=st.interleaved,
                 amplitude=st.amplitude, inverse=st.inverse, q_out=st.q_out, k_out=st.k_out)


def _own_store(st):
    from flashprefill_amd.int4_cache import reshape_and_cache_int4

    reshape_and_cache_int4(st.key, st.value, st.key_cache, st.value_cache, st.key_groups,
                           st.value_groups, st.slots, k_scale=st.k_scale, v_scale=st.v_scale)


def _own_gather(st):
    from flashprefill_amd.int4_cache import gather_cache_int4

    gather_cache_int4(st.key_cache, st.value_cache, st.key_groups, st.value_groups, st.key_out,
                      st.value_out, st.cu, st.table, starts=st.starts, k_scale=st.k_scale,
                      v_scale=st.v_scale)


def _own_attend(st):
    from flashprefill_amd.int4_cache import paged_decode_attention_int4

    paged_decode_attention_int4(st.query, st.key_cache, st.value_cache, st.key_groups,
                                st.value_groups, st.out, st.cu, st.used, st.table, st.scale,
                                k_scale=st.k_scale, v_scale=st.v_scale)


def _plain_tables(st):
    page, (R, W), P, N = st.page, st.block_table.shape, st.free_pages.numel(), st.slots.numel()
    lens, new, free = st.seq_lens.long(), st.new_lens.long(), st.num_free.long()
    column = torch.arange(W, device=lens.device)
    # the finished requests' pages go behind the free ones, in the order of the rows
    held = (lens + page - 1) // page
    back = torch.where(st.finished, held, 0)
    behind = back.cumsum(0)
    ends = st.finished & ((back == 0) | (free + behind <= P))
    back = torch.where(ends, back, 0)
    at = free + (behind - back).view(-1, 1) + column
    moved = column < back.view(-1, 1)
    st.free_pages[at[moved]] = st.block_table[moved]
    free = free + back.sum()
    lens = torch.where(ends, 0, lens)
    # the new tokens' pages come from their end, in the order of the rows
    first = new.cumsum(0) - new
    fits = (st.finished == ends) & (first + new <= N) & ((lens + new + page - 1) // page <= W)
    held = (lens + page - 1) // page
    need = torch.where(fits, (lens + new + page - 1) // page - held, 0)
    taken = need.cumsum(0)
    granted = fits & ((need == 0) | (taken <= free))
    need = torch.where(granted, need, 0)
    at = free - 1 - (taken - need).view(-1, 1) - (column - held.view(-1, 1))
    moved = (column >= held.view(-1, 1)) & (column < (held + need).view(-1, 1))
    st.block_table[moved] = st.free_pages[at[moved]]
    st.num_free_out.copy_(free - need.sum())
    st.seq_lens_out.copy_(torch.where(granted, lens + new, lens))
    st.granted.copy_(granted)
    st.cu[:1] = 0
    st.cu[1:] = (first + new).clamp(max=N)
    # every token's request, position and slot
    row = torch.arange(N, device=lens.device)
    r = torch.bucketize(row, st.cu.long(), right=True) - 1
    inside = r < R
    r = r.clamp(max=R - 1)
    position = torch.where(inside, lens[r] + row - first[r], 0)
    slot = st.block_table[r, (position // page).clamp(max=W - 1)].long() * page + position % page
    st.positions.copy_(position)
    st.slots.copy_(torch.where(inside & granted[r], slot, -1))


def _plain_rotate(st):
    angle = st.positions.double().view(-1, 1) * st.frequencies
    cos, sin = ((f(angle) * st.amplitude).float().unsqueeze(1) for f in (torch.cos, torch.sin))
    if st.inverse:
        sin = -sin
    n = st.frequencies.numel()
    for x, y in ((st.q, st.q_out), (st.k, st.k_out)):
        z = x.float()
        part = z[..., :2 * n]
        a, b = (part[..., 0::2], part[..., 1::2]) if st.interleaved else part.split(n, -1)
        u, v = a * cos - b * sin, b * cos + a * sin
        part = torch.stack([u, v], -1).flatten(-2) if st.interleaved else torch.cat([u, v], -1)
        y.copy_(torch.cat([part, z[..., 2 * n:]], -1))


def _plain_store(st):
    rows = (st.slots >= 0).nonzero().view(-1)
    slots = st.slots[rows]
    page, at = slots // st.page, slots % st.page
    for x, cache, groups, t in ((st.key, st.key_cache, st.key_groups, st.k_scale),
                                (st.value, st.value_cache, st.value_groups, st.v_scale)):
        cache[page, at], groups[page, :, at] = _quantise(x[rows], t)


def _plain_gather(st):
    cu = st.cu.long()
    n = torch.arange(st.key_out.shape[0], device=cu.device)
    b = torch.bucketize(n, cu, right=True) - 1
    rows = (b < cu.numel() - 1).nonzero().view(-1)
    b = b[rows]
    token = rows - cu[b] + (st.starts.long()[b] if st.starts is not None else 0)
    page, at = st.table[b, token // st.page].long(), token % st.page
    for x, cache, groups, t in ((st.key_out, st.key_cache, st.key_groups, st.k_scale),
                                (st.value_out, st.value_cache, st.value_groups, st.v_scale)):
        x[rows] = _values(cache[page, at], groups[page, :, at], t).to(x.dtype)


def _plain_attend(st):
    B, new = st.used.numel(), st.new
    T, hq, d = st.query.shape
    hkv = st.key_cache.shape[2]
    pages = st.table.long()
    # (B, heads, keys, d)
    k, v = (_values(cache[pages], groups[pages].transpose(2, 3), t).flatten(1, 2).transpose(1, 2)
            for cache, groups, t in ((st.key_cache, st.key_groups, st.k_scale),
                                     (st.value_cache, st.value_groups, st.v_scale)))
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


# ---------------------------------------------------------------------------
# work and 64-bit results
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "tables":
        # lengths, flags, offsets and grants of the requests; a slot and a position for
        # every token, and for about half as many tokens as a page has a page's number
        # read and written
        R, n = case["requests"], case["tokens"] + 5
        return {"bytes": 21 * R + 16 * n + 8 * (n // case["page"]), "flops": 4 * n}
    if kind == "rotate":
        elements = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": 4 * elements * case["d"] + 8 * case["tokens"] + 4 * case["rot"],
                "flops": 3 * elements * case["rot"]}
    lens, new, d, hq, hkv = _lens(case), case["new"], case["d"], case["hq"], case["hkv"]
    n = sum(lens)
    token = 2 * hkv * (d // 2 + d // 16)  # a token's K and V in the cache, groups included
    pages = sum((m + case["page"] - 1) // case["page"] for m in lens)
    if kind == "store":  # rows read and written back, the cache written and read
        return {"bytes": n * (8 * hkv * d + 2 * token + 8) + 4 * pages, "flops": 10 * n * hkv * d}
    if kind == "attend":
        T = len(lens) * new
        seen = sum(new * m - new * (new - 1) // 2 for m in lens)
        return {"bytes": n * token + 4 * pages + 4 * T * hq * d + 8 * len(lens),
                "flops": 4 * seen * hq * d}
    if case["starts"]:
        n = sum(m - m // 3 for m in lens)
    return {"bytes": n * (4 * hkv * d + token) + 4 * pages, "flops": 4 * n * hkv * d}


def _exact_values(byte, word, t, h):
    """Cached rows (tokens, heads, d) in 64 bits, dim by dim."""
    d = 2 * byte.shape[-1]
    dim = torch.arange(d, device=byte.device)
    group, inner = dim // GROUP, dim % GROUP
    c = (byte[..., inner // 2 * (d // GROUP) + group] >> (inner % 2 * 4).to(torch.uint8)) & 15
    w = word[..., group].long()
    e, m = w >> 10 & 31, w >> 7 & 7
    step = torch.where(e > 0, (8 + m).double() * torch.exp2((e - 18).double()),
                       m.double() * 2.0 ** -17)
    x = step * (c.long() + (w & 127) - 64).double()
    return x if t is None else x * t.double().expand(h).view(-1, 1)


def _exact_quantised(x, t):
    """What the cache holds of rows x (tokens, heads, d), in 64 bits: the format's rule
    on frexp's mantissas."""
    n, h, d = x.shape
    x = x.double() if t is None else x.double() / t.double().view(1, -1, 1)
    x = torch.clamp(x.view(n, h, -1, GROUP), -MOST, MOST)
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    want = torch.maximum((hi - lo) / 15, torch.maximum(hi.abs(), lo.abs()) / WIDEST)
    one = torch.frexp(want.clamp(min=2.0 ** -14)).exponent - 4  # the last bit kept
    one = torch.exp2(one.double())
    step = torch.round(want / one) * one
    some = torch.where(step > 0, step, 1.0)
    zero = torch.round(lo / some)
    y = torch.clamp(torch.round(x / some) - zero, 0, 15) + zero
    y = (y * step).view(n, h, d)
    return y if t is None else y * t.double().view(1, -1, 1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None
    st = prepare(case, seed)
    if kind == "rotate":
        f = _frequencies(case).tolist()
        sign = -1.0 if case["inverse"] else 1.0
        pos = st.positions.double()
        out = {"q": st.q.double(), "k": st.k.double()}
        for i, w in enumerate(f):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + len(f))
            c = (torch.cos(pos * w) * st.amplitude).view(-1, 1)
            s = (torch.sin(pos * w) * st.amplitude * sign).view(-1, 1)
            for name, x in (("q", st.q), ("k", st.k)):
                u, v = x[..., a].double(), x[..., b].double()
                out[name][..., a], out[name][..., b] = u * c - v * s, u * s + v * c
        return out
    lens, page, hkv = _lens(case), case["page"], case["hkv"]
    if kind == "store":
        out = {}
        skipped = torch.arange(sum(lens), device="cuda") % 97 == 96
        for name, x, t in (("key", st.key, st.k_scale), ("value", st.value, st.v_scale)):
            y = torch.cat([_exact_quantised(r, t) for r in x.split(1 << 15)])
            y[skipped] = 0.0
            out[name] = y
        return out

    def tokens_of(b, cache, groups, t, lo, hi):
        """Tokens lo .. hi - 1 of sequence b: (tokens, heads, d)."""
        at = torch.arange(lo, hi, device="cuda")
        p, o = st.table[b][at // page].long(), at % page
        return _exact_values(cache[p, o], groups[p, :, o], t, hkv)

    if kind == "gather":
        key, value = (torch.ones(x.shape, dtype=torch.float64, device="cuda")
                      for x in (st.key_out, st.value_out))
        cu = st.cu.tolist()
        for b in range(len(lens)):
            lo = int(st.starts[b]) if st.starts is not None else 0
            hi = lo + cu[b + 1] - cu[b]
            key[cu[b]:cu[b + 1]] = tokens_of(b, st.key_cache, st.key_groups, st.k_scale, lo, hi)
            value[cu[b]:cu[b + 1]] = tokens_of(b, st.value_cache, st.value_groups, st.v_scale, lo,
                                               hi)
        return {"key": key, "value": value}

    new, group = case["new"], case["hq"] // hkv
    out = torch.empty(st.query.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        k = tokens_of(b, st.key_cache, st.key_groups, st.k_scale, 0, n)
        v = tokens_of(b, st.value_cache, st.value_groups, st.v_scale, 0, n)
        after = torch.ones(new, n, dtype=torch.bool, device="cuda").triu(n - new + 1)
        for h in range(case["hq"]):
            q = st.query[b * new:(b + 1) * new, h].double()
            s = (q @ k[:, h // group].t().contiguous()) * st.scale
            s[after] = -math.inf
            out[b * new:(b + 1) * new, h] = torch.softmax(s, -1) @ v[:, h // group].contiguous()
    return out

"""Inputs and 64-bit results of the 8-bit KV cache's operators, on the CPU."""

import math

import torch

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4M3: 448.0, E5M2: 57344.0}
NAN_CODE = 0x7f  # a NaN of either format
MODES = ("none", "tensor", "head", "slot")


def quantise(x, fmt, scale):
    """(codes, scale) of rows x (tokens, heads, d): scale None (found per row) or fp32
    values that broadcast against (tokens, heads)."""
    x = x.float()
    if scale is None:
        size = x.abs().masked_fill(~x.isfinite(), 0.0).amax(-1) / TOP[fmt]
        scale = torch.where(size > 0, size, torch.ones_like(size))
    y = (x / scale.expand(x.shape[:2]).unsqueeze(-1)).clamp(-TOP[fmt], TOP[fmt])
    return y.to(fmt), scale


def values(cache, scale):
    """A cache's values in 64 bits: (blocks, slots, heads, d)."""
    x = cache.double()
    if scale is None:
        return x
    if scale.dim() == 3:
        return x * scale.double().transpose(1, 2).unsqueeze(-1)
    return x * scale.double().view(-1, 1)


def scales(mode, total, page, hkv, g):
    """One cache's scales: positive, of different sizes."""
    if mode == "none":
        return None
    shape = {"tensor": (1,), "head": (hkv,), "slot": (total, hkv, page)}[mode]
    return torch.exp(torch.randn(shape, generator=g) - 4.0)


def attention_case(lens, news, hq, hkv, d, page, dtype, fmt, mode, seed=0, index=torch.int32,
                   width=None, spare=3):
    """q, k cache, v cache, cu, used, table, k scale, v scale. Slots past a sequence's
    end hold NaN, in the codes and in the scales of a slot."""
    g = torch.Generator().manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    total = sum(per) + spare
    perm = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(width or 0, max(per), 1)), -1, dtype=index)
    at = 0
    for b, m in enumerate(per):
        table[b, :m] = perm[at:at + m].to(index)
        at += m
    caches, found = [], []
    used = torch.zeros(total, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(per[b]):
            used[table[b, j], :min(page, n - j * page)] = True
    for _ in range(2):
        s = scales(mode, total, page, hkv, g)
        size = 1.0 if s is None else s.double().transpose(1, 2).unsqueeze(-1) if mode == "slot" \
            else s.double().view(-1, 1)
        x = torch.randn(total, page, hkv, d, generator=g, dtype=torch.float64)
        codes = (x / size).clamp(-TOP[fmt], TOP[fmt]).float().to(fmt).view(torch.uint8)
        codes[~used] = NAN_CODE
        if mode == "slot":
            s = s.transpose(1, 2).contiguous()
            s[~used] = math.nan
            s = s.transpose(1, 2).contiguous()
        caches.append(codes.view(fmt))
        found.append(s)
    q = (1.5 * torch.randn(sum(news), hq, d, generator=g)).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=index)
    return [q, *caches, cu, torch.tensor(lens, dtype=index), table, *found]


def attention(q, kc, vc, cu, used, table, ks, vs, scale):
    """(out, sum of P |v|) in 64 bits; rows of a sequence of no cached tokens are 0."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    hq, hkv, page, d = q.shape[1], kc.shape[2], kc.shape[1], q.shape[2]
    kv, vv = values(kc, ks), values(vc, vs)
    for b in range(used.numel()):
        n, q0, q1 = int(used[b]), int(cu[b]), int(cu[b + 1])
        if n == 0 or q0 == q1:
            continue
        rows = table[b, :(n + page - 1) // page].long()
        k = kv[rows].reshape(-1, hkv, d)[:n].repeat_interleave(hq // hkv, 1)
        v = vv[rows].reshape(-1, hkv, d)[:n].repeat_interleave(hq // hkv, 1)
        s = torch.einsum("qhd,khd->hqk", q[q0:q1].double(), k) * scale
        pos = torch.arange(n - (q1 - q0), n).view(1, -1, 1)
        hidden = torch.arange(n).view(1, 1, -1) > pos
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        out[q0:q1] = torch.einsum("hqk,khd->qhd", p, v)
        size[q0:q1] = torch.einsum("hqk,khd->qhd", p, v.abs())
    return out, size


def bound(want, size, dtype):
    """What a row may differ by: the output is rounded once, half a spacing (2^-8 of the
    value in bf16, 2^-11 in fp16, 2^-25 below fp16's normal range). Before that P s_v is
    held to 2^-17 (two bf16 parts), and scores of magnitude below 64 in fp32 are off by
    64 x 2^-24 and the rounding of their d = 256 sums, less than 2^-18 together with the
    sums over the keys: 2^-16 of sum P |v| covers both."""
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    least = 0.0 if dtype == torch.bfloat16 else 2.0 ** -25
    return want.abs() * eps * 1.01 + size * 2.0 ** -16 + least

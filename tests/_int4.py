"""Inputs and 64-bit results of the 4-bit KV cache's operators, on the CPU."""

import math

import torch

MODES = ("none", "tensor", "head")
NAN_WORD = 0x7f80


def held(x, scale):
    """(values, steps) that a 4-bit cache holds of rows x (tokens, heads, d), by the
    format's rule in 64 bits; the steps are of each element. NaN groups are NaN."""
    n, h, d = x.shape
    t = torch.ones(1, dtype=torch.float64) if scale is None else scale.double()
    x = (x.double() / t.view(1, -1, 1)).view(n, h, -1, 32).clamp(-16384.0, 16384.0)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    want = torch.maximum((hi - lo) / 15, torch.maximum(hi, -lo) / 56)
    unit = 2.0 ** (torch.floor(torch.log2(want.clamp(min=2.0 ** -14))) - 3)
    s = torch.round(want / unit) * unit
    some = torch.where(s == 0, torch.ones_like(s), s)
    z = torch.round(lo / some).clamp(-64, 63)
    y = ((torch.round(x / some) - z).clamp(0, 15) + z) * s
    y = torch.where(s == 0, torch.zeros_like(y), y)
    return y.view(n, h, d) * t.view(1, -1, 1), (s * torch.ones_like(x)).view(n, h, d)


def values(codes, words, scale):
    """What codes (..., heads, d / 2) and words (..., heads, d / 32) stand for, in 64 bits."""
    nb = words.shape[-1]
    out = torch.empty(*codes.shape[:-1], 32 * nb, dtype=torch.float64)
    for j in range(nb):
        w = words[..., j].long()
        s = (w & 0x7f80).to(torch.int16).contiguous().view(torch.float16).double()
        for m in range(16):
            b = codes[..., m * nb + j].long()
            for p in range(2):
                out[..., 32 * j + 2 * m + p] = s * ((b >> 4 * p & 15) + (w & 127) - 64).double()
    return out if scale is None else out * scale.double().view(-1, 1)


def scales(mode, hkv, g):
    if mode == "none":
        return None
    return torch.exp(torch.randn(hkv if mode == "head" else 1, generator=g) - 1.0)


def random_cache(total, page, hkv, d, g, size=0.15):
    """Codes and words of pages in use: elements of magnitude about 8 `size`."""
    codes = torch.randint(0, 256, (total, page, hkv, d // 2), generator=g, dtype=torch.uint8)
    shape = (total, hkv, page, d // 32)
    step = size * torch.randint(8, 16, shape, generator=g) / 8 * 2.0 ** torch.randint(
        -2, 1, shape, generator=g)
    bits = step.to(torch.float16).view(torch.int16) & 0x7f80
    zero = torch.randint(-12, -3, shape, generator=g, dtype=torch.int16)
    return codes, bits | (zero + 64)


def attention_case(lens, news, hq, hkv, d, page, dtype, mode, seed=0, index=torch.int32,
                   width=None, spare=3):
    """q, k / v codes, k / v words, cu, used, table, k scale, v scale. Groups of slots past a
    sequence's end are NaN."""
    g = torch.Generator().manual_seed(seed)
    per = [(n + page - 1) // page for n in lens]
    total = sum(per) + spare
    perm = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(width or 0, max(per), 1)), -1, dtype=index)
    used = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for b, m in enumerate(per):
        table[b, :m] = perm[at:at + m].to(index)
        for j in range(m):
            used[perm[at + j], :min(page, lens[b] - j * page)] = True
        at += m
    codes, words, found = [], [], []
    for _ in range(2):
        c, w = random_cache(total, page, hkv, d, g)
        w.transpose(1, 2)[~used] = NAN_WORD
        codes.append(c)
        words.append(w)
        found.append(scales(mode, hkv, g))
    q = (1.5 * torch.randn(sum(news), hq, d, generator=g)).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=index)
    return [q, *codes, *words, cu, torch.tensor(lens, dtype=index), table, *found]


def attention(q, kc, vc, kg, vg, cu, used, table, ks, vs, scale):
    """(out, sum of P |v|, largest sum |q| |k| scale) in 64 bits; rows of a sequence of no
    cached tokens are 0."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    hq, hkv, page, d = q.shape[1], kc.shape[2], kc.shape[1], q.shape[2]
    most = 0.0
    for b in range(used.numel()):
        n, q0, q1 = int(used[b]), int(cu[b]), int(cu[b + 1])
        if n == 0 or q0 == q1:
            continue
        rows = table[b, :(n + page - 1) // page].long()
        k, v = (values(c[rows], w[rows].transpose(1, 2), s).reshape(-1, hkv, d)[:n]
                .repeat_interleave(hq // hkv, 1) for c, w, s in ((kc, kg, ks), (vc, vg, vs)))
        s = torch.einsum("qhd,khd->hqk", q[q0:q1].double(), k) * scale
        most = max(most, float(torch.einsum("qhd,khd->hqk", q[q0:q1].double().abs(), k.abs()
                                            ).nan_to_num().max()) * abs(scale))
        pos = torch.arange(n - (q1 - q0), n).view(1, -1, 1)
        hidden = torch.arange(n).view(1, 1, -1) > pos
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        if v.isnan().any():  # (a hidden key's reaches nothing)
            for i in range(q1 - q0):
                see = n - (q1 - q0) + i + 1
                out[q0 + i] = torch.einsum("hk,khd->hd", p[:, i, :see], v[:see])
                size[q0 + i] = torch.einsum("hk,khd->hd", p[:, i, :see], v[:see].abs())
            continue
        out[q0:q1] = torch.einsum("hqk,khd->qhd", p, v)
        size[q0:q1] = torch.einsum("hqk,khd->qhd", p, v.abs())
    return out, size, most


def bound(want, size, most, dtype):
    """What a row may differ by. The output is rounded once, half a spacing: 2^-8 of the
    value in bf16, 2^-11 in fp16 (2^-25 below fp16's normal range). Scores are fp32 sums of
    exact products: of d <= 256 terms in chains of at most 16 MFMAs, off by less than
    2^-19 `most`, and so is P, relatively. P is held to 2^-11 (fp16), and sums over the keys
    and factors to 2^-17: all of it of sum P |v|."""
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    least = 0.0 if dtype == torch.bfloat16 else 2.0 ** -25
    inner = most * 2.0 ** -19 + 2.0 ** -17 + 2.0 ** -11
    return want.abs() * eps * 1.01 + size * inner + least


def rows(n, heads, d, dtype, seed=0):
    """Rows with what a cache meets: every size, zeros, constants, largest values,
    infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g) * torch.exp(2 * torch.randn(n, 1, 1, generator=g))
    x += 3 * torch.randn(n, heads, 1, generator=g) * (torch.rand(n, heads, 1, generator=g) < 0.2)
    kinds = torch.randint(0, 40, (n, heads), generator=g)
    x[kinds == 0] = 0.0
    x[kinds == 1] = -2.25
    x[kinds == 2] *= 1e-5
    x[kinds == 3] *= 3e-8
    x[kinds == 4] *= 2e4
    x[kinds == 5, 3] = math.inf
    x[kinds == 6, d - 1] = -math.inf
    x[kinds == 7, 32] = math.nan
    x[kinds == 8, 7] *= 60
    x[kinds == 9] = torch.randint(-8, 9, (d,), generator=g).float()  # ties
    return x.to(dtype)

"""Inputs and 64-bit results of rotary positions."""

import torch


def rows(n, heads, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, heads, d, generator=g) * torch.exp(torch.randn(n, 1, 1, generator=g))
    return x.to(dtype)


def positions(n, seed=0, dtype=torch.int64):
    """Far, near and negative ones."""
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 1 << 20, (n,), generator=g)
    p[::3] = torch.arange(n)[::3]
    p[1::7] = -p[1::7]
    return p.to(dtype)


def rotated(x, pos, f, interleaved, amplitude, inverse):
    """Pair by pair in 64 bits."""
    y = x.double().clone()
    n = f.numel()
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, n + i)
        angle = pos.double() * f[i]
        c, s = (amplitude * t.view(-1, 1) for t in (angle.cos(), angle.sin()))
        s = -s if inverse else s
        u, v = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y

"""The 4-bit key/value cache in plain 64-bit arithmetic, value by value from its definition: what a group of 16 values is held as,
where in a unit each of them lies, and attention over what is held."""
from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
SCALES = (torch.arange(227, dtype=torch.int16) << 7).view(torch.float16).double()        # by their byte, up to 10,240


def held(x: torch.Tensor):
    """(values, codes, scale bytes) that float64 rows [.., features] are held as; NaN and 255 where a group is not finite."""
    g = x.double().cpu().unflatten(-1, (-1, 16))
    finite = torch.isfinite(g).all(-1)
    g = torch.where(finite.unsqueeze(-1), g, torch.zeros_like(g))
    wanted = (g.abs().amax(-1) / 6).clamp(max=10240.0)
    away = (SCALES - wanted.unsqueeze(-1)).abs()
    least = away.amin(-1, keepdim=True)
    # the nearest byte; of two equally near ones the even one
    byte = torch.where(away == least, torch.arange(227) + 1000 * (torch.arange(227) % 2), 10 ** 6).amin(-1) % 1000
    scale = SCALES[byte].unsqueeze(-1)
    # above the last level a value is nearest to it; the difference to a huge value is the same for all levels in 64 bits
    away = (LEVELS * scale.unsqueeze(-1) - torch.minimum(g.abs(), 6 * scale).unsqueeze(-1)).abs()
    near = away == away.amin(-1, keepdim=True)
    code = torch.where(near, torch.arange(8) + 100 * (torch.arange(8) % 2), 10 ** 6).amin(-1) % 100
    code = torch.where(scale > 0, code, torch.zeros_like(code))
    values = torch.copysign(LEVELS[code] * scale, g)
    values = torch.where(finite.unsqueeze(-1), values, torch.full_like(values, math.nan))
    code = code + 8 * (g < 0)
    return values.flatten(-2), torch.where(finite.unsqueeze(-1), code, torch.zeros_like(code)).flatten(-2), torch.where(finite, byte, 255)


def code_at(dim: int, r: int, f: int, value: bool) -> int:
    """The byte of a unit that holds the code of feature ``f`` of token ``r`` (in its low half where ``f`` is even)."""
    if not value:
        return r * dim // 2 + f // 2
    lane, pair, odd = f // (dim // 8), r // 2 % 4, r % 2
    return 8 * dim + r // 8 * 4 * dim + (lane * 8 + pair * 2 + odd) * (dim // 16) + f % (dim // 8) // 2


def scale_at(dim: int, r: int, s: int, value: bool) -> int:
    if not value:
        per = dim // 64
        return 16 * dim + (r % 8 * 4 + s // per) * 2 * per + r // 8 * per + s % per
    return 17 * dim + (s * 4 + r // 2 % 4) * 4 + r // 8 * 2 + r % 2


def unit_of(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """The bytes of a unit of float64 rows [16, dim]."""
    dim = k.shape[1]
    unit = torch.zeros(18 * dim, dtype=torch.int64)
    for x, value in ((k, False), (v, True)):
        _, code, byte = held(x)
        for r in range(16):
            for f in range(dim):
                unit[code_at(dim, r, f, value)] |= int(code[r, f]) << 4 * (f % 2)
            for s in range(dim // 16):
                unit[scale_at(dim, r, s, value)] = int(byte[r, s])
    return unit.to(torch.uint8)


def units_of(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """The bytes [.., 18 dim] of float64 rows [.., 16, dim]: :func:`unit_of` for many."""
    dim = k.shape[-1]
    out = torch.zeros((*k.shape[:-2], 18 * dim), dtype=torch.int64)
    r, f, s = torch.arange(16).view(-1, 1), torch.arange(dim), torch.arange(dim // 16)
    for x, value in ((k, False), (v, True)):
        _, code, byte = held(x)
        at = torch.tensor([[code_at(dim, int(i), int(j), value) for j in f] for i in r])
        out.scatter_add_(-1, at.expand(*k.shape[:-2], 16, dim).reshape(*k.shape[:-2], -1), (code << 4 * (f % 2)).flatten(-2))
        at = torch.tensor([[scale_at(dim, int(i), int(j), value) for j in s] for i in r])
        out[..., at] = byte
    return out.to(torch.uint8)


def first_visible(pos: int, window: int) -> int:
    if window > 0:
        return max(0, pos - window + 1)
    return pos - pos % -window if window < 0 else 0


def attend(q, k, v, positions, scale, window=0, seen=None):
    """Float64 [tokens, heads, dim]: q [tokens, heads, dim] over keys and values [length, kv heads, dim]; ``seen``: keys whose page is
    held."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out = torch.zeros_like(q)
    for i, pos in enumerate(positions):
        if pos < 0:
            continue
        at = torch.arange(first_visible(pos, window), min(pos + 1, k.shape[0]))
        if seen is not None:
            at = at[seen[at]]
        if not at.numel():
            continue
        kk, vv = (x[at].repeat_interleave(group, 1) for x in (k, v))
        score = torch.einsum("hd,khd->hk", q[i], kk) * scale
        out[i] = torch.einsum("hk,khd->hd", torch.softmax(score, -1), vv)
    return out

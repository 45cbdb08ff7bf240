"""The paged-cache operators in float64 (numpy), test infrastructure only: slot maps from lengths,
rotary positions, attention of drafted tokens over a paged cache. Written from the formulas in
include/kta_b200.h, request by request and row by row.
"""

from __future__ import annotations

import math

import numpy as np


def cache_slots(ctx, new, tables, free, block: int, rows: int):
    """(tables, slots, positions, offsets, used) of one step, with what does not fit cut off."""
    tables = np.array(tables, dtype=np.int64)
    slots, positions = np.full(rows, -1, dtype=np.int64), np.zeros(rows, dtype=np.int64)
    offsets, taken, row = [0], 0, 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        c, n = int(c), int(n)
        if c < 0 or n < 0 or c + n > tables.shape[1] * block:
            c = n = 0
        for j in range(-(-c // block), -(-(c + n) // block)):
            tables[b, j] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(c, c + n):
            if row < rows:
                block_id = tables[b, p // block]
                slots[row] = block_id * block + p % block if block_id >= 0 else -1
                positions[row] = p
                row += 1
        offsets.append(row)
    return tables, slots, positions, np.array(offsets), min(taken, len(free))


_TURN_BITS = 320


def _radian() -> int:
    """1 / (2 pi) in units of 2^-_TURN_BITS of a turn, pi from Machin's 4 (4 acot 5 - acot 239) in integers."""
    bits = _TURN_BITS + 32

    def acot(n: int) -> int:
        power = total = (1 << bits) // n
        k = 1
        while power:
            power //= -n * n
            k += 2
            total += power // k
        return total

    return (1 << (bits + _TURN_BITS)) // (8 * (4 * acot(5) - acot(239)))


_RADIAN = _radian()


def rope(x, positions, freqs, interleaved: bool, inverse: bool = False, scale: float = 1.0):
    """x [N, H, D] float64; the frequencies become turns and whole turns are taken off in integers of
    320 bits, so that positions of any size keep their angle."""
    x = np.asarray(x, dtype=np.float64)
    y = x.copy()
    half = len(freqs)
    for i, f in enumerate(freqs):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        num, den = float(f).as_integer_ratio()
        t = np.array([int(n) * num * _RADIAN // den % (1 << _TURN_BITS) / (1 << _TURN_BITS)
                      for n in positions]) * 2 * math.pi
        t = (-t if inverse else t)[:, None]
        y[..., a] = scale * (x[..., a] * np.cos(t) - x[..., b] * np.sin(t))
        y[..., b] = scale * (x[..., b] * np.cos(t) + x[..., a] * np.sin(t))
    return y


def tree_bits(parents) -> list[int]:
    """Per drafted token the bits of itself and of those that it continues (parent -1: the
    context), as signed 64-bit integers."""
    bits: list[int] = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def seen(ctx: int, new: int, bits) -> np.ndarray:
    """[new, ctx + new]: which keys each drafted token sees (bits None: a chain)."""
    s = np.zeros((new, ctx + new), dtype=bool)
    s[:, :ctx] = True
    for i in range(new):
        for j in range(new):
            s[i, ctx + j] = j <= i if bits is None else bool(int(bits[i]) >> j & 1)
    return s


def attention(q, k, v, sight, scale: float):
    """Rows q [R, D] over keys k, v [L, D], row i over the keys of sight[i]. Returns O, LSE, and
    per row what error bounds need: sum p |v| [R, D], sum |v| / sum e [R, D], max |s| [R] and
    max sum |q| |k| [R]. Keys that a row does not see have no part in it, whatever they hold."""
    R, D = q.shape
    o, lse = np.zeros((R, D)), np.full(R, -np.inf)
    pv, tiny, smax, dot = np.zeros((R, D)), np.zeros((R, D)), np.zeros(R), np.zeros(R)
    for i in range(R):
        on = sight[i]
        if not on.any():
            continue
        ki, vi = k[on], v[on]
        s = scale * (ki @ q[i])
        top = s.max()
        e = np.exp(s - top)
        total = e.sum()
        o[i] = (e / total) @ vi
        lse[i] = top + math.log(total) if np.isfinite(total) else np.nan
        pv[i], tiny[i] = (e / total) @ np.abs(vi), np.abs(vi).sum(0) / total
        smax[i], dot[i] = np.abs(s).max(), scale * (np.abs(ki) @ np.abs(q[i])).max()
    return o, lse, pv, tiny, smax, dot


def attention_bounds(sight, eps: float, sub: float, o, lse, pv, tiny, smax, dot):
    """How far O [R, D] and LSE [R] of the 16-bit kernel may be from attention()'s results (the rest
    of the arguments). eps: half a step of the storage type; sub: half a subnormal step of the
    weights' type. In fp32 a score of D products is off by D 2^-24 sum |q||k| scale, the exponent by
    roundings of |s|, 2^x by 2 ulp: d32 relative, on a weight and again on the sum."""
    D, keys = o.shape[1], sight.sum(1)
    d32 = D * 2.0 ** -24 * dot + 6 * smax * 2.0 ** -24 + 2.0 ** -22
    f = pv * (eps + 2 * d32 + keys * 2.0 ** -24)[:, None] + sub * tiny
    z = np.where(keys == 0, 0, lse)
    return f + eps * (np.abs(o) + f) + 2.0 ** -25, d32 + (keys + 2 * np.abs(z)) * 2.0 ** -24

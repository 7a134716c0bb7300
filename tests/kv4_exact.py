"""Rows of the paged cache held in 4 bits from their definition in exact fractions, and rows at its borders.  (Doubles lose what a value far below another one leaves of their difference.)"""
from fractions import Fraction

import torch

BF = torch.bfloat16
TOP = Fraction(255, 128) * 2 ** 127   # bf16's largest number
NAN, INF = float("nan"), float("inf")


def to_bf16(x: Fraction) -> Fraction:
    """x to bf16, once: to nearest, ties to even; None where that is infinite."""
    if x == 0:
        return x
    a, e = abs(x), -126
    while a >= Fraction(2) ** (e + 1):
        e += 1
    unit = Fraction(2) ** (e - 7)
    y = round(a / unit) * unit   # (of a fraction: ties to even)
    return None if y > TOP else y if x > 0 else -y


def held(row):
    """Codes, scale and minimum of a row of finite bf16 values (a list of floats), and the values that stand for it, rounded once; None for a row that is NaN."""
    x = [Fraction(v) for v in row]
    low, spread = min(x), max(x) - min(x)
    if spread >= Fraction(2) ** 128 - Fraction(2) ** 103:   # (passes fp32)
        return None
    scale = to_bf16(spread / 15)
    if scale < Fraction(2) ** -126:
        scale = Fraction(0)
    codes = [int((v - low) / scale + Fraction(1, 2)) if scale else 0 for v in x]
    values = [to_bf16(scale * c + low) for c in codes]
    return codes, float(scale), float(low), [INF if v is None else float(v) for v in values]


def cache_of(x, slots, pages, S, byte=0):
    """Rows x [M, KV, hd] in the slots of a new cache, and their values [M, KV, hd]."""
    M, KV, hd = x.shape
    cache = torch.full((pages, KV, S * (hd // 2 + 4)), byte, dtype=torch.uint8)
    codes_of, pairs_of = cache[:, :, :S * (hd // 2)].unflatten(2, (S, hd // 2)), cache[:, :, S * (hd // 2):].unflatten(2, (S, 4))
    values = torch.empty(M, KV, hd, dtype=BF)
    for m in range(M):
        page, off = divmod(int(slots[m]), S)
        for h in range(KV):
            row = held(x[m, h].double().tolist())
            codes, scale, low, v = row or ([0] * hd, NAN, NAN, [NAN] * hd)
            values[m, h] = torch.tensor(v, dtype=torch.float64).to(BF)   # (exact)
            c = torch.tensor(codes, dtype=torch.uint8)
            codes_of[page, h, off] = c[::2] + 16 * c[1::2]
            pairs_of[page, h, off] = torch.tensor([scale, low], dtype=torch.float64).to(BF).view(torch.uint8)
    return cache, values


def _rows(rows, hd):
    return torch.tensor([r + [r[i % len(r)] for i in range(hd - len(r))] for r in rows], dtype=torch.float64).to(BF).view(-1, 1, hd)


def far_below_borders(hd):
    """Rows whose values lie at a border but for something far below it: a tiny minimum, or a tiny value above a minimum that lies at a border itself."""
    rows = []
    for k in (-80, -30, -25, -17, -9):
        for sign in (1, -1):
            t = sign * 2.0 ** k
            rows.append([t if sign > 0 or k < -9 else 0.0, 15.0] + [i + 0.5 for i in range(15)] + [1.0, 7.0, 14.0])
            for c in (0, 2, 7, 14):   # the minimum has `c` and a half scales below zero
                low = -(c + 0.5)
                rows.append([low, low + 15.0, t, -t, 2 * t, 0.0] + [low + i for i in range(1, 15)])
    return _rows(rows, hd)


def every_scale(hd):
    """Of every mantissa of a scale a row whose difference of largest and smallest is fifteen of it, with the values of bf16 next to every border, below, at and above."""
    rows = []
    for n in range(128, 256):
        top = (15 * n // 16 + 1) * 16   # (eight bits)
        low = top - 15 * n
        row = [float(low), float(top)]
        for c in range(15):
            v = to_bf16(low + (c + Fraction(1, 2)) * n)
            for step in (-1, 0, 1):
                near = torch.tensor([float(v)]).to(BF).view(torch.int16) + step
                row.append(float(near.view(BF)))
        rows.append([min(max(v, float(low)), float(top)) / 128 for v in row[:hd]] if hd < len(row) else [v / 128 for v in row])
    return _rows(rows, hd)


def rounded_twice(hd):
    """Rows whose values are a border of bf16 but for a minimum far below it."""
    rows = []
    for k in (-20, -24, -30, -70, -120):
        for sign in (1, -1):
            t = sign * 2.0 ** k
            for n in (129, 131, 135, 203, 255):
                s = n / 128
                top = float(to_bf16(Fraction(15 * n, 128)))
                rows.append([t, top] + [float(to_bf16(Fraction(c * n, 128))) for c in range(1, 15)] + [t * 2, s])
    return _rows(rows, hd)

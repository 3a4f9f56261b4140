"""A paged cache in 4 bits and what is done with it, in 64 bits on the host, one row at a time, from the definitions.

A group of 32 numbers has a scale, a number with 5 bits of exponent and 3 of mantissa, the nearest one to its largest magnitude / 7, and each number is the nearest multiple
of it from -7 to 7, stored plus 8; halves go to the even one.  Keys lie in words of 8 numbers, values in half words of 4 (``place``).
"""
import math
from fractions import Fraction

import numpy as np
import torch

#: Every scale there is, ascending: byte b stands for SCALES[b].
SCALES = [Fraction(m, 1 << 17) for m in range(8)] + [Fraction(8 + m) * Fraction(2) ** (e - 18) for e in range(1, 31) for m in range(8)]


def _nearest(x, steps):
    """The index of the number nearest to x among ascending ones, the even index of two."""
    best = min(range(len(steps)), key=lambda i: (abs(steps[i] - x), i % 2))
    return best


def group_bits(x):
    """(codes, byte of the scale) of 32 numbers."""
    if not all(math.isfinite(v) for v in x):
        return [8] * len(x), 255
    top = max(abs(Fraction(v)) for v in x) / 7
    byte = 247 if top >= SCALES[-1] else _nearest(top, SCALES)
    scale = SCALES[byte]
    if scale == 0:
        return [8] * len(x), byte
    codes = []
    for v in x:
        r = Fraction(v) / scale
        n = r.numerator // r.denominator
        left = r - n
        n += 1 if left > Fraction(1, 2) or (left == Fraction(1, 2) and n % 2) else 0
        codes.append(max(-7, min(7, n)) + 8)
    return codes, byte


def scale_of(byte):
    return float(SCALES[byte]) if byte < len(SCALES) else (math.inf if byte == 248 else math.nan)


def place(d, values):
    """Which number of a head lies at each place of a stored row."""
    run, groups = (4 if values else 8), d // 32
    return [32 * ((p // run) % groups) + run * ((p // run) // groups) + p % run for p in range(d)]


def row_bits(x, values):
    """(bytes of codes, bytes of scales) of one head's row."""
    d = len(x)
    codes, scales = [0] * d, []
    for j in range(d // 32):
        c, b = group_bits(x[32 * j:32 * j + 32])
        codes[32 * j:32 * j + 32] = c
        scales.append(b)
    stored = [codes[n] for n in place(d, values)]
    return [stored[i] | stored[i + 1] << 4 for i in range(0, d, 2)], scales


def page_parts(cache, page, d):
    """Views of a pool [..., bytes]: codes [..., page, d / 2], scales [..., page, d / 32]."""
    n = page * d // 2
    return cache[..., :n].reshape(*cache.shape[:-1], page, d // 2), cache[..., n:].reshape(*cache.shape[:-1], page, d // 32)


_SCALE_TABLE = np.array([scale_of(b) for b in range(256)])


def numbers(cache, page, d, values):
    """The numbers [..., page, d] of a pool, in 64 bits."""
    codes, scales = page_parts(cache.cpu().numpy(), page, d)
    stored = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], d).astype(np.float64) - 8
    out = np.empty_like(stored)
    with np.errstate(invalid="ignore"):
        order = np.array(place(d, values))
        out[..., order] = stored * _SCALE_TABLE[scales][..., order // 32]
    return torch.from_numpy(out)


def random_pool(pages, n_kv, page, d, generator, low=100, high=130, finite=True):
    """A pool of random codes from 1 to 15 and scales of these bytes."""
    g = generator
    codes = torch.randint(1, 16, (pages, n_kv, page, d // 2), generator=g) | torch.randint(1, 16, (pages, n_kv, page, d // 2), generator=g) << 4
    scales = torch.randint(low, high, (pages, n_kv, page, d // 32), generator=g)
    return torch.cat([codes.flatten(2), scales.flatten(2)], dim=2).to(torch.uint8)


def attention(q, k, v, count, held, group, scale, window=None, sink=None, softcap=None):
    """One request.  q [n, heads, d]; k, v [heads / group, keys, d], or v None; the n tokens are the last of ``held`` keys.  Returns out [n, heads, d], lse [n, heads],
    the weights [n, heads, keys] and each row's sum of |weight * value| [n, heads, d], in 64 bits."""
    n, heads, d = q.shape
    dv = d if v is None else v.shape[2]
    out, mass = torch.zeros(n, heads, dv, dtype=torch.float64), torch.zeros(n, heads, dv, dtype=torch.float64)
    lse, p = torch.full((n, heads), -math.inf, dtype=torch.float64), torch.zeros(n, heads, held, dtype=torch.float64)
    for i in range(n):
        at = held - count + i
        lo = max(0, at - window + 1) if window else 0
        if at < lo and sink is None:
            continue
        for h in range(heads):
            x = k[h // group, lo:at + 1].double() @ q[i, h].double() * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            full = torch.cat([x, sink[h].double().reshape(1)]) if sink is not None else x
            if full.numel() == 0:
                continue
            lse[i, h] = torch.logsumexp(full, 0)
            w = torch.softmax(full, 0)[:x.numel()]
            p[i, h, lo:at + 1] = w
            if v is not None and w.numel():
                out[i, h] = (w[:, None] * v[h // group, lo:at + 1].double()).sum(0)
                mass[i, h] = (w[:, None] * v[h // group, lo:at + 1].double().abs()).sum(0)
    return out, lse, p, mass


def kept_places(weights, held, keep, first, last):
    """The places that stay of ``held`` keys with these sums, ascending."""
    if held <= keep:
        return list(range(held))
    first = min(first, keep)
    last = min(last, keep - first)
    always = list(range(first)) + list(range(held - last, held))
    above = lambda w: (2, 0.0) if math.isnan(w) else (1, float(w))       # noqa: E731   a NaN is above infinity
    rest = sorted(range(first, held - last), key=lambda j: above(weights[j]), reverse=True)      # stable: reverse keeps the order of equals
    return sorted(always + rest[:keep - first - last])

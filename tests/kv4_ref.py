"""The 4-bit KV cache restated in numpy, in 64 bits and element by element: block quantisation, the place of every code
and scale in a tile, rotary positions, and attention with a window and sinks."""
import numpy as np

TILE = 16


def tile_bytes(hd):
    return 18 * hd


def cache_bytes(kv_heads, hd, positions):
    return (positions + TILE - 1) // TILE * kv_heads * tile_bytes(hd)


def rotate(x, table, pos, rope, neox):
    """x [T][heads][hd] float; table [positions][rope / 2][2]; in float64."""
    y = np.array(x, dtype=np.float64)
    for t, p in enumerate(pos):
        for i in range(rope // 2):
            a, b = (i, i + rope // 2) if neox else (2 * i, 2 * i + 1)
            c, s = np.float64(table[p, i, 0]), np.float64(table[p, i, 1])
            x0, x1 = y[t, :, a].copy(), y[t, :, b].copy()
            y[t, :, a], y[t, :, b] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def quantise(x):
    """(codes [.., hd] int, scales [.., hd / 32] float16) of x in float64."""
    b = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32)
    hi, lo = b.max(-1), b.min(-1)
    with np.errstate(invalid="ignore", divide="ignore"):
        d = np.clip((np.where(hi >= -lo, hi, lo) / -8).astype(np.float32), -65504, 65504).astype(np.float16)
        d = np.where(np.isfinite(b).all(-1), d, np.float16(np.nan))
        inv = np.where(d == 0, 0.0, 1 / d.astype(np.float64))
        c = np.floor(b * inv[..., None] + 8.5)
    c = np.where(np.isnan(c), 0, np.clip(c, 0, 15)).astype(np.int64)
    return c.reshape(x.shape), d


def _word(hd, half, lane, b):
    w = min(4, hd // 32)
    return (b // 4) * 256 + (half * 32 + lane) * w + b % 4


def _places(hd, p, is_v):
    """(byte offset, shift) of every dim's code, and the byte offset of every block's scale, in position p's tile."""
    r = p % TILE
    code, shift = np.empty(hd, np.int64), np.empty(hd, np.int64)
    for d in range(hd):
        b = d // 32
        if is_v:
            nib = d % 4 + 4 * (r % 2)
            word = _word(hd, r // 8, (d % 32) // 4 * 4 + (r % 8) // 2, b)
        else:
            nib = d % 8
            word = _word(hd, r // 8, (r % 8) * 4 + (d % 32) // 8, b)
        code[d] = (8 * hd if is_v else 0) + 4 * word + nib // 2
        shift[d] = 4 * (nib % 2)
    nb = hd // 32
    return code, shift, (17 if is_v else 16) * hd + 2 * (r * nb + np.arange(nb))


def write(cache, kv_heads, hd, p, codes, scales, is_v):
    """Puts position p's codes [kv_heads][hd] and scales into a cache (uint8 array)."""
    code, shift, sc = _places(hd, p, is_v)
    for h in range(kv_heads):
        t = cache[((p // TILE) * kv_heads + h) * tile_bytes(hd):][:tile_bytes(hd)]
        for d in range(hd):
            t[code[d]] = (t[code[d]] & ~(15 << shift[d]) & 255) | (int(codes[h, d]) << shift[d])
        raw = scales[h].astype(np.float16).view(np.uint8).reshape(-1, 2)
        t[sc], t[sc + 1] = raw[:, 0], raw[:, 1]


def read(cache, kv_heads, hd, n, is_v):
    """float64 values [n][kv_heads][hd] of a cache's first n positions."""
    out = np.empty((n, kv_heads, hd))
    nb = hd // 32
    for r in range(TILE):
        p = np.arange(r, n, TILE)
        if not p.size:
            continue
        code, shift, sc = _places(hd, r, is_v)
        for h in range(kv_heads):
            t = cache[: cache.size // (kv_heads * tile_bytes(hd)) * kv_heads * tile_bytes(hd)].reshape(-1, kv_heads, tile_bytes(hd))[p // TILE, h]
            c = ((t[:, code] >> shift) & 15).astype(np.float64) - 8
            d = (t[:, sc].astype(np.uint16) | (t[:, sc + 1].astype(np.uint16) << 8)).view(np.float16).astype(np.float64)
            with np.errstate(invalid="ignore"):
                out[p, h] = (c.reshape(-1, nb, 32) * d[:, :, None]).reshape(-1, hd)
    return out


def visible(p, window, sinks):
    j = np.arange(max(0, p + 1))
    return j[(j > p - window) | (j < sinks)] if window else j


def attention(q, k, v, p, scale, window=0, sinks=0):
    """One row: q [heads][hd], k and v [n][kv_heads][hd] float64, position p. Returns (out [heads][hd], bound [heads]): the
    result and how far 32-bit arithmetic with 22-bit queries may be from it.

    The bound. A score's error: the query's remainder after two fp16 roundings is at most 2^-22 of the row's largest value
    (2^-23 of it for the value, twice for the scaled product's own rounding), so a score is off by at most
    2^-22 * qmax * sum |k|; its sums run over hd products in fp32, at most 16 + hd / 32 roundings of partial sums below
    qmax * sum |k|, 2^-23 each (an MMA may truncate). Together below 2^-18 of qmax * sum |k| * scale =: s. A weight is off by
    a factor exp(2 delta), delta = 2^-18 s + 2^-21 (the exponential's own error); the output by 2 delta times the largest
    |v|, and by as many roundings again as it has terms in sequence: below 2^-17 of the largest |v|."""
    heads, hd = q.shape
    g = heads // k.shape[1]
    j = visible(p, window, sinks)
    out, bound = np.zeros((heads, hd)), np.zeros(heads)
    if not j.size:
        return out, bound
    for h in range(heads):
        kk, vv = k[j, h // g], v[j, h // g]
        s = kk @ np.asarray(q[h], np.float64) * scale
        w = np.exp(s - s.max())
        out[h] = w @ vv / w.sum()
        size = np.abs(q[h]).max() * np.abs(kk).sum(1).max() * abs(scale)
        bound[h] = (4 * (2.0 ** -18 * size + 2.0 ** -21) + 2.0 ** -17) * np.abs(vv).max()
    return out, bound

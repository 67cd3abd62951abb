"""Float64 restatement of the 8-bit paged cache: its format, append, read and attention.

Test infrastructure only. A cache is bytes ``[blocks, block_size, heads, dim]`` with exponents
``scales [blocks, heads, 2]`` (K, V); a byte stands for ``e4m3 * 2**(e - 127)``.
"""

import numpy as np


def _table():
    """Value of each e4m3 byte: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7F is NaN."""
    values = np.empty(256)
    for byte in range(256):
        exponent, mantissa = byte >> 3 & 15, byte & 7
        value = mantissa * 2.0 ** -9 if exponent == 0 else (8 + mantissa) * 2.0 ** (exponent - 10)
        if byte & 127 == 127:
            value = np.nan
        values[byte] = -value if byte & 128 else value
    return values


E4M3 = _table()
LEAST = 27


def encode(x):
    """Nearest e4m3 byte, ties to even; NaN, infinities and what rounds past 448 are NaN."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    fine = a < 465
    a = np.where(fine, a, 0.0)
    _, exponent = np.frexp(a)  # a < 2**exponent
    step = np.exp2(np.maximum(exponent - 1, -6) - 3.0)
    a = np.round(a / step) * step
    byte = np.searchsorted(E4M3[:127], a)
    byte = np.where(fine & (a <= 448), byte, 127)
    return (byte + 128 * np.signbit(x)).astype(np.uint8)


def exponent(amax):
    """Least e >= LEAST with amax <= 448 * 2**(e - 127)."""
    e = LEAST
    while amax > 448 * 2.0 ** (e - 127):
        e += 1
    return e


def append(cache, scales, part, rows, tables, lengths, cu=None):
    """In place on ``cache`` and ``scales[..., part]``; ``rows`` float64 [rows, heads, dim]."""
    blocks, bs, heads, _ = cache.shape
    for s, n in enumerate(lengths):
        first_row, q = (s, 1) if cu is None else (cu[s], cu[s + 1] - cu[s])
        if n <= 0 or q <= 0:
            continue
        positions = [p for p in range(max(0, n - q), min(n, tables.shape[1] * bs))]
        for page in sorted({p // bs for p in positions}):
            block = tables[s, page]
            if not 0 <= block < blocks:
                continue
            mine = [p for p in positions if p // bs == page]
            old = mine[0] - page * bs if mine[0] == max(0, n - q) else 0
            x = rows[[first_row + p - (n - q) for p in mine]]
            for h in range(heads):
                finite = np.abs(x[:, h][np.isfinite(x[:, h])])
                e = exponent(finite.max() if finite.size else 0.0)
                if old:
                    was = int(scales[block, h, part])
                    e = max(e, was)
                    kept = E4M3[cache[block, :old, h]] * 2.0 ** (was - e)
                    cache[block, :old, h] = encode(kept) if was != e else cache[block, :old, h]
                cache[block, old : old + len(mine), h] = encode(x[:, h] * 2.0 ** (127 - e))
                scales[block, h, part] = e


def values(cache, scales, part, pages):
    """Float64 values of ``pages``: [pages, block_size, heads, dim]."""
    return E4M3[cache[pages]] * 2.0 ** (scales[pages][:, None, :, part, None].astype(np.float64) - 127)


def attend(q, k, v, first, window=0):
    """Causal attention of q [n, Hq, D] at positions first.. over k, v [m, Hkv, D] (positions 0..).

    Returns the output, the weighted mean of |v| (what an error of the weights is relative to),
    and the largest sum_i |q_i k_i| / sqrt(D) (what an error of a score is relative to)."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = np.zeros((n, heads, dim))
    mean, reach = np.zeros((n, heads, dim)), np.zeros((n, heads, 1))
    for i in range(n):
        end = min(first + i + 1, k.shape[0])
        start = max(0, end - window) if window else 0
        if end <= 0:
            continue
        for h in range(heads):
            kk, vv = k[start:end, h // group], v[start:end, h // group]
            scores = kk @ q[i, h] / np.sqrt(dim)
            p = np.exp(scores - scores.max())
            p /= p.sum()
            out[i, h], mean[i, h] = p @ vv, p @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(dim)
    return out, mean, reach

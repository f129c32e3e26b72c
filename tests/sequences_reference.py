"""Plain 64-bit definitions of the operators over several sequences, in numpy, and batches to try them on."""
import math

import numpy as np


def rotate(x, positions, frequencies, magnitude, pairs):
    """x [heads, rows, d] turned by positions [rows], frequencies in radians a position."""
    out = x.astype(np.float64).copy()
    n = len(frequencies)
    for i, f in enumerate(frequencies):
        t = np.asarray(positions, np.float64) * f
        c, s = magnitude * np.cos(t), magnitude * np.sin(t)
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + n)
        xa, xb = x[..., a].astype(np.float64), x[..., b].astype(np.float64)
        out[..., a], out[..., b] = xa * c - xb * s, xa * s + xb * c
    return out


def attention(q, k, v, scale, temp=1.0, causal=True):
    """q [heads, r, d] over k, v [kv_heads, n, d]; a row that sees nothing gives zeros, and what it does not see
    does not count, whatever it holds."""
    heads, r, d = q.shape
    kv, n, _ = k.shape
    out = np.zeros((heads, r, d))
    for h in range(heads):
        kh, vh = k[h // (heads // kv)].astype(np.float64), v[h // (heads // kv)].astype(np.float64)
        for j in range(r):
            end = max(0, j + n - r + 1) if causal else n
            if end == 0:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                s = kh[:end] @ q[h, j].astype(np.float64) * (scale / temp)
                w = np.exp(s - s.max())
                out[h, j] = (w / w.sum()) @ vh[:end]
    return out


def close_enough(got, want, value_max, keys):
    """|got - want| within the roundings of the kernels, for |value| <= value_max and rows of at most `keys` keys:
    the result to fp16 (half a step: 2^-11 of it, 2^-25 below the normal numbers); each probability to fp16 while the sum
    of the weights stays unrounded (2^-11 of sum w |v| <= value_max, and 2^-25 each for probabilities below 2^-14, where
    the largest is at least 1); 32-bit sums over the keys (keys * 2^-24 of sum w |v|, numerator and denominator); and
    the scores, 32-bit sums of d <= 256 products whose absolute values add up to less than 2^5 in the tests here: an
    error below 256 * 2^-24 * 2^5 = 2^-11 in each exponent moves the weighted mean by at most twice that of value_max."""
    want = np.asarray(want, np.float64)
    bound = (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 +
             value_max * (2.0 ** -11 + keys * 2.0 ** -25 + 2 * keys * 2.0 ** -24 + 2 * 2.0 ** -11))
    bad = ~(np.abs(np.asarray(got, np.float64) - want) <= bound)
    bad &= ~(np.isnan(got) & np.isnan(want))
    return not bad.any()


def pages_of(lengths, page_size, rng, spare=2):
    """(number of pages, table [sequences, widest + 1]) with every sequence's pages drawn at random; unused -1."""
    need = [-(-n // page_size) for n in lengths]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(need + [0]) + 1), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return pages, table


def gathered(pool, table_row, n):
    """[kv_heads, n, d] of a [pages, kv_heads, page_size, d] pool."""
    page_size = pool.shape[2]
    parts = [pool[p] for p in table_row[:-(-n // page_size)]]
    if not parts:
        return np.zeros((pool.shape[1], 0, pool.shape[3]), pool.dtype)
    return np.concatenate(parts, axis=1)[:, :n]


def offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def yarn_reference(dims, base, factor, original, fast, slow):
    """Frequencies of the ramp between the dimensions that turn `fast` and `slow` times, one by one."""
    def dim_of(turns):
        return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(dim_of(fast)), 0), min(math.ceil(dim_of(slow)), dims - 1)
    out = []
    for i in range(dims // 2):
        f = 1.0 / base ** (2 * i / dims)
        t = min(max((i - lo) / (hi - lo if hi > lo else 0.001), 0.0), 1.0)
        out.append(f * (1 - t) + f / factor * t)
    return out

"""Plain 64-bit definitions of the heads' norms with rotation over several axes, of the cache in 8 bits and of attention
for drafted trees, in numpy."""
import numpy as np

import sequences_reference as ref


def normed(x, weight, eps):
    """x [..., d], each head by its root mean square."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)


def turned(x, positions, axis, frequencies, magnitude, pairs):
    """x [heads, rows, d] turned by positions [axes, rows], pair i by the axis axis[i]."""
    out = x.astype(np.float64).copy()
    n = len(frequencies)
    for i, f in enumerate(frequencies):
        t = np.asarray(positions[axis[i]], np.float64) * f
        c, s = magnitude * np.cos(t), magnitude * np.sin(t)
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + n)
        xa, xb = out[..., a].copy(), out[..., b].copy()
        out[..., a], out[..., b] = xa * c - xb * s, xa * s + xb * c
    return out


def turned_bound(want, x, n, magnitude, pairs, weight=None):
    """How far the kernels may be off from `want`, for x as it was before the rotation of n pairs: the result's rounding to fp16
    (half a step, 2^-11 of it, 2^-25 below the normal numbers); cosine and sine, whose argument (at most one, in half turns) is
    rounded to 32 bits, pi 2^-25, and which are off by two units, 2^-23: 2^-22 of each partner together, times the magnitude; and
    the roundings of 32 bits, each 2^-24 of a partner: a square mean of d values (d of them, halved by the root), the root, the
    quotient and four products or sums behind them."""
    d = x.shape[-1]
    both = np.abs(x).astype(np.float64)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if pairs else (slice(0, n), slice(n, 2 * n))
    total = both[..., a] + both[..., b]
    both[..., a] = both[..., b] = total
    return np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + both * magnitude * (2.0 ** -22 + (d / 2 + 8) * 2.0 ** -24)


def quantised(y):
    """(codes, scales) of y [..., d] in 64 bits."""
    with np.errstate(invalid="ignore"):
        top = np.abs(y).max(-1)
        exact = np.where(np.isfinite(y).all(-1), top / 127.5, np.nan)
        scale = np.minimum(exact, 513.5).astype(np.float16)
        low = scale.astype(np.float64) < np.minimum(exact, 513.5)
        scale = np.where(low, np.nextafter(scale, np.float16(np.inf)), scale)
        s = scale.astype(np.float64)[..., None]
        codes = np.where(s > 0, np.floor(y / np.where(s > 0, s, 1.0)) + 128, 128)
    return np.clip(codes, 0, 255).astype(np.uint8), scale


def value_of(codes, scales):
    with np.errstate(invalid="ignore"):
        return (codes.astype(np.float64) - 127.5) * scales.astype(np.float64)[..., None]


def ancestors(parents):
    """[rows, rows] booleans: what each drafted token sees of the draft."""
    seen = np.zeros((len(parents), len(parents)), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            seen[j] = seen[p]
        seen[j, j] = True
    return seen


def attention(q, k, v, scale, temp, seen):
    """q [heads, r, d] over k, v [kv_heads, n, d]; seen [r, n].  A row that sees nothing gives zeros, and what it does not
    see does not count, whatever it holds."""
    heads, r, d = q.shape
    kv = k.shape[0]
    out = np.zeros((heads, r, d))
    for h in range(heads):
        for j in range(r):
            at = np.flatnonzero(seen[j])
            if at.size == 0:
                continue
            kh, vh = (t[h // (heads // kv)][at].astype(np.float64) for t in (k, v))
            with np.errstate(invalid="ignore", over="ignore"):
                s = kh @ q[h, j].astype(np.float64) * (scale / temp)
                w = np.exp(s - s.max())
                out[h, j] = (w / w.sum()) @ vh
    return out


def close_enough(got, want, value_max, keys, codes):
    """As for the cache in 16 bits (sequences_reference.py).  Values of codes are not rounded, but a step of 2^-11 more of sum
    w |v| <= value_max is allowed (and 2^-25) for a kernel that rounds them to fp16 first.  Scores of codes are 32-bit sums of
    d <= 128 products of codes up to 255, which begin at -127.5 sum(q): whatever the order, what is summed so far is at most
    127.5 sum |q|, as codes are at most 127.5 off 127.5.  In the tests here sum |q| <= 130, scales are below 0.042, a head's norm keeps
    sum |q| below 80 where they are above 0.03, and the factor is at most 1 / (0.9 sqrt(d)): d roundings of 2^-24 of
    127.5 * 130 * 0.03 / (0.9 * 11.3) for d = 128 make less than 2^-11 in each exponent, as there; of smaller d, where sum |q| is
    below 1.3 d, less still."""
    want = np.asarray(want, np.float64)
    extra = value_max * 2.0 ** -11 + 2.0 ** -25 if codes else 0.0
    bound = (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + extra +
             value_max * (2.0 ** -11 + keys * 2.0 ** -25 + 2 * keys * 2.0 ** -24 + 2 * 2.0 ** -11))
    bad = ~(np.abs(np.asarray(got, np.float64) - want) <= bound)
    bad &= ~(np.isnan(got) & np.isnan(want))
    return not bad.any()


def causal(r, n):
    return np.arange(n)[None, :] <= np.arange(r)[:, None] + n - r


def with_past(tree, n):
    """[r, n] of a draft that is the last r of n keys (more drafted tokens than keys: the last n of them)."""
    r = len(tree)
    return np.concatenate([np.ones((r, max(n - r, 0)), bool), tree[:, max(r - n, 0):]], axis=1)


def pages_for(lengths, page_size, rng):
    return ref.pages_of(lengths, page_size, rng)

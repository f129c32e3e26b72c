"""How much of what a kernel of attention over codes is off may be roundings, told by the root mean square over many results.

The last rounding, to fp16, is the definition's own: r = rms(fp16(want) - want).  A rounding to fp16 of factors whose size is spread evenly
over a power of two is off by 2^-11 / sqrt(3) * sqrt(E[1 / m^2]) = 2^-11 * 0.577 * 0.736 = 2^-11 * 0.425 in the mean (m the mantissa, from
1 to 2, E[1 / m^2] = 0.75 / (2 ln 2)).  Results have that of their own size; and where results are sums of many products w v of either
sign, one rounding of each w, or of each v, has the same of the sum's.  So with k such roundings of different origin the root mean square is
sqrt(1 + k) r: 1 with probabilities of 22 bits, 1.41 with those of 11, 1.73 with values of 11 bits as well.

What 32 bits leave is far less: a score is a sum of d products, each partial sum off by 2^-24 of at most 127.5 sum |q|; here sum |q| <=
1.2 d, scales are 0.03 at most and the factor is 1 / sqrt(d), so sqrt(d) independent ones are 2^-24 * 127.5 * 1.2 * d * 0.03 <= 2^-15 of
a weight for d <= 128, and 2^-24 of 127.5 times the weights' sum at each of n / 32 + 2 steps <= 20 is 2^-15 of the values' size: together less than
0.1 r, 1.005 of it.  The rms over N results is itself known to 1 / sqrt(2 N), under 0.01 for N > 6000, three times that for chance: the
bounds are 1.005 * 1.03 < 1.04 and 1.42 * 1.03 < 1.5."""
import numpy as np

import step_reference as step

WHOLE, ROUNDED = 1.04, 1.5   # probabilities of 22 bits, and of 11


def times_the_last(got, want):
    """rms(got - want) over that of the last rounding alone."""
    want = np.asarray(want, np.float64)
    rms = lambda x: np.sqrt(np.mean(x * x))  # noqa: E731
    return rms(np.asarray(got, np.float64) - want) / rms(want.astype(np.float16) - want)


def rounded(q, codes, scales, scale, seen, weights=None, values=False, top=9.0):
    """The definition (step_reference.attention) for one key head of codes [2][n, d] and scales [2][n], q [rows, d], with probabilities (times the value's
    scale) as fp16 ("half") or as two of them ("two halves"), and values as fp16 or as they are."""
    k, v = (step.value_of(codes[t], scales[t]) for t in (0, 1))
    s = q.astype(np.float64) @ k.T * (scale * np.log2(np.e))
    s = np.where(seen, s, -np.inf)
    by = np.ones(len(s[0])) if values else scales[1].astype(np.float64)  # (what goes into the probability)
    p = np.exp2(s - (s + np.log2(by)).max(-1, keepdims=True) + top)
    ps, units = p * by, v.astype(np.float16).astype(np.float64) if values else codes[1].astype(np.float64) - 127.5
    if weights == "half":
        ps = ps.astype(np.float16).astype(np.float64)
    elif weights == "two halves":
        h = ps.astype(np.float16).astype(np.float64)
        ps = h + (ps - h).astype(np.float16).astype(np.float64)
    return (ps @ units / p.sum(-1, keepdims=True)).astype(np.float16)

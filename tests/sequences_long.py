"""Attention over long contexts: data whose result depends on every place that a division of the keys can lose, the definition in
64 bits, and a bound on the kernels' error that is far below what losing one of them changes."""
import math

import torch

TILE = 64   # keys: the larger of the kernels' tiles


def marked_keys(n):
    """Keys that share most of the weight: in the first tile, at a tile's and at a piece's border, in the middle, and in the last
    tiles down to the last key, which lies in a page of its own where n is one more than whole pages."""
    at = {0, TILE - 1, TILE, 127, n // 4, n // 2 - 1, n // 2, 3 * n // 4, n - TILE - 1, n - 33, n - 17, n - 2, n - 1}
    return sorted(x for x in at if 0 <= x < n)


def sequence(rows, n, heads, kv, d, gen, device):
    """q [heads, rows, d], k, v [kv, n, d] of fp16.  The marked keys weigh as much as all others together: they point the way of
    every query (to which noise is added), by 1 / 13 of the sum each where a row sees them all."""
    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=device)
    way = normal(d)
    way *= math.sqrt(d) / way.norm()
    scale = 1.0 / math.sqrt(d)
    q, k, v = way + 0.3 * normal(heads, rows, d), normal(kv, n, d), normal(kv, n, d)
    k -= (k @ way)[..., None] * way / d                       # (the others: across the way)
    at = marked_keys(n)
    k[:, at] = way * math.log(n / len(at)) * scale            # scores of ln(n / 13): exp of it is their share
    return q.half(), k.half(), v.half(), scale


class Definition:
    """out [heads, rows, d] in 64 bits over the keys that `keep` leaves (all: None), causal from the last key on; `error(steps)`,
    how far a kernel may be off."""

    def __init__(self, q, k, v, scale, causal=True, keep=None):
        heads, rows, d = q.shape
        kv, n, _ = k.shape
        parts = []
        for h in range(heads):
            key, value = k[h // (heads // kv)].double(), v[h // (heads // kv)].double()
            s = q[h].double() @ key.t().contiguous() * scale
            sizes = (q[h].double().abs() @ key.abs().t().contiguous()).amax(-1, keepdim=True) * scale
            if causal:
                s.masked_fill_(torch.arange(n, device=q.device)[None] > torch.arange(n - rows, n, device=q.device)[:, None], -math.inf)
            if keep is not None:
                s[:, ~keep] = -math.inf
            w = (s - s.amax(-1, keepdim=True)).exp()
            total = w.sum(-1, keepdim=True)
            parts.append((w @ value / total, w @ value.abs() / total, value.abs().sum(0) / total, sizes))
        self.out, self.weighed, self.values, self.sizes = (torch.stack(x) for x in zip(*parts))
        self.n, self.d = n, d

    def error(self, steps):
        """With w the weights over their sum, `weighed` = sum w |v|, and `steps` the 32-bit additions that one key's product goes
        through on its way to the result:
        - the result to fp16: 2^-11 of it, 2^-25 below the normal numbers;
        - each weight to fp16: 2^-11 of weighed; below 2^-14, 2^-25 where the largest is at least 2^6: 2^-31 of it, for
          every key, over the sum of the weights;
        - sums in 32 bits: 2^-24 a step of weighed, and of the result for the sum of the weights, which a lane makes of
          at most a quarter of the keys, a part at a time: n / 4 + 600 steps;
        - a score, 32-bit sums of d products: d 2^-24 of the sum of their sizes, and its exponential 2^-18 (32-bit exponents below
          2^6): twice that of weighed, as it moves the weight and the sum."""
        score = self.d * 2.0 ** -24 * self.sizes + 2.0 ** -18
        return (self.out.abs() * (2.0 ** -11 + (self.n / 4 + 600) * 2.0 ** -24) + 2.0 ** -25 +
                self.weighed * (2.0 ** -11 + steps * 2.0 ** -24 + 2 * score) + self.values * 2.0 ** -31)

    def agrees(self, got, steps):
        return bool(((got.double() - self.out).abs() <= self.error(steps)).all())


def matrix_steps(n):
    """Of the matrix-core kernels: 16 keys or more to an instruction (whose own sums are counted among the 600, with the parts')."""
    return n / 16 + 600


def row_steps(n):
    """Of the kernel of a wavefront per row: one key after the other."""
    return n + 64

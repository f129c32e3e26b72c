"""Attention over long contexts in 8 bits: the definition in 64 bits over what the codes stand for, and a bound on the error of the
kernels that take the codes as they are (sequences_long.py has the data, and what is said of values in 16 bits)."""
import torch

from sequences_long import Definition


def quantised(x):
    """Codes and fp16 scales of x [..., d], in 64 bits."""
    x = x.double()
    exact = x.abs().amax(-1) / 127.5
    scale = exact.half()
    scale = torch.where(scale.double() < exact, (scale.view(torch.int16) + 1).view(torch.float16), scale)  # (the next one up)
    assert (scale.double() >= exact).all() and (scale > 0).all()
    codes = (torch.floor(x / scale.double()[..., None]) + 128).clamp(0, 255).to(torch.uint8)
    return codes, scale


class Codes(Definition):
    """q [heads, rows, d]; keys and values as pairs of codes [kv, n, d] and scales [kv, n]."""

    def __init__(self, q, keys, values, scale, causal=True, keep=None):
        k, v = ((codes.double() - 127.5) * scales.double()[..., None] for codes, scales in (keys, values))
        super().__init__(q, k, v, scale, causal, keep)
        self.sums = q.double().abs().sum(-1, keepdim=True) * 382.5 * float(keys[1].max()) * scale
        self.steps_of = 382.5 * float(values[1].max())
        self.spread = float(values[1].max()) / float(values[1].min())

    def matrix_error(self, steps):
        """Of the matrix-core kernels, as Definition.error but for
        - a score: the sum of codes up to 255 begins at -127.5 sum(q), so that its parts add up to 382.5 sum |q| times the key's scale;
        - sums over the keys: of the rounded probability, which holds the value's scale, times a code up to 255, less 127.5 times the
          sum of those probabilities: 382.5 times the largest scale for each step;
        - a probability below 2^-14: 2^-25, or 2^-31 of the largest one with its scale, times the code's distance from 127.5: the
          largest scale over its own of the value."""
        score = self.d * 2.0 ** -24 * self.sums + 2.0 ** -18
        return (self.out.abs() * (2.0 ** -11 + (self.n / 4 + 600) * 2.0 ** -24) + 2.0 ** -25 + self.steps_of * steps * 2.0 ** -24 +
                self.weighed * (2.0 ** -11 + 2 * score) + self.values * self.spread * 2.0 ** -31)

    def matrix_agrees(self, got, steps):
        return bool(((got.double() - self.out).abs() <= self.matrix_error(steps)).all())

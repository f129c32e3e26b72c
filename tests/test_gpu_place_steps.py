"""Heads normed, turned and put to their places where rows are so many that a wavefront goes through several steps of heads: from one
step's queries to keys to values, each with norms of its own.  Against the definitions of step_reference.py, whose tolerance this is;
codes and scales are those of 64 bits."""
import numpy as np
import pytest

import torch

from adrastea_amd import GpuKernels, HeadNorm, PagedBatch, PagedCache, RotaryAxes, RotaryLayout, TensorView, rotary_frequencies
import sequences_reference as ref
import step_reference as step
from test_gpu_cache_u8 import SENTINEL, Cache, axis_of, dev, f16, heads_view, ints, sections_of

pytestmark = pytest.mark.gpu

EPS = 1e-5

# (sequences of (rows, keys), heads, kv heads, d, page, rotated values, axes, pairs): steps of heads, and wavefronts that share them
CASES = {"three steps": ([(4000, 4017), (200, 205)], 8, 8, 128, 16, 128, 1, False),        # queries, keys, values
         "six steps, two wavefronts": ([(2000, 2000), (100, 900)], 32, 8, 128, 64, 128, 3, True),
         "two steps of 16": ([(4100, 4100)], 20, 4, 64, 32, 32, 2, False),                 # queries, keys and values in the last
         "two steps of 4": ([(4096, 4100), (9, 9)], 3, 1, 256, 16, 256, 1, True),
         "two steps, five lanes of eight": ([(4200, 4200)], 6, 2, 80, 16, 80, 2, False),
         "a step each": ([(700, 700), (300, 301)], 8, 8, 128, 16, 128, 1, False)}


class Step:
    def __init__(self, case, q_norm, k_norm, seed):
        self.seqs, self.heads, self.kv, self.d, self.page, self.rot, axes, self.pairs = case
        rng = np.random.default_rng(seed)
        rows, self.lengths = [r for r, _ in self.seqs], [n for _, n in self.seqs]
        self.starts = ref.offsets(rows)
        self.n, self.total = int(self.starts[-1]), sum(rows) + 2
        self.qkv = f16(rng, self.total, self.heads + 2 * self.kv, self.d, std=2.0)
        self.weights = f16(rng, self.d) if q_norm else None, f16(rng, self.d) if k_norm else None
        self.norms = [None if w is None else HeadNorm(dev(w), EPS) for w in self.weights]
        sections = sections_of(self.rot // 2, axes)
        self.axis, self.positions = axis_of(sections), rng.integers(0, 100000, (axes, self.total))
        self.rotary = RotaryAxes.new(self.rot, sections, layout=RotaryLayout.PAIRS if self.pairs else RotaryLayout.HALVES)
        packed = dev(self.qkv)
        at = self.heads, self.heads + self.kv
        self.views = [heads_view(t) for t in (packed[:, :at[0]], packed[:, at[0]:at[1]], packed[:, at[1]:]) if t.shape[1] > 0]
        self.out = torch.full((self.total, self.heads, self.d), SENTINEL, dtype=torch.float16, device="cuda")
        self.place = [(i, n - r + j) for i, (r, n) in enumerate(self.seqs) for j in range(r)]

    def turned(self, which):
        """(what is turned, the result) [heads, rows, d] of queries (0) or keys (1)."""
        first = 0 if which == 0 else self.heads
        x = self.qkv[:self.n, first:first + (self.heads if which == 0 else self.kv)]
        y = x.astype(np.float64) if self.weights[which] is None else step.normed(x, self.weights[which], EPS)
        y = y.transpose(1, 0, 2)
        return y, step.turned(y, self.positions[:, :self.n], self.axis, rotary_frequencies(self.rot)[0], 1.0, self.pairs)

    def near(self, got, which):
        y, want = self.turned(which)
        return (np.abs(got.transpose(1, 0, 2) - want) <= step.turned_bound(want, y, self.rot // 2, 1.0, self.pairs)).all()

    def check_queries(self):
        got = self.out.cpu().numpy()
        assert (got[self.n:] == SENTINEL).all()
        assert self.near(got[:self.n], 0)

    def slots(self, table):
        """(page, slot) of each row"""
        return np.array([table[i, x // self.page] for i, x in self.place]), np.array([x % self.page for _, x in self.place])


@pytest.mark.parametrize("norms", ["both", "keys", "queries", "none"])
@pytest.mark.parametrize("name", CASES)
def test_into_16_bits(name, norms):
    s = Step(CASES[name], norms in ("both", "queries"), norms in ("both", "keys"), len(name))
    pages, table = ref.pages_of(s.lengths, s.page, np.random.default_rng(1))
    pool = torch.full((2, pages, s.kv, s.page, s.d), SENTINEL, dtype=torch.float16, device="cuda")
    q, k, v = s.views
    GpuKernels().append_norm_f16(PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1])),
                                 PagedBatch(ints(s.starts), ints(s.lengths), ints(table)), k, v, s.rotary, heads_view(s.out), q, ints(s.positions), *s.norms)
    s.check_queries()
    keys, values = pool.cpu().numpy()
    at = s.slots(table)
    assert s.near(keys[at[0], :, at[1]], 1)
    assert np.array_equal(values[at[0], :, at[1]], s.qkv[:s.n, s.heads + s.kv:])
    free = np.ones((pages, s.page), bool)
    free[at] = False
    assert (keys.transpose(0, 2, 1, 3)[free] == SENTINEL).all() and (values.transpose(0, 2, 1, 3)[free] == SENTINEL).all()


@pytest.mark.parametrize("norms", ["both", "queries", "none"])
@pytest.mark.parametrize("name", CASES)
def test_into_8_bits(name, norms):
    s = Step(CASES[name], norms in ("both", "queries"), norms == "both", len(name) + 1)
    cache = Cache(s.lengths, s.kv, s.d, s.page, np.random.default_rng(2), "tokens" if s.pairs else "heads")
    codes, scales = cache.codes.copy(), cache.scales.copy()
    q, k, v = s.views
    batch = PagedBatch(ints(s.starts), ints(s.lengths), ints(cache.table))
    GpuKernels().append_u8(cache.handle, batch, k, v, s.rotary, heads_view(s.out), q, ints(s.positions), *s.norms)
    s.check_queries()
    at = s.slots(cache.table)
    for t, y in ((0, s.turned(1)[1].transpose(1, 0, 2)), (1, s.qkv[:s.n, s.heads + s.kv:].astype(np.float64))):
        codes[t][at[0], :, at[1]], scales[t][at[0], :, at[1]] = step.quantised(y)
    h = cache.handle
    for t, (c, f) in enumerate(((h.key, h.key_scale), (h.value, h.value_scale))):
        assert np.array_equal(f.storage.cpu().numpy(), scales[t], equal_nan=True), "scales"
        assert np.array_equal(c.storage.cpu().numpy(), codes[t]), "codes"


@pytest.mark.parametrize("norm", [True, False], ids=["normed", "plain"])
@pytest.mark.parametrize("heads,rows,d,rot,axes,pairs", [(16, 4200, 80, 80, 2, False), (32, 2100, 128, 128, 1, False), (40, 4097, 64, 48, 3, True),
                                                         (5, 4500, 512, 512, 1, False), (33, 5000, 24, 16, 1, False)])
def test_alone(heads, rows, d, rot, axes, pairs, norm):
    s = Step(([(rows, rows)], heads, 0, d, 16, rot, axes, pairs), norm, False, rows)
    GpuKernels().norm_rotary_f16(heads_view(s.out[:rows]), heads_view(dev(s.qkv)[:rows]), ints(s.positions[:, :rows]), s.rotary, s.norms[0])
    s.check_queries()

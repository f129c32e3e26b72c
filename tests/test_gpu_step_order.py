"""Blocks that start with the longest sequence, and queries that are turned where they are: more blocks than compute units, sequences of
equal lengths, without keys or rows, up to and beyond as many as are ordered."""
import numpy as np
import pytest
import torch

from adrastea_amd import GpuKernels, HeadNorm, PagedBatch, PagedCache, RotaryAxes, TensorView
import sequences_reference as ref
import step_reference as step
from test_gpu_cache_u8 import CAUSAL, NONE, SENTINEL, Cache, Paged, dev, f16, heads_view, ints
from test_gpu_draft_tree import Drafts, random_parents

pytestmark = pytest.mark.gpu

COUNTS = [2, 63, 64, 65, 130]


def lengths_of(n, rng):
    out = rng.integers(0, 400, n)
    out[rng.integers(0, n, n // 3)] = 77       # (equal ones)
    out[rng.integers(0, n, n // 8)] = 0
    out[rng.integers(0, n)] = 1500
    return [int(x) for x in out]


@pytest.mark.parametrize("n", COUNTS)
def test_tokens_of_sequences_of_any_order(n):
    rng = np.random.default_rng(n)
    seqs = [(int(r), x) for r, x in zip(rng.integers(0, 3, n), lengths_of(n, rng))]
    p = Paged(seqs, 300 if n == 2 else 16, 150 if n == 2 else 16, 64, 16, seed=n)
    kern = GpuKernels()
    for mask in (CAUSAL, NONE):
        p.out_t.fill_(SENTINEL)
        kern.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125, 1.0, mask)
        p.check(0.125, mask)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", COUNTS)
def test_drafts_of_sequences_of_any_order(n, bits):
    rng = np.random.default_rng(n)
    rows = [int(r) for r in rng.integers(0, 9, n)]
    heads, kv = (300, 150) if n == 2 else (32, 8)
    t = Drafts([random_parents(r, rng) for r in rows], lengths_of(n, rng), heads, kv, 64, 16, bits, seed=n)
    t.check(t.run(GpuKernels(), 0.125), t.want(0.125))


def test_offsets_that_decrease():
    """Rows that only one sequence claims are right, whatever the order of the blocks."""
    p = Paged([(10, 300), (0, 40), (10, 500), (5, 900)], 128, 64, 64, 16, seed=65)
    want = p.want(0.125, CAUSAL)
    batch = PagedBatch(ints([0, 10, 5, 20, 25]), p.batch.lengths, p.batch.table)
    GpuKernels().attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, batch, 0.125)
    got = p.out_t.cpu().numpy()
    behind = ref.attention(p.q[5:20].transpose(1, 0, 2), *p.cache.values(2, 500), 0.125).transpose(1, 0, 2)
    top = 127.5 * np.nanmax(p.cache.scales[1].astype(np.float64))
    for part, expect, keys in ((slice(0, 5), want[:5], 300), (slice(10, 20), behind[5:], 500), (slice(20, 25), want[20:25], 900)):
        assert step.close_enough(got[part], expect, top, keys, True)
    assert np.isfinite(got[5:10]).all() and (got[25:] == SENTINEL).all()


@pytest.mark.parametrize("d,heads,kv", [(128, 32, 8), (64, 5, 5), (80, 12, 4), (7, 3, 1)])
@pytest.mark.parametrize("rows", [1, 3, 70, 5000])
def test_queries_turned_in_place(rows, d, heads, kv):
    """What the calls write into another tensor, to the bit."""
    rng = np.random.default_rng(d + rows)
    kern, total = GpuKernels(), rows + 1
    qkv = dev(f16(rng, total, heads + 2 * kv, d))
    weight, dims = HeadNorm(dev(f16(rng, d)), 1e-6), d // 2 * 2 if d < 64 else d
    rotary, positions = RotaryAxes.new(dims, [dims // 2]), ints(rng.integers(0, 9999, (1, total)))
    batch = PagedBatch(ints([0, rows]), ints([rows + 3]), ints(np.arange(rows // 16 + 1)[None]))
    half = [torch.zeros(rows // 16 + 1, kv, 16, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    codes = Cache([rows + 3], kv, d, 16, rng)
    codes_batch = PagedBatch(batch.row_offsets, batch.lengths, ints(codes.table))

    def run(into):
        x, y = qkv.clone(), qkv.clone()
        out = [torch.full((total, heads, d), SENTINEL, dtype=torch.float16, device="cuda") for _ in range(3)] if not into else [x[:, :heads], y[:, :heads],
                                                                                                                      qkv[:, :heads].clone()]
        kern.append_norm_f16(PagedCache(*(TensorView.of(t) for t in half)), batch, heads_view(x[:, heads:heads + kv]), heads_view(x[:, heads + kv:]),
                             rotary, heads_view(out[0]), heads_view(x[:, :heads]), positions, weight, weight)
        kern.append_u8(codes.handle, codes_batch, heads_view(y[:, heads:heads + kv]), heads_view(y[:, heads + kv:]), rotary, heads_view(out[1]),
                       heads_view(y[:, :heads]), positions, weight, weight)
        z = out[2] if into else qkv[:, :heads]
        kern.norm_rotary_f16(heads_view(out[2]), heads_view(z), positions, rotary, weight)
        return [t.clone() for t in out]
    for i, (apart, within) in enumerate(zip(run(False), run(True))):
        assert torch.equal(apart[:rows], within[:rows]) and apart[:rows].isfinite().all()
        if i < 2:                                  # (the row of no sequence is left)
            assert (apart[rows:] == SENTINEL).all() and torch.equal(within[rows:], qkv[rows:, :heads])

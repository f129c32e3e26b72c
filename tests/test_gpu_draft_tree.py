"""Attention of drafted trees over the paged cache in 16 and in 8 bits, on the GPU, against a plain 64-bit definition
(step_reference.py)."""
import numpy as np
import pytest
import torch

from adrastea_amd import (AdrasteaError, DraftTree, GpuKernels, MatmulTracer, PagedBatch, PagedCache, PagedCacheU8, TensorView, _ffi)
import sequences_reference as ref
import step_reference as step

pytestmark = pytest.mark.gpu

SENTINEL = 777.0
KNOBS = {"a row to a wavefront": 1, "few rows, 2 waves": 2, "few rows, 4 waves": 3, "few rows, shared": 4, "many rows": 5,
         "many rows, 2 groups": 6, "many rows, shared": 7, "many rows, 2 groups, shared": 8}


@pytest.fixture(params=["unshared", "pool", "workspace", *KNOBS])
def kern(request):
    lib = _ffi.lib()
    forced = KNOBS.get(request.param, 0)
    assert lib.adr_debug_knob(2, forced) == 0
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES if request.param == "pool" or forced else 0)
    yield GpuKernels(workspace_bytes=(96 << 20) if request.param == "workspace" else 0)
    lib.adr_set_held_workspace_limit(0)
    lib.adr_debug_knob(2, 0)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def heads_view(t):
    return TensorView.of(t.permute(1, 0, 2))


class Drafts:
    """Drafts of `parents` over sequences of so many keys in front of them; what no row may read is NaN."""

    def __init__(self, parents, past, heads, kv, d, page, bits, seed=0, spare=2):
        rng = np.random.default_rng(seed)
        self.heads, self.d, self.bits = heads, d, bits
        self.trees = [step.ancestors(p) for p in parents]
        rows = [len(p) for p in parents]
        self.lengths = [max(n + r, 0) for n, r in zip(past, rows)]
        self.starts = ref.offsets(rows)
        self.rows = sum(rows) + spare
        pages, self.table = ref.pages_of(self.lengths, page, rng)
        self.q = rng.standard_normal((self.rows, heads, d)).astype(np.float16)
        self.q_t = dev(self.q)
        shape = (2, pages, kv, page)
        if bits == 16:
            pool = np.full((*shape, d), np.nan, np.float16)
        else:
            pool, scales = np.zeros((*shape, d), np.uint8), np.full(shape, np.nan, np.float16)
        for i, n in enumerate(self.lengths):
            for x0 in range(0, n, page):
                m, at = min(page, n - x0), self.table[i, x0 // page]
                if bits == 16:
                    pool[:, at, :, :m] = rng.standard_normal((2, kv, m, d)).astype(np.float16)
                else:
                    pool[:, at, :, :m] = rng.integers(0, 256, (2, kv, m, d))
                    scales[:, at, :, :m] = rng.uniform(0.008, 0.016, (2, kv, m)).astype(np.float16)
        self.pool, self.scales = pool, None if bits == 16 else scales
        self.upload()
        self.batch = PagedBatch(ints(self.starts), ints(self.lengths), ints(self.table), max(rows), max(self.lengths))
        self.tree = DraftTree(torch.cat([DraftTree.of(parents).bits, torch.full((spare, (max(rows + [1]) + 31) // 32), -1,
                                                                                dtype=torch.int32, device="cuda")]))
        self.out_t = torch.full((self.rows, heads, d), SENTINEL, dtype=torch.float16, device="cuda")

    def upload(self):
        k, v = dev(self.pool[0]), dev(self.pool[1])
        if self.bits == 16:
            self.cache = PagedCache(TensorView.of(k), TensorView.of(v))
        else:
            self.cache = PagedCacheU8(TensorView.of(k), TensorView.of(dev(self.scales[0])), TensorView.of(v),
                                      TensorView.of(dev(self.scales[1])))

    def run(self, kern, scale, temp=1.0):
        f = kern.attention_tree_f16 if self.bits == 16 else kern.attention_tree_u8
        f(heads_view(self.out_t), heads_view(self.q_t), self.cache, self.batch, self.tree, scale, temp)
        return self.out_t.cpu().numpy()

    def values(self, i, n):
        if self.bits == 16:
            return [ref.gathered(self.pool[t], self.table[i], n) for t in (0, 1)]
        return [step.value_of(ref.gathered(self.pool[t], self.table[i], n),
                              ref.gathered(self.scales[t][..., None], self.table[i], n)[..., 0]) for t in (0, 1)]

    def want(self, scale, temp=1.0, trees=None):
        out = np.full((self.rows, self.heads, self.d), SENTINEL)
        for i, n in enumerate(self.lengths):
            tree = (trees or self.trees)[i]
            a, b = self.starts[i], self.starts[i + 1]
            k, v = self.values(i, n)
            out[a:b] = step.attention(self.q[a:b].transpose(1, 0, 2), k, v, scale, temp, step.with_past(tree, n)).transpose(1, 0, 2)
        return out

    def top(self):
        return 127.5 * 0.016 if self.bits == 8 else np.nanmax(np.abs(self.pool[1].astype(np.float64)), initial=0.0)

    def check(self, got, want):
        assert (got[self.starts[-1]:] == SENTINEL).all(), "rows behind the last sequence"
        n = self.starts[-1]
        assert step.close_enough(got[:n], want[:n], self.top(), max(self.lengths + [1]), self.bits == 8)


def random_parents(rows, rng):
    return [-1] + [int(rng.integers(-1, j)) for j in range(1, rows)] if rows else []


# (rows of each draft, keys in front of each, heads, kv heads, d, page)
CASES = [([1], [0], 1, 1, 64, 16), ([5], [37], 4, 4, 128, 16), ([3, 0, 16, 1], [300, 9, 0, 63], 8, 2, 128, 16), ([31], [1], 4, 1, 64, 32),
         ([32, 33], [31, 64], 4, 1, 64, 16), ([64, 65, 100], [500, 3, 128], 2, 2, 128, 64), ([61], [1100], 8, 2, 64, 16),
         ([7, 7], [-3, 20], 2, 1, 64, 16), ([12], [90], 3, 1, 80, 16), ([4, 9], [30, 11], 2, 1, 7, 4), ([150], [200], 4, 1, 128, 16),
         ([20], [77], 5, 1, 96, 16), ([13] * 30, list(range(0, 300, 10)), 4, 2, 64, 32)]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("case", CASES, ids=["r%s_h%d_%d_d%d" % ("-".join(map(str, c[0][:4])), *c[2:5]) for c in CASES])
def test_trees(kern, case, bits):
    rng = np.random.default_rng(sum(case[0]))
    p = Drafts([random_parents(r, rng) for r in case[0]], *case[1:], bits, seed=sum(case[1]) % 1000)
    scale = 1.0 / np.sqrt(p.d)
    p.check(p.run(kern, scale, 1.2), p.want(scale, 1.2))


@pytest.mark.parametrize("bits", [16, 8])
def test_any_bits(kern, bits):
    """Rows that see nothing of their draft, not even themselves, all of it, or what no tree would say; fewer words than tokens;
    a pitch between the rows' words."""
    rng = np.random.default_rng(3)
    p = Drafts([random_parents(r, rng) for r in (40, 3, 70)], [21, 0, 130], 4, 2, 64, 16, bits)
    trees = [rng.random((r, r)) < 0.5 for r in (40, 3, 70)]
    trees[0][3], trees[0][4], trees[1][:] = False, True, False
    for words in (3, 1):
        wide = np.zeros((p.rows, 5), np.int64)
        for i, t in enumerate(trees):
            for j, seen in enumerate(t):
                for w in range(words):
                    wide[p.starts[i] + j, w] = sum(1 << b for b in range(32) if 32 * w + b < len(seen) and seen[32 * w + b])
        wide[:, words:] = -1
        bits_t = dev(wide.astype(np.uint32).view(np.int32))
        p.tree = DraftTree(bits_t[:, :words])
        cut = [t & (np.arange(len(t)) < 32 * words) for t in trees]
        got = p.run(kern, 0.125)
        p.check(got, p.want(0.125, trees=cut))
        assert (got[40:43] == 0).all(), "rows that see no key"


@pytest.mark.parametrize("bits", [16, 8])
def test_a_chain_is_the_causal_mask(kern, bits):
    p = Drafts([list(range(-1, 49))], [333], 4, 2, 64, 16, bits)
    want = p.want(0.125)
    p.check(p.run(kern, 0.125), want)
    p.out_t.fill_(SENTINEL)
    f = kern.attention_paged_f16 if bits == 16 else kern.attention_paged_u8
    f(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.125)
    p.check(p.out_t.cpu().numpy(), want)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows,past", [(6, 40), (70, 100)])
def test_what_a_row_does_not_see_never_reaches_it(kern, bits, rows, past):
    """A drafted token whose key or value is no number: only the rows that see it change."""
    parents = [-1] + [0] * (rows - 1)
    p = Drafts([parents, [-1]], [past, 30], 4, 2, 64, 16, bits)
    want = p.want(0.125)
    x = past + rows // 2  # the key of drafted token rows // 2, which no other row sees
    at = (p.table[0, x // 16], slice(None), x % 16)
    target = p.pool if bits == 16 else p.scales
    clean = target.copy()
    for which, bad in ((0, np.nan), (1, np.nan), (1, np.inf)):
        target[:] = clean
        target[(which, *at)] = bad
        p.upload()
        got = p.run(kern, 0.125)
        assert not np.isfinite(got[rows // 2]).any()
        rest = np.arange(p.starts[-1]) != rows // 2
        assert step.close_enough(got[:p.starts[-1]][rest], want[:p.starts[-1]][rest], p.top(), past + rows, bits == 8)


def test_refusals_through_python():
    kern = GpuKernels()
    p = Drafts([[-1, 0, 0]], [20], 4, 2, 64, 16, 16)
    out, q = heads_view(p.out_t), heads_view(p.q_t)
    for bad in (lambda: DraftTree(torch.zeros(5, dtype=torch.int32, device="cuda")), lambda: DraftTree(torch.zeros(5, 1, device="cuda")),
                lambda: kern.attention_tree_f16(out, q, p.cache, p.batch, DraftTree(p.tree.bits[:2]), 0.1),
                lambda: kern.attention_tree_f16(out, q, p.cache, p.batch, DraftTree(p.tree.bits.cpu()), 0.1)):
        with pytest.raises(AssertionError):
            bad()
    for bad in ([[0]], [[-1, 1]], [[-1, -2]]):
        with pytest.raises(ValueError):
            DraftTree.of(bad)
    with pytest.raises(AdrasteaError):
        kern.attention_tree_f16(out, q, p.cache, p.batch, p.tree, 0.0)
    assert (p.out_t == SENTINEL).all()


def test_the_tracer_forwards():
    kern = MatmulTracer(GpuKernels())
    for bits in (16, 8):
        p = Drafts([[-1, 0, 0]], [20], 4, 2, 64, 16, bits)
        p.check(p.run(kern, 0.125), p.want(0.125))

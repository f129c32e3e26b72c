"""Heads normed and turned, the caches in 16 and 8 bits and drafted trees as they are used together, and over the sizes and the
circumstances that a program has: long contexts, offsets beyond 32 bits, graphs, streams, sequences that do not fit their hints."""
import numpy as np
import pytest
import torch

from adrastea_amd import (attention_paged_u8_workspace_bytes, attention_tree_workspace_bytes, DraftTree, GpuKernels, HeadNorm, MatmulMask, PagedBatch, PagedCache, PagedCacheU8,
                          RotaryAxes, TensorLayout, TensorView, _ffi, rotary_frequencies)
import sequences_reference as ref
import step_reference as step
from sequences_long import matrix_steps, row_steps, sequence
from step_long import Codes, quantised
from test_gpu_cache_u8 import FORMS, SENTINEL, Paged, dev, f16, heads_view, ints, shared_keys  # noqa: F401 (a fixture)
from test_gpu_draft_tree import Drafts, random_parents

pytestmark = pytest.mark.gpu

CAUSAL, NONE = MatmulMask.CAUSAL, MatmulMask.NONE


# ---- a conversation ---------------------------------------------------------------------------------------------

class Conversation:
    """Two sequences whose heads are normed and turned by positions on two axes, and what the caches have to hold."""
    heads, kv, d, page, total = 8, 2, 64, 16, 10

    def __init__(self, kern, bits):
        self.kern, self.bits, self.rng = kern, bits, np.random.default_rng(bits)
        rng, shape = self.rng, (self.total * 2, self.page, self.kv)
        self.weights = [f16(rng, self.d, std=0.2) + np.float16(1.0) for _ in range(2)]
        self.norms = [HeadNorm(dev(w), 1e-6) for w in self.weights]
        self.rotary = RotaryAxes.new(self.d, [20, 12])
        self.axis, self.frequencies = [0] * 20 + [1] * 12, rotary_frequencies(self.d)[0]
        self.table = rng.permutation(2 * self.total).reshape(2, self.total).astype(np.int32)
        if bits == 16:
            self.pools = [torch.full((*shape, self.d), torch.nan, dtype=torch.float16, device="cuda") for _ in range(2)]
            self.cache = PagedCache(*(TensorView.of(t.permute(0, 2, 1, 3)) for t in self.pools))
        else:
            self.pools = [torch.zeros(*shape, self.d, dtype=torch.uint8, device="cuda") for _ in range(2)]
            self.scales = [torch.full(shape, torch.nan, dtype=torch.float16, device="cuda") for _ in range(2)]
            self.cache = PagedCacheU8(*(TensorView.of(t.permute(0, 2, 1, 3) if t.dim() == 4 else t.permute(0, 2, 1))
                                        for pair in zip(self.pools, self.scales) for t in pair))
        self.done = [0, 0]
        self.held = [[np.zeros((0, self.kv, self.d))] * 2 for _ in range(2)]   # keys and values of each sequence, in 64 bits

    def batch(self, rows):
        return PagedBatch(ints(ref.offsets(rows)), ints(self.done), ints(self.table), max(rows), max(self.done))

    def append(self, qkv, positions, rows):
        """Rows behind the `done` keys of each sequence: the turned queries, checked; the cache's content, checked too."""
        self.done = [n + r for n, r in zip(self.done, rows)]
        packed, h, kv = dev(qkv), self.heads, self.kv
        turned = torch.full((len(qkv), h, self.d), SENTINEL, dtype=torch.float16, device="cuda")
        f = self.kern.append_norm_f16 if self.bits == 16 else self.kern.append_u8
        f(self.cache, self.batch(rows), heads_view(packed[:, h:h + kv]), heads_view(packed[:, h + kv:]), self.rotary, heads_view(turned),
          heads_view(packed[:, :h]), ints(positions).contiguous(), *self.norms)
        x = [step.normed(qkv[:, a:b], w, 1e-6).transpose(1, 0, 2) for (a, b), w in zip(((0, h), (h, h + kv)), self.weights)]
        want = [step.turned(t, positions, self.axis, self.frequencies, 1.0, False) for t in x]
        got = turned.cpu().numpy().transpose(1, 0, 2)
        assert (np.abs(got - want[0]) <= step.turned_bound(want[0], x[0], self.d // 2, 1.0, False)).all()
        written = [want[1].transpose(1, 0, 2), qkv[:, h + kv:].astype(np.float64)]
        bounds = [step.turned_bound(want[1], x[1], self.d // 2, 1.0, False).transpose(1, 0, 2), 0.0 * written[1]]
        at = 0
        for s, r in enumerate(rows):
            for t in (0, 1):
                new, n = written[t][at:at + r], self.done[s]
                content = self.content(s, t, n)
                if self.bits == 16:
                    assert (np.abs(content[n - r:] - new) <= bounds[t][at:at + r]).all()
                else:
                    assert np.array_equal(content[n - r:], step.value_of(*step.quantised(new)))
                assert np.array_equal(content[:n - r], self.held[s][t][:n - r]), "what was there before"
                self.held[s][t] = content
            at += r
        return turned

    def content(self, s, t, n):
        pages = self.table[s][:-(-n // self.page)]
        c = self.pools[t][ints(pages).long()].flatten(0, 1)[:n].cpu().numpy()
        if self.bits == 16:
            return c.astype(np.float64)
        return step.value_of(c, self.scales[t][ints(pages).long()].flatten(0, 1)[:n].cpu().numpy())

    def attend(self, turned, rows, trees=None):
        out = torch.full_like(turned, SENTINEL)
        scale, name = 1.0 / np.sqrt(self.d), "f16" if self.bits == 16 else "u8"
        args = (heads_view(out), heads_view(turned), self.cache, self.batch(rows))
        if trees is None:
            getattr(self.kern, "attention_paged_" + name)(*args, scale)
        else:
            getattr(self.kern, "attention_tree_" + name)(*args, DraftTree.of(trees), scale)
        q, got, at = turned.cpu().numpy(), out.cpu().numpy(), 0
        top = max(np.abs(self.held[s][1]).max(initial=0.0) for s in (0, 1))
        for s, r in enumerate(rows):
            n = self.done[s]
            seen = step.causal(r, n) if trees is None else step.with_past(step.ancestors(trees[s]), n)
            k, v = (t.transpose(1, 0, 2) for t in self.held[s])
            want = step.attention(q[at:at + r].transpose(1, 0, 2), k, v, scale, 1.0, seen).transpose(1, 0, 2)
            assert step.close_enough(got[at:at + r], want, top, n, self.bits == 8), (s, r, n)
            at += r


@pytest.mark.parametrize("bits", [16, 8])
def test_a_conversation_with_drafts(shared_keys, bits):  # noqa: F811
    """Prompts in pieces, tokens, then drafts that form trees, of which one branch is kept and written again behind the keys
    that are certain; each call's result by the definition over what the cache holds."""
    c = Conversation(shared_keys, bits)
    rng = c.rng

    def fresh(rows):
        return f16(rng, sum(rows), c.heads + 2 * c.kv, c.d)

    def places(rows):
        x = np.concatenate([n + np.arange(r) for n, r in zip(c.done, rows)])
        return np.stack([x, x // 3])
    for rows in ([50, 20], [1, 1], [0, 33], [17, 1]):
        at = places(rows)
        c.attend(c.append(fresh(rows), at, rows), rows)
    for rows in ([7, 12], [3, 0], [1, 21]):
        trees = [random_parents(r, rng) for r in rows]
        depths = [[] for _ in rows]
        for tree, depth in zip(trees, depths):
            for parent in tree:
                depth.append(depth[parent] + 1 if parent >= 0 else 0)
        x, certain = fresh(rows), list(c.done)
        at = np.concatenate([n + np.array(d, int) for n, d in zip(certain, depths)])
        at = np.stack([at, at // 3])
        c.attend(c.append(x, at, rows), rows, trees)
        # the branch of each draft's last token is kept
        kept, first = [], 0
        for tree, r in zip(trees, rows):
            j = r - 1
            branch = []
            while j >= 0:
                branch.append(first + j)
                j = tree[j]
            kept.append(branch[::-1])
            first += r
        c.done = certain
        c.held = [[t[:n] for t in pair] for pair, n in zip(c.held, certain)]
        again = [len(k) for k in kept]
        index = np.array(sum(kept, []), int)
        c.attend(c.append(x[index], at[:, index], again), again)
    rows = [1, 1]
    at = places(rows)
    c.attend(c.append(fresh(rows), at, rows), rows)


# ---- sizes and offsets ------------------------------------------------------------------------------------------

# (sequences of (rows, keys), heads, kv heads, d, page size)
LONG = [([(1, 40011)], 16, 2, 64, 16), ([(3, 70017), (1, 20001)], 8, 4, 128, 32), ([(300, 20011)], 8, 2, 128, 64), ([(1, 131073)], 4, 1, 128, 16)]


@pytest.mark.parametrize("case", LONG, ids=["%dx%d_h%d_%d_d%d" % (*c[0][0], *c[1:4]) for c in LONG])
def test_long_contexts_in_8_bits(shared_keys, request, case):  # noqa: F811
    """(The tree is a chain, which sees what the causal mask lets through.)"""
    seqs, heads, kv, d, page = case
    gen = torch.Generator(device="cuda").manual_seed(len(seqs) + d)
    data = [sequence(r, n, heads, kv, d, gen, "cuda") for r, n in seqs]
    scale, rows, lengths = data[0][3], [r for r, _ in seqs], [n for _, n in seqs]
    codes = [[quantised(x) for x in s[1:3]] for s in data]
    pages, table = ref.pages_of(lengths, page, np.random.default_rng(3))
    pools = torch.zeros(2, pages, page, kv, d, dtype=torch.uint8, device="cuda")
    scales = torch.full((2, pages, page, kv), torch.nan, dtype=torch.float16, device="cuda")
    for i, n in enumerate(lengths):
        at = ints(table[i, :-(-n // page)]).long()
        for t in (0, 1):
            for pool, x in ((pools[t], codes[i][t][0].permute(1, 0, 2)), (scales[t], codes[i][t][1].permute(1, 0))):
                whole = pool[at].flatten(0, 1)
                whole[:n] = x
                pool[at] = whole.view(-1, *pool.shape[1:])
    cache = PagedCacheU8(*(TensorView.of(t) for i in (0, 1) for t in (pools[i].permute(0, 2, 1, 3), scales[i].permute(0, 2, 1))))
    q = torch.cat([s[0] for s in data], 1).permute(1, 0, 2).contiguous()
    batch = PagedBatch(ints(ref.offsets(rows)), ints(lengths), ints(table), max(rows), max(lengths))
    outs = [torch.empty_like(q) for _ in range(2)]
    shared_keys.attention_paged_u8(heads_view(outs[0]), heads_view(q), cache, batch, scale)
    shared_keys.attention_tree_u8(heads_view(outs[1]), heads_view(q), cache, batch, DraftTree.of([list(range(-1, r - 1)) for r in rows]), scale)
    by_rows = request.node.callspec.params["shared_keys"] == FORMS[0]
    at = 0
    for s, (r, n), c in zip(data, seqs, codes):
        want = Codes(s[0], *c, scale)
        for out in outs:
            got = out[at:at + r].permute(1, 0, 2)
            assert want.agrees(got, row_steps(n)) if by_rows else want.matrix_agrees(got, matrix_steps(n)), (r, n)
        at += r


@pytest.fixture(scope="module")
def wide_pools():
    """Codes of 10 GiB and scales of 10 GiB, of which a few pages are used."""
    return torch.empty((5 << 31) + (1 << 16), dtype=torch.uint8, device="cuda"), torch.empty((5 << 30) + (1 << 12), dtype=torch.float16, device="cuda")


def test_offsets_beyond_32_bits(shared_keys, wide_pools):  # noqa: F811
    """Pages whose offsets pass 2^31, 2^32 and 2^33 elements, written, read back and attended to."""
    kv, page, d, heads, n = 2, 16, 64, 4, 91
    rng = np.random.default_rng(12)
    views = []
    for i in range(2):
        views.append(TensorView(wide_pools[0], TensorLayout((6, kv, page, d), (1 << 31, page * d, d, 1)), i * kv * page * d))
        views.append(TensorView(wide_pools[1], TensorLayout((6, kv, page), (1 << 30, page, 1)), i * kv * page))
    cache, table = PagedCacheU8(*views), np.array([[5, 0, 3, 4, 2, 1]], np.int32)
    k, v, q = f16(rng, n, kv, d), f16(rng, n, kv, d), f16(rng, 20, heads, d)
    whole = PagedBatch(ints([0, n]), ints([n]), ints(table))
    shared_keys.append_u8(cache, whole, heads_view(dev(k)), heads_view(dev(v)))
    back = [torch.zeros(n, kv, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    shared_keys.read_u8(*(heads_view(t) for t in back), cache, whole)
    held = [step.value_of(*step.quantised(t.astype(np.float64))) for t in (k, v)]
    for t, want in zip(back, held):
        assert (np.abs(t.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
    out = [torch.zeros(20, heads, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    batch = PagedBatch(ints([0, 20]), ints([n]), ints(table))
    tree = random_parents(20, rng)
    shared_keys.attention_paged_u8(heads_view(out[0]), heads_view(dev(q)), cache, batch, 0.125)
    shared_keys.attention_tree_u8(heads_view(out[1]), heads_view(dev(q)), cache, batch, DraftTree.of([tree]), 0.125)
    keys, values = (t.transpose(1, 0, 2) for t in held)
    for got, seen in zip(out, (step.causal(20, n), step.with_past(step.ancestors(tree), n))):
        want = step.attention(q.transpose(1, 0, 2), keys, values, 0.125, 1.0, seen).transpose(1, 0, 2)
        assert step.close_enough(got.cpu().numpy(), want, np.abs(values).max(), n, True)


DRAWN = range(16)


@pytest.mark.parametrize("seed", DRAWN)
def test_drawn_batches(shared_keys, seed):  # noqa: F811
    """Sizes drawn over their range: causal, unmasked, and drafts in both widths."""
    rng = np.random.default_rng(1000 + seed)

    def size(low, high):
        return int(round(np.exp(rng.uniform(np.log(low), np.log(high)))))
    d, page, kv = int(rng.choice([16, 48, 64, 80, 96, 112, 128])), int(rng.choice([16, 32, 64, 128])), size(1, 6)
    heads = kv * size(1, 8)
    seqs = [(size(1, 40) - 1, size(1, 900) - 1) for _ in range(size(1, 12))] + [(size(1, 300), size(1, 900))]
    p = Paged(seqs, heads, kv, d, page, seed=seed, order="tokens" if seed % 2 else "heads")
    scale = 1.0 / np.sqrt(d)
    for mask in (CAUSAL, NONE):
        p.out_t.fill_(SENTINEL)
        shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, scale, 0.9, mask)
        p.check(scale, mask, 0.9)
    rows = [size(1, 60) - 1 for _ in range(size(1, 8))] + [size(1, 80)]
    past = [size(1, 700) - 1 for _ in rows]
    trees = [random_parents(r, rng) for r in rows]
    for bits in (16, 8):
        t = Drafts(trees, past, heads, kv, d, page, bits, seed=seed)
        t.check(t.run(shared_keys, scale), t.want(scale))


def test_many_sequences(shared_keys):  # noqa: F811
    rng = np.random.default_rng(10)
    seqs = [(int(rng.integers(0, 3)), int(rng.integers(0, 60))) for _ in range(700)]
    p = Paged(seqs, 4, 2, 64, 16, seed=11)
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125)
    p.check(0.125, CAUSAL)
    for bits in (16, 8):
        t = Drafts([random_parents(r, rng) for r, _ in seqs], [n for _, n in seqs], 4, 2, 64, 16, bits, seed=12)
        t.check(t.run(shared_keys, 0.125), t.want(0.125))


def test_more_sequences_than_a_launch_has_workgroups():
    """Sequences of one row and one key: each row's result is its value, to one rounding."""
    n, heads, d = 280000, 32, 16
    gen = torch.Generator(device="cuda").manual_seed(5)
    kern = GpuKernels()
    q = torch.randn(n, heads, d, dtype=torch.float16, device="cuda", generator=gen)
    codes = torch.randint(0, 256, (2, 1, heads, 16, d), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.rand(2, 1, heads, 16, device="cuda", generator=gen).half() + 0.5
    views = [TensorView.of(t) for i in (0, 1) for t in (codes[i], scales[i])]
    at, out = torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.zeros_like(q)
    batch = PagedBatch(at, torch.ones(n, dtype=torch.int32, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda"))
    want = (codes[1, 0, :, 0].double() - 127.5) * scales[1, 0, :, 0].double()[:, None]
    tree = DraftTree(torch.ones(n, 1, dtype=torch.int32, device="cuda"))
    for call in (lambda: kern.attention_paged_u8(heads_view(out), heads_view(q), PagedCacheU8(*views), batch, 0.3),
                 lambda: kern.attention_tree_u8(heads_view(out), heads_view(q), PagedCacheU8(*views), batch, tree, 0.3)):
        out.zero_()
        call()
        # (the probability is 1; its product with the scale is exact; 255 times it, less 127.5 times it, in 32 bits)
        assert ((out.double() - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -25 + 3 * 255 * 1.5 * 2.0 ** -24).all()


# ---- hints, lengths and offsets that do not fit -------------------------------------------------------------------

def test_hints_never_change_what_is_computed(shared_keys):  # noqa: F811
    p = Paged([(1, 700), (20, 300), (1, 3), (150, 400)], 8, 2, 128, 16, seed=9)
    t = Drafts([random_parents(r, np.random.default_rng(1)) for r in (1, 20, 70)], [700, 100, 3], 8, 2, 128, 16, 8)
    scale, batch = 1.0 / np.sqrt(128), t.batch
    want = t.want(scale)
    for rows, longest in ((0, 0), (1, 1), (1, 700), (150, 700), (2 ** 30, 2 ** 30), (-1, -1)):
        p.out_t.fill_(SENTINEL)
        b = PagedBatch(p.batch.row_offsets, p.batch.lengths, p.batch.table, rows, longest)
        shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, b, scale)
        p.check(scale, CAUSAL)
        t.batch = PagedBatch(batch.row_offsets, batch.lengths, batch.table, rows, longest)
        t.out_t.fill_(SENTINEL)
        t.check(t.run(shared_keys, scale), want)


def test_lengths_out_of_range_are_clamped(shared_keys):  # noqa: F811
    """A length beyond the table is the table's, and a negative one none, for writing and reading too."""
    p = Paged([(2, 30), (1, 17)], 2, 2, 64, 16, seed=8)
    c = p.cache
    width = c.table.shape[1]
    table = c.table.copy()
    table[table < 0] = 0          # (every entry a page of the cache: sequence 0 uses them all)
    c.scales = np.where(np.isfinite(c.scales), c.scales, np.float16(0.01))
    c.upload()
    batch = PagedBatch(ints(p.row_offsets), ints([1 << 30, -5]), ints(table))
    for call in (lambda: shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), c.handle, batch, 0.125, 1.0, NONE),
                 lambda: shared_keys.attention_tree_u8(heads_view(p.out_t), heads_view(p.q_t), c.handle, batch,
                                                       DraftTree(torch.full((p.rows, 1), -1, dtype=torch.int32, device="cuda")), 0.125)):
        p.out_t.fill_(SENTINEL)
        call()
        got, n = p.out_t.cpu().numpy(), width * 16
        keys, values = (step.value_of(ref.gathered(c.codes[t], table[0], n), ref.gathered(c.scales[t][..., None], table[0], n)[..., 0]) for t in (0, 1))
        want = step.attention(p.q[:2].transpose(1, 0, 2), keys, values, 0.125, 1.0, np.ones((2, n), bool)).transpose(1, 0, 2)
        assert step.close_enough(got[:2], want, np.abs(values).max(), n, True)
        assert (got[2] == 0).all() and (got[3:] == SENTINEL).all()
    before = [x.storage.clone() for x in (c.handle.key, c.handle.key_scale)]
    far = PagedBatch(ints(p.row_offsets), ints([2 ** 31 - 1, -2 ** 31]), ints(table))
    kv = dev(f16(np.random.default_rng(2), p.rows, 2, 64))
    shared_keys.append_u8(c.handle, far, heads_view(kv), heads_view(kv))       # (places beyond the table and in front of the first)
    assert torch.equal(before[0], c.handle.key.storage) and torch.equal(before[1], c.handle.key_scale.storage)
    out = torch.full((2, p.rows, 2, 64), SENTINEL, dtype=torch.float16, device="cuda")
    shared_keys.read_u8(heads_view(out[0]), heads_view(out[1]), c.handle, far)
    n = int(p.row_offsets[-1])
    assert out[:, :n].isnan().all() and (out[:, n:] == SENTINEL).all()


def test_offsets_that_decrease(shared_keys):  # noqa: F811
    """Rows that only one sequence claims are right; the others hold some result, and nothing else is written."""
    p = Paged([(10, 300), (0, 40), (10, 500)], 4, 2, 64, 16, seed=65)
    want = p.want(0.125, CAUSAL)
    batch = PagedBatch(ints([0, 10, 5, 20]), p.batch.lengths, p.batch.table)
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, batch, 0.125)
    got = p.out_t.cpu().numpy()
    behind = ref.attention(p.q[5:20].transpose(1, 0, 2), *p.cache.values(2, 500), 0.125).transpose(1, 0, 2)
    top = 127.5 * np.nanmax(p.cache.scales[1].astype(np.float64))
    assert step.close_enough(got[:5], want[:5], top, 300, True) and step.close_enough(got[10:20], behind[5:], top, 500, True)
    assert np.isfinite(got[5:10]).all() and (got[20:] == SENTINEL).all()


# ---- graphs, streams, memory --------------------------------------------------------------------------------------

def calls(kern, seed):
    """Attention over codes and of drafts in both widths, each with shared keys and with what it has to give."""
    rng = np.random.default_rng(seed)
    p = Paged([(1, 3000), (1, 70), (90, 800)], 4, 2, 64, 16, seed=seed)
    drafts = [Drafts([random_parents(r, rng) for r in (9, 40)], [1500, 64], 4, 2, 128, 16, bits, seed=seed) for bits in (16, 8)]

    def run():
        kern.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125)
        for t in drafts:
            f = kern.attention_tree_f16 if t.bits == 16 else kern.attention_tree_u8
            f(heads_view(t.out_t), heads_view(t.q_t), t.cache, t.batch, t.tree, 0.1)

    def check():
        p.check(0.125, CAUSAL)
        for t in drafts:
            t.check(t.out_t.cpu().numpy(), t.want(0.1))

    def clear():
        for x in (p, *drafts):
            x.out_t[:int((x.row_offsets if x is p else x.starts)[-1])] = 0
    return run, check, clear


def test_two_graphs_share_a_workspace():
    """Two captured runs with one instance's buffer, replayed by turns on a stream, beside eager ones."""
    kern = GpuKernels(workspace_bytes=64 << 20)
    both = [calls(kern, 63), calls(kern, 64)]
    graphs = []
    for run, _, _ in both:
        run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run()
    for i in range(3):
        for (run, check, clear), g in zip(both, graphs):
            clear()
            g.replay()
            both[1 - i % 2][0]()
        torch.cuda.synchronize()
        for _, check, _ in both:
            check()


def test_two_streams_at_once(shared_keys):  # noqa: F811
    """Calls that run beside each other on two streams, each with its own part of the library's pool."""
    if shared_keys._workspace is not None:
        pytest.skip("an instance with a workspace serves one stream")
    both, streams = [calls(shared_keys, 61), calls(shared_keys, 62)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for (run, _, _), s in zip(both, streams):
            with torch.cuda.stream(s):
                run()
    torch.cuda.synchronize()
    for _, check, _ in both:
        check()


def test_a_captured_draft_serves_later_ones():
    """One graph of filling, reading back and a tree's attention, replayed while lengths, trees and values change under it."""
    kern, rng = GpuKernels(workspace_bytes=64 << 20), np.random.default_rng(50)
    heads, kv, d, page, rows = 8, 2, 128, 16, [5, 3]
    c = Paged([(5, 1100), (3, 90)], heads, kv, d, page, seed=51, spare=0)
    lengths = ints([900, 7])
    batch = PagedBatch(ints(ref.offsets(rows)), lengths, ints(c.cache.table), 5, 1100)
    qkv = torch.zeros(8, heads + 2 * kv, d, dtype=torch.float16, device="cuda")
    bits, positions = torch.zeros(8, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    rotary, norm = RotaryAxes.new(d, [40, 24]), HeadNorm(dev(f16(rng, d)), 1e-6)
    turned, out, read = (torch.zeros(8, n, d, dtype=torch.float16, device="cuda") for n in (heads, heads, 2 * kv))
    tree = DraftTree(bits)

    def work():
        kern.append_u8(c.cache.handle, batch, heads_view(qkv[:, heads:heads + kv]), heads_view(qkv[:, heads + kv:]), rotary, heads_view(turned),
                       heads_view(qkv[:, :heads]), positions, norm, norm)
        kern.read_u8(heads_view(read[:, :kv]), heads_view(read[:, kv:]), c.cache.handle, batch)
        kern.attention_tree_u8(heads_view(out), heads_view(turned), c.cache.handle, batch, tree, 0.1)
    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    h = c.cache.handle
    state = [v.storage for v in (h.key, h.key_scale, h.value, h.value_scale)]
    for i in range(5):
        lengths += 1
        qkv.copy_(dev(f16(rng, *qkv.shape)))
        bits.copy_(DraftTree.of([random_parents(r, rng) for r in rows]).bits)
        positions.copy_(ints(rng.integers(0, 2000, (2, 8))))
        before = [t.clone() for t in state]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (turned, out, read, *state)]
        for t, b in zip(state, before):
            t.copy_(b)
        for t in (turned, out, read):
            t.zero_()
        work()
        for a, b in zip(got, (turned, out, read, *state)):
            assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)
        assert out.isfinite().all() and out.abs().max() > 0


@pytest.mark.parametrize("seqs", [[(1, 3000), (1, 70)], [(60, 3000)], [(300, 1900), (1, 1700)]])
def test_workspace_bytes(seqs):
    """What is reported is what is used: the same bits with it as through the pool; with less, or none, still right."""
    kern, lib = GpuKernels(), _ffi.lib()
    p = Paged(seqs, 8, 2, 128, 16, seed=66)
    batch = PagedBatch(p.batch.row_offsets, p.batch.lengths, p.batch.table, max(r for r, _ in seqs), 3000)
    nbytes = attention_paged_u8_workspace_bytes(p.cache.handle, batch, 8, p.rows)
    assert nbytes > 0
    tree = DraftTree(torch.ones(p.rows, 10, dtype=torch.int32, device="cuda"))

    def run(k):
        outs = []
        for f, arg in ((k.attention_paged_u8, ()), (k.attention_tree_u8, (tree,))):
            p.out_t.fill_(SENTINEL)
            f(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, batch, *arg, 0.1)
            if not arg:
                p.check(0.1, CAUSAL)
            outs.append(p.out_t.clone())
        return outs
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES)
    pool = run(kern)
    lib.adr_set_held_workspace_limit(0)
    for got, want in zip(run(GpuKernels(workspace_bytes=nbytes)), pool):
        assert torch.equal(got, want)
    for part in (nbytes // 2, nbytes // 7, 64):
        run(GpuKernels(workspace_bytes=part))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows,past", [([8], [5000]), ([61], [2100]), ([100, 3], [3000, 40])])
def test_workspaces_of_trees(rows, past, bits):
    """As above: the same bits with what is reported as through the pool; with less still right."""
    lib, rng = _ffi.lib(), np.random.default_rng(4)
    t = Drafts([random_parents(r, rng) for r in rows], past, 8, 2, 128, 16, bits, seed=67)
    want, nbytes = t.want(0.1), attention_tree_workspace_bytes(t.cache, t.batch, 8, t.rows)
    assert nbytes > 0
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES)
    pool = t.run(GpuKernels(), 0.1).copy()
    lib.adr_set_held_workspace_limit(0)
    t.check(pool, want)
    assert np.array_equal(t.run(GpuKernels(workspace_bytes=nbytes), 0.1), pool)
    for part in (nbytes // 2, nbytes // 7, 64):
        t.check(t.run(GpuKernels(workspace_bytes=part), 0.1), want)


def test_calls_allocate_nothing():
    kern = GpuKernels(workspace_bytes=64 << 20)
    run, _, _ = calls(kern, 70)
    p = Paged([(3, 40)], 4, 2, 64, 16, spare=0)
    x = torch.zeros(4, 3, 4, 64, dtype=torch.float16, device="cuda")
    q, turned, key, value = (heads_view(t[:, :n]) for t, n in zip(x, (4, 4, 2, 2)))
    rotary, norm = RotaryAxes.new(64, [16, 16]), HeadNorm(x.new_ones(64))
    half = PagedCache(*(TensorView.of(torch.zeros(8, 2, 16, 64, dtype=torch.float16, device="cuda")) for _ in range(2)))

    def work():
        run()
        kern.norm_rotary_f16(turned, q, positions, rotary, norm)
        kern.append_norm_f16(half, p.batch, key, value, rotary, turned, q, None, norm, norm)
        kern.append_u8(p.cache.handle, p.batch, key, value, rotary, turned, q, None, norm, norm)
        kern.read_u8(key, value, p.cache.handle, p.batch)
    positions = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    work()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    work()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before

"""Rotary positions, the paged cache and attention over it and over packed prompts, on the GPU, against plain 64-bit
definitions (sequences_reference.py, which also derives the tolerance)."""
import numpy as np
import pytest
import torch

from adrastea_amd import (AdrasteaError, attention_packed_workspace_bytes, attention_paged_workspace_bytes, GpuKernels, MatmulMask, MatmulTracer, PackedBatch, PagedBatch, PagedCache, Rotary,
                          RotaryLayout, RotaryScaling, TensorLayout, TensorView, _ffi, rotary_frequencies)
import sequences_reference as ref

pytestmark = pytest.mark.gpu

CAUSAL, NONE = MatmulMask.CAUSAL, MatmulMask.NONE
SENTINEL = 777.0  # in output rows that belong to no sequence


@pytest.fixture(scope="module")
def kern():
    return GpuKernels()


FORMS = ["a row to a wavefront", "few rows, 2 waves", "few rows, 4 waves", "few rows, shared", "many rows", "many rows, 2 groups",
         "many rows, shared", "many rows, 2 groups, shared"]   # by value of adr_debug_knob(2, 1 + i)


@pytest.fixture(params=["unshared", "pool", "workspace", *FORMS])
def shared_keys(request):
    """Kernels whose keys are not shared over workgroups, shared through the library's pool, or through their own buffer;
    and each form of the kernels by itself, whatever the sizes are."""
    lib = _ffi.lib()
    forced = FORMS.index(request.param) + 1 if request.param in FORMS else 0
    assert lib.adr_debug_knob(2, forced) == 0
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES if request.param == "pool" or forced else 0)
    yield GpuKernels(workspace_bytes=(96 << 20) if request.param == "workspace" else 0)
    lib.adr_set_held_workspace_limit(0)
    lib.adr_debug_knob(2, 0)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


def f16(rng, *shape, std=1.0):
    return (rng.standard_normal(shape) * std).astype(np.float16)


def heads_view(t):
    """[heads, rows, d] view of a [rows, heads, d] tensor."""
    return TensorView.of(t.permute(1, 0, 2))


class Paged:
    """Sequences of (rows, keys) over pages; everything that no row may read is NaN."""

    def __init__(self, seqs, heads, kv, d, page, seed=0, order="tokens", spare=3, std=1.0):
        rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.kv, self.d, self.page = seqs, heads, kv, d, page
        self.rows = sum(r for r, _ in seqs) + spare
        self.row_offsets = ref.offsets([r for r, _ in seqs])
        lengths = [n for _, n in seqs]
        pages, self.table = ref.pages_of(lengths, page, rng)
        self.q = f16(rng, self.rows, heads, d, std=std)
        self.q[self.row_offsets[-1]:] = np.nan
        pool = np.full((2, pages, kv, page, d), np.nan, np.float16)
        for i, n in enumerate(lengths):
            for x0 in range(0, n, page):
                m = min(page, n - x0)
                pool[:, self.table[i, x0 // page], :, :m] = f16(rng, 2, kv, m, d)
        self.k, self.v = pool
        self.lengths = lengths
        if order == "tokens":
            self.k_t, self.v_t = (dev(t.transpose(0, 2, 1, 3)).permute(0, 2, 1, 3) for t in (self.k, self.v))
        else:
            self.k_t, self.v_t = dev(self.k), dev(self.v)
        self.q_t = dev(self.q)
        self.out_t = torch.full((self.rows, heads, d), SENTINEL, dtype=torch.float16, device="cuda")
        self.cache = PagedCache(TensorView.of(self.k_t), TensorView.of(self.v_t))
        self.batch = PagedBatch(ints(self.row_offsets), ints(lengths), ints(self.table))

    def want(self, scale, mask, temp=1.0):
        out = np.full((self.rows, self.heads, self.d), SENTINEL)
        for i, (r, n) in enumerate(self.seqs):
            a = self.row_offsets[i]
            k, v = (ref.gathered(t, self.table[i], n) for t in (self.k, self.v))
            out[a:a + r] = ref.attention(self.q[a:a + r].transpose(1, 0, 2), k, v, scale, temp,
                                         mask == CAUSAL).transpose(1, 0, 2)
        return out

    def check(self, scale, mask, temp=1.0):
        want, got = self.want(scale, mask, temp), self.out_t.cpu().numpy()
        n = self.row_offsets[-1]
        assert np.array_equal(got[n:], want[n:].astype(np.float16)), "rows behind the last sequence"
        top = np.nanmax(np.abs(self.v.astype(np.float64)), initial=0.0)
        assert ref.close_enough(got[:n], want[:n], top, max([n for _, n in self.seqs] + [1]))


# (sequences of (rows, keys), heads, kv heads, d, page size): lengths of zero and one, rows without keys, ends inside
# a page and inside a tile, groups that are no power of two, head dimensions beside 64 and 128
PAGED = [
    ([(1, 1)], 1, 1, 64, 16), ([(1, 37)], 4, 4, 128, 16), ([(1, 300), (1, 1), (0, 0), (1, 64), (1, 65), (0, 9)], 8, 2, 128, 16),
    ([(5, 5), (3, 130), (0, 20), (2, 2)], 6, 2, 64, 32), ([(4, 2), (3, 0), (1, 0)], 4, 4, 64, 16),
    ([(70, 200), (1, 513), (129, 129)], 4, 1, 128, 64), ([(33, 140)], 5, 1, 128, 16), ([(17, 17), (16, 600)], 7, 7, 64, 128),
    ([(2, 75), (40, 41)], 3, 1, 40, 16), ([(3, 90)], 2, 2, 8, 32), ([(9, 100), (1, 260)], 4, 2, 72, 16),
    ([(3, 50)], 2, 1, 7, 4), ([(3, 70), (1, 5)], 2, 2, 160, 16), ([(2, 40)], 2, 1, 256, 16), ([(3, 21), (1, 64)], 4, 2, 64, 1),
    ([(3, 50), (1, 49)], 4, 2, 128, 5), ([(2, 100), (65, 300)], 4, 4, 64, 48),
]
IDS = ["%s_h%d_%d_d%d_p%d" % ("-".join("%dx%d" % s for s in c[0]), *c[1:]) for c in PAGED]


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("case", PAGED, ids=IDS)
def test_paged_attention(shared_keys, case, mask):
    p = Paged(*case, seed=len(case[0]) * 100 + case[3], order="heads" if case[4] == 64 else "tokens")
    scale = 1.0 / np.sqrt(p.d)
    shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, scale, 1.0, mask)
    p.check(scale, mask)


class Packed:
    def __init__(self, seqs, heads, kv, d, seed=0, spare=2):
        rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.kv, self.d = seqs, heads, kv, d
        self.row_offsets, self.key_offsets = (ref.offsets([s[i] for s in seqs]) for i in (0, 1))
        self.rows, self.keys = self.row_offsets[-1] + spare, self.key_offsets[-1] + 1
        self.q, self.k, self.v = f16(rng, self.rows, heads, d), f16(rng, self.keys, kv, d), f16(rng, self.keys, kv, d)
        self.q[self.row_offsets[-1]:] = np.nan
        self.k[-1], self.v[-1] = np.nan, np.nan
        self.q_t, self.k_t, self.v_t = dev(self.q), dev(self.k), dev(self.v)
        self.out_t = torch.full((int(self.rows), heads, d), SENTINEL, dtype=torch.float16, device="cuda")
        self.batch = PackedBatch(ints(self.row_offsets), ints(self.key_offsets))

    def want(self, scale, mask, temp=1.0):
        out = np.full((self.rows, self.heads, self.d), SENTINEL)
        for i, (r, n) in enumerate(self.seqs):
            a, b = self.row_offsets[i], self.key_offsets[i]
            out[a:a + r] = ref.attention(self.q[a:a + r].transpose(1, 0, 2), self.k[b:b + n].transpose(1, 0, 2),
                                         self.v[b:b + n].transpose(1, 0, 2), scale, temp, mask == CAUSAL).transpose(1, 0, 2)
        return out

    def check(self, scale, mask, temp=1.0):
        want, got = self.want(scale, mask, temp), self.out_t.cpu().numpy()
        n = self.row_offsets[-1]
        assert np.array_equal(got[n:], want[n:].astype(np.float16)), "rows behind the last sequence"
        top = np.nanmax(np.abs(self.v[:-1].astype(np.float64)), initial=0.0)
        assert ref.close_enough(got[:n], want[:n], top, max(n for _, n in self.seqs))


PACKED = [
    ([(1, 1)], 1, 1, 64), ([(5, 5), (1, 1), (0, 0), (130, 130), (64, 64)], 4, 2, 128), ([(77, 77), (12, 12), (33, 33)], 3, 3, 64),
    ([(1, 200), (40, 90), (200, 200)], 6, 2, 64), ([(10, 3), (7, 0), (4, 40)], 4, 4, 128), ([(300, 300)], 2, 1, 128),
    ([(20, 20), (3, 50)], 2, 1, 24), ([(9, 9)], 2, 2, 100), ([(70, 131)], 2, 1, 120), ([(5, 9)], 1, 1, 200), ([(4, 4)], 2, 2, 3),
    ([(16, 16), (15, 17), (1, 640)], 16, 1, 128),
]


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("case", PACKED, ids=["%s_h%d_%d_d%d" % ("-".join("%dx%d" % s for s in c[0]), *c[1:]) for c in PACKED])
def test_packed_attention(shared_keys, case, mask):
    p = Packed(*case, seed=case[3])
    scale = 1.0 / np.sqrt(p.d)
    shared_keys.attention_packed_f16(heads_view(p.out_t), heads_view(p.q_t), heads_view(p.k_t), heads_view(p.v_t), p.batch,
                                     scale, 1.3, mask)
    p.check(scale, mask, 1.3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,keys", [(2, 9), (7, 200), (40, 40), (200, 330)])
def test_what_a_row_does_not_see_never_reaches_it(shared_keys, rows, keys, d):
    """The last key's value holds infinities, the one before's key NaN: only rows that see them change."""
    p = Packed([(rows, keys), (3, 3)], 4, 2, d, seed=rows)
    p.v[keys - 1, :, ::3], p.v[keys - 1, :, 1::3] = np.inf, -np.inf
    p.v_t = dev(p.v)
    scale = 1.0 / np.sqrt(d)

    def run():
        shared_keys.attention_packed_f16(heads_view(p.out_t), heads_view(p.q_t), heads_view(p.k_t), heads_view(p.v_t),
                                         p.batch, scale)
        want, got = p.want(scale, CAUSAL), p.out_t.cpu().numpy()
        seen = np.ones(p.row_offsets[-1], bool)
        seen[rows - 1] = False
        top = np.abs(p.v[:keys - 1].astype(np.float64)).max()
        assert ref.close_enough(got[:p.row_offsets[-1]][seen], want[:p.row_offsets[-1]][seen], top, keys)
        return got
    got = run()
    assert np.isposinf(got[rows - 1, :, ::3]).all() and np.isneginf(got[rows - 1, :, 1::3]).all()
    p.v[keys - 1], p.k[keys - 1] = 1.0, np.nan
    p.v_t, p.k_t = dev(p.v), dev(p.k)
    assert np.isnan(run()[rows - 1]).all()


def test_pages_outside_the_cache_are_nan_and_never_read(shared_keys):
    p = Paged([(1, 40), (3, 40), (1, 100), (1, 20)], 4, 2, 64, 16, seed=5)
    for bad in (-1, 1 << 20, p.k.shape[0], -2 ** 31):
        table = p.table.copy()
        table[1, 2] = bad         # keys 32 .. 39 of sequence 1, which all of its rows see
        table[2, 7:] = bad        # behind the last key
        p.batch = PagedBatch(ints(p.row_offsets), ints(p.lengths), ints(table))
        shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.125)
        got = p.out_t.cpu().numpy()
        assert np.isnan(got[1:4]).all()
        want = p.want(0.125, CAUSAL)
        for row in (0, 4, 5):
            assert ref.close_enough(got[row], want[row], np.nanmax(np.abs(p.v)), 100)
    # only the rows that see the page
    q = Paged([(30, 40)], 4, 2, 64, 16, seed=6)
    table = q.table.copy()
    table[0, 2] = -7              # keys 32 .. 39: rows 22 .. 29
    batch = PagedBatch(ints(q.row_offsets), ints(q.lengths), ints(table))
    shared_keys.attention_paged_f16(heads_view(q.out_t), heads_view(q.q_t), q.cache, batch, 0.125)
    got = q.out_t.cpu().numpy()
    assert np.isnan(got[22:30]).all()
    assert ref.close_enough(got[:22], q.want(0.125, CAUSAL)[:22], np.nanmax(np.abs(q.v)), 40)


def test_lengths_and_offsets_out_of_range_are_clamped(kern):
    p = Paged([(2, 30), (1, 17)], 2, 2, 64, 16, seed=8)
    width = p.table.shape[1]
    table = p.table.copy()
    table[table < 0] = 0          # (every entry a page of the cache: sequence 0 uses them all)
    k = np.nan_to_num(p.k, nan=0.5)
    v = np.nan_to_num(p.v, nan=0.25)
    cache = PagedCache(TensorView.of(dev(k)), TensorView.of(dev(v)))
    batch = PagedBatch(ints(p.row_offsets), ints([1 << 30, -5]), ints(table))
    kern.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), cache, batch, 0.125, 1.0, NONE)
    got = p.out_t.cpu().numpy()
    keys, values = (ref.gathered(t, table[0], width * 16) for t in (k, v))
    want = ref.attention(p.q[:2].transpose(1, 0, 2), keys, values, 0.125, causal=False).transpose(1, 0, 2)
    assert ref.close_enough(got[:2], want, np.abs(v).max(), width * 16)
    assert (got[2] == 0).all()    # no keys
    p.out_t.fill_(SENTINEL)
    batch = PagedBatch(ints([-3, 1, 1 << 30]), ints([30, 17]), ints(p.table))  # rows 0; 1 .. the last
    p.q_t.nan_to_num_(nan=1.0)
    kern.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, batch, 0.125, 1.0, NONE)
    got = p.out_t.cpu().numpy()
    q = p.q_t.cpu().numpy()
    for rows, i in ((slice(0, 1), 0), (slice(1, p.rows), 1)):
        keys, values = (ref.gathered(t, p.table[i], p.lengths[i]) for t in (p.k, p.v))
        want = ref.attention(q[rows].transpose(1, 0, 2), keys, values, 0.125, causal=False).transpose(1, 0, 2)
        assert ref.close_enough(got[rows], want, np.nanmax(np.abs(p.v)), 30)


@pytest.mark.parametrize("layout", ["fused", "heads_first", "x2", "odd_rows", "unaligned", "backwards", "close_rows"])
def test_strides_and_alignment(shared_keys, layout):
    rng = np.random.default_rng(3)
    seqs, heads, kv, d = [(40, 40), (1, 90), (25, 60)], 4, 2, 64
    p = Packed(seqs, heads, kv, d, seed=4)
    scale = 1.0 / np.sqrt(d)

    def place(a):
        """`a` [rows, heads, d] in a larger buffer at other strides; (tensor, view)."""
        rows, h, _ = a.shape
        if layout == "heads_first":
            t = dev(a.transpose(1, 0, 2))
            return t, TensorView.of(t), lambda: t.cpu().numpy().transpose(1, 0, 2)
        x, y, z, offset, size = {
            "fused": (1, (h + 3) * d, d, 2 * d, (rows + 1) * (h + 3) * d), "x2": (2, 2 * h * d, 2 * d, 0, 2 * rows * h * d),
            "odd_rows": (1, h * d + 3, d, 0, rows * (h * d + 3)), "unaligned": (1, h * d, d, 1, rows * h * d + 8),
            "backwards": (1, -h * d, d, (rows - 1) * h * d, rows * h * d),
            "close_rows": (1, h * d, d, 0, rows * h * d)}[layout]
        flat = np.full(size, np.nan, np.float16)
        r, hh, xx = np.ogrid[:rows, :h, :d]
        at = offset + r * y + hh * z + xx * x
        flat[at] = a
        t = dev(flat)
        return t, TensorView(t, TensorLayout((h, rows, d), (z, y, x)), offset), lambda: t.cpu().numpy()[at]
    if layout == "close_rows":  # keys that overlap: every key starts 8 values behind the one before
        flat = f16(rng, (p.keys - 1) * 8 + kv * d)
        r, hh, xx = np.ogrid[:p.keys, :kv, :d]
        p.k = flat[r * 8 + hh * d + xx]
        t = dev(flat)
        k_view = TensorView(t, TensorLayout((kv, int(p.keys), d), (d, 8, 1)))
        keep = t
    else:
        keep, k_view, _ = place(p.k)
    placed = [place(a) for a in (p.q, p.v, np.full(p.q.shape, SENTINEL, np.float16))]
    shared_keys.attention_packed_f16(placed[2][1], placed[0][1], k_view, placed[1][1], p.batch, scale)
    p.out_t = torch.from_numpy(placed[2][2]().copy())
    p.check(scale, CAUSAL)


def test_hints_never_change_what_is_computed(shared_keys):
    p = Paged([(1, 700), (20, 300), (1, 3), (150, 400)], 8, 2, 128, 16, seed=9)
    scale = 1.0 / np.sqrt(128)
    for rows, longest in ((0, 0), (1, 1), (1, 700), (150, 700), (2 ** 30, 2 ** 30), (-1, -1)):
        p.out_t.fill_(SENTINEL)
        b = PagedBatch(p.batch.row_offsets, p.batch.lengths, p.batch.table, rows, longest)
        shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, b, scale)
        p.check(scale, CAUSAL)


@pytest.mark.parametrize("value", [-1, 9, 1 << 30])
def test_unknown_forms_force_nothing(kern, value):
    lib = _ffi.lib()
    p = Paged([(1, 700), (70, 300)], 8, 2, 128, 16, seed=13)
    try:
        assert lib.adr_debug_knob(2, value) == 0
        kern.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.1)
    finally:
        lib.adr_debug_knob(2, 0)
    p.check(0.1, CAUSAL)


def test_many_sequences(shared_keys):
    rng = np.random.default_rng(10)
    seqs = [(int(rng.integers(0, 3)), int(rng.integers(0, 60))) for _ in range(700)]
    p = Paged(seqs, 4, 2, 64, 16, seed=11)
    shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.125)
    p.check(0.125, CAUSAL)


def wide_attention(q, k, v, scale, causal=True):
    """The definition in 64 bits on the GPU, for sizes that the one in numpy takes too long for: q [heads, r, d]."""
    heads, r, d = q.shape
    kv, n, _ = k.shape
    out = torch.empty(heads, r, d, dtype=torch.float64, device="cuda")
    hidden = (torch.arange(n, device="cuda")[None, :] > torch.arange(n - r, n, device="cuda")[:, None]) if causal else None
    for h in range(heads):
        s = (q[h].double() @ k[h // (heads // kv)].double().t().contiguous()) * scale
        if causal:
            s.masked_fill_(hidden, -float("inf"))
        out[h] = torch.softmax(s, -1) @ v[h // (heads // kv)].double()
    return out


# more rows and keys than one workgroup's: blocks that are divided several times, one sequence among many, a batch of tokens
LARGE = [([(700, 2900)], 8, 2, 128, 16), ([(300, 5100)], 8, 1, 64, 64), ([(500, 1800), *[(1, 37 * i + 1) for i in range(40)]], 8, 4, 64, 32),
         ([(1, 150 * i) for i in range(1, 60)], 4, 4, 128, 16), ([(4, 9000), (3, 20), (4, 4000)], 4, 2, 128, 16),
         ([(130, 1000)] * 5, 6, 2, 128, 128), ([(1, 40000)], 16, 2, 64, 16)]


@pytest.mark.parametrize("case", LARGE, ids=["%dx_%dx%d_h%d_%d_d%d" % (len(c[0]), *c[0][0], *c[1:4]) for c in LARGE])
def test_large_batches(shared_keys, case):
    seqs, heads, kv, d, page = case
    gen = torch.Generator(device="cuda").manual_seed(70)
    rows, longest = sum(r for r, _ in seqs), max(n for _, n in seqs)
    pages, table = ref.pages_of([n for _, n in seqs], page, np.random.default_rng(71))
    table_t = ints(table)
    pool = torch.randn(2, pages, page, kv, d, dtype=torch.float16, device="cuda", generator=gen)
    q = torch.randn(rows, heads, d, dtype=torch.float16, device="cuda", generator=gen)
    at, scale = ref.offsets([r for r, _ in seqs]), 1.0 / np.sqrt(d)
    cache = PagedCache(*(TensorView.of(t).permute([0, 2, 1, 3]) for t in pool))
    batch = PagedBatch(ints(at), ints([n for _, n in seqs]), table_t, max(r for r, _ in seqs), longest)
    starts = ref.offsets([n for _, n in seqs])
    packed = torch.empty(2, int(starts[-1]), kv, d, dtype=torch.float16, device="cuda")
    for i, (_, n) in enumerate(seqs):
        packed[:, starts[i]:starts[i + 1]] = pool[:, table_t[i, :-(-n // page)].long()].reshape(2, -1, kv, d)[:, :n]
    packed_batch = PackedBatch(batch.row_offsets, ints(starts), batch.longest_rows, longest)
    for mask in (CAUSAL, NONE):
        paged, from_packed = torch.empty_like(q), torch.empty_like(q)
        for again in range(2):   # (the same bits: nothing depends on who comes first)
            out, other = torch.empty_like(q), torch.empty_like(q)
            shared_keys.attention_paged_f16(heads_view(out), heads_view(q), cache, batch, scale, 1.0, mask)
            shared_keys.attention_packed_f16(heads_view(other), heads_view(q), *(heads_view(x) for x in packed), packed_batch, scale,
                                             1.0, mask)
            assert again == 0 or (torch.equal(out, paged) and torch.equal(other, from_packed))
            paged, from_packed = out, other
        for i, (r, n) in enumerate(seqs):
            k, v = (x[starts[i]:starts[i + 1]].permute(1, 0, 2).contiguous() for x in packed)
            want = wide_attention(q[at[i]:at[i + 1]].permute(1, 0, 2).contiguous(), k, v, scale, mask == CAUSAL).permute(1, 0, 2).cpu()
            for got in (paged, from_packed):
                assert ref.close_enough(got[at[i]:at[i + 1]].cpu().numpy(), want.numpy(), float(v.abs().max()), n), (i, mask)


def test_offsets_beyond_32_bits(shared_keys):
    """Pages whose element offsets pass 2^31 and 2^32, through a page stride that spreads few pages over a large buffer."""
    kv, page, d, stride = 2, 16, 64, 1 << 30
    pool = torch.empty(5 * stride + 2 * kv * page * d, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(12)
    k, v = f16(rng, 6, kv, page, d), f16(rng, 6, kv, page, d)
    views = []
    for i, a in enumerate((k, v)):
        at = i * kv * page * d
        for g in range(6):
            pool[at + g * stride:at + g * stride + kv * page * d] = dev(a[g]).flatten()
        views.append(TensorView(pool, TensorLayout((6, kv, page, d), (stride, page * d, d, 1)), at))
    table = np.array([[5, 0, 3, 4, 2, 1]], np.int32)
    q = f16(rng, 20, 4, d)
    out = torch.zeros(20, 4, d, dtype=torch.float16, device="cuda")
    batch = PagedBatch(ints([0, 20]), ints([91]), ints(table))
    shared_keys.attention_paged_f16(heads_view(out), heads_view(dev(q)), PagedCache(*views), batch, 0.125)
    keys, values = (ref.gathered(t, table[0], 91) for t in (k, v))
    want = ref.attention(q.transpose(1, 0, 2), keys, values, 0.125).transpose(1, 0, 2)
    assert ref.close_enough(out.cpu().numpy(), want, np.abs(v).max(), 91)


# ---- rotary positions ------------------------------------------------------------------------------

def turned_close(got, want):
    """Two products and a sum in 32 bits of cosines good to a few 2^-24 (sincospi's own error and the angle's rounding
    to 32 bits, at most pi 2^-24): below 2^-20 of the pair's size, and the result's rounding to fp16."""
    want = np.asarray(want, np.float64)
    size = np.abs(want).max(axis=-1, keepdims=True)
    return (np.abs(got.astype(np.float64) - want) <= np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + size * 2.0 ** -19).all()


ROTARY = [(1, 1, 64, 64), (5, 3, 128, 128), (130, 2, 64, 32), (7, 40, 128, 64), (3, 2, 80, 20), (33, 1, 6, 4), (2, 3, 7, 6), (4, 2, 64, 0),
          (2, 2, 512, 512), (700, 1, 16, 16)]


@pytest.mark.parametrize("pairs", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: "r%d_h%d_d%d_rot%d" % c)
def test_rotary(kern, case, pairs):
    rows, heads, d, rot = case
    rng = np.random.default_rng(rows * 31 + d)
    x = f16(rng, rows, heads, d)
    positions = rng.integers(-50, 1 << 20, rows).astype(np.int32)
    scaling = RotaryScaling.Yarn(4.0, 2048) if rot > 8 else RotaryScaling.Linear(2.0)
    rotary = Rotary.new(rot, 10000.0, RotaryLayout.PAIRS if pairs else RotaryLayout.HALVES, scaling)
    want = ref.rotate(x.transpose(1, 0, 2), positions, *rotary_frequencies(rot, 10000.0, scaling), pairs).transpose(1, 0, 2)
    out = torch.full((rows, heads, d), np.nan, dtype=torch.float16, device="cuda")
    t = dev(x)
    kern.rotary_f16(heads_view(out), heads_view(t), ints(positions), rotary)
    assert turned_close(out.cpu().numpy(), want)
    kern.rotary_f16(heads_view(t), heads_view(t), ints(positions), rotary)  # in place: the same bits
    assert torch.equal(t, out)


def test_rotary_far_positions_and_back(kern):
    """The largest positions are as exact as small ones; turning back by the negative position restores the values to
    two roundings."""
    d = 64
    x = f16(np.random.default_rng(1), 4, 2, d)
    positions = np.array([2 ** 31 - 1, 2 ** 31 - 2, 10 ** 9 + 7, -2 ** 31], np.int32)
    rotary = Rotary.new(d)
    out = torch.zeros(4, 2, d, dtype=torch.float16, device="cuda")
    kern.rotary_f16(heads_view(out), heads_view(dev(x)), ints(positions), rotary)
    # angles of 2^31 turns' order carry an error of 2^31 2^-53 in 64 bits: 2^-20 of the pair more, on either side
    want = ref.rotate(x.transpose(1, 0, 2), positions, *rotary_frequencies(d), False).transpose(1, 0, 2)
    size = np.abs(want).max()
    assert (np.abs(out.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -11 + size * 2.0 ** -17).all()
    small = np.array([5, 100, 70000, 3], np.int32)
    kern.rotary_f16(heads_view(out), heads_view(dev(x)), ints(small), rotary)
    kern.rotary_f16(heads_view(out), heads_view(out), ints(-small), rotary)
    pair = np.hypot(x[..., :d // 2].astype(np.float64), x[..., d // 2:].astype(np.float64))
    assert (np.abs(out.cpu().numpy() - x.astype(np.float64)) <= np.tile(pair, 2) * (2 ** 1.5 * 2.0 ** -11 + 2.0 ** -11)).all()


@pytest.mark.parametrize("offset,stride", [(0, 1), (1, 1), (0, 3)])
def test_rotary_strides(kern, offset, stride):
    rng = np.random.default_rng(2)
    rows, heads, d = 9, 3, 32
    x = f16(rng, rows, heads, d)
    flat = torch.full((offset + rows * heads * d * stride,), np.nan, dtype=torch.float16, device="cuda")
    view = TensorView(flat, TensorLayout((heads, rows, d), (d * stride, heads * d * stride, stride)), offset)
    flat[offset::stride][:x.size] = dev(x).flatten()
    positions = np.arange(rows, dtype=np.int32) * 1000
    rotary = Rotary.new(16)
    kern.rotary_f16(view, view, ints(positions), rotary)
    want = ref.rotate(x.transpose(1, 0, 2), positions, *rotary_frequencies(16), False).transpose(1, 0, 2)
    assert turned_close(flat[offset::stride][:x.size].cpu().numpy().reshape(x.shape), want)


# ---- the cache ----------------------------------------------------------------------------------------

APPEND = [([(1, 1)], 4, 4, 64, 16, 64), ([(1, 17), (5, 5), (0, 3), (1, 300)], 8, 2, 128, 16, 128), ([(40, 100), (2, 2)], 3, 1, 40, 5, 20),
          ([(100, 100), (3, 70)], 4, 4, 64, 64, 32), ([(4, 9)], 2, 1, 7, 3, 6), ([(6, 30)], 2, 2, 64, 16, 0)]


@pytest.mark.parametrize("pairs", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("given", [False, True], ids=["cache_positions", "own_positions"])
@pytest.mark.parametrize("case", APPEND, ids=lambda c: "%s_h%d_%d_d%d_p%d_rot%d" % ("-".join("%dx%d" % s for s in c[0]), *c[1:]))
def test_append(kern, case, pairs, given):
    *shape, rot = case
    p = Paged(*shape, seed=rot + 1)
    rng = np.random.default_rng(20)
    n = p.row_offsets[-1]
    key, value = f16(rng, p.rows, p.kv, p.d), f16(rng, p.rows, p.kv, p.d)
    place = np.concatenate([np.arange(m - r, m) for r, m in p.seqs] + [np.zeros(p.rows - n)]).astype(np.int64)
    positions = rng.integers(0, 1 << 17, p.rows).astype(np.int32) if given else place
    layout = RotaryLayout.PAIRS if pairs else RotaryLayout.HALVES
    rotary = Rotary.new(rot, layout=layout) if rot else None
    freq = rotary_frequencies(rot)
    k0, v0 = p.k_t.clone(), p.v_t.clone()
    kern.append_f16(p.cache, p.batch, heads_view(dev(key)), heads_view(dev(value)), rotary, heads_view(p.out_t),
                    heads_view(p.q_t), ints(positions) if given else None)
    turn = lambda a: ref.rotate(a.transpose(1, 0, 2), positions[:len(a)], *freq, pairs).transpose(1, 0, 2)
    got = p.out_t.cpu().numpy()
    assert turned_close(got[:n], turn(p.q[:n])) and (got[n:] == SENTINEL).all()
    k_want, k_got, v_got = turn(key[:n]), p.k_t.cpu().numpy(), p.v_t.cpu().numpy()
    touched = np.zeros(k_got.shape[:1] + (p.page,), bool)
    for i, (r, m) in enumerate(p.seqs):
        for j in range(r):
            row, x = p.row_offsets[i] + j, m - r + j
            page, slot = p.table[i, x // p.page], x % p.page
            assert turned_close(k_got[page, :, slot], k_want[row])
            assert np.array_equal(v_got[page, :, slot], value[row])
            touched[page, slot] = True
    same = lambda a, b: (a == b) | (np.isnan(a) & np.isnan(b))
    for before, after in ((k0, k_got), (v0, v_got)):  # nothing else was written
        assert same(before.cpu().numpy(), after).transpose(0, 2, 1, 3)[~touched].all()
    # rotation of the queries in place, and none at all
    q = p.q_t.clone()
    kern.append_f16(p.cache, p.batch, heads_view(dev(key)), heads_view(dev(value)), rotary, heads_view(q), heads_view(q),
                    ints(positions) if given else None)
    assert torch.equal(q[:n], p.out_t[:n])
    kern.append_f16(p.cache, p.batch, heads_view(dev(key)), heads_view(dev(value)), rotary,
                    positions=ints(positions) if given else None)
    assert np.array_equal(p.k_t.cpu().numpy().view(np.uint16), k_got.view(np.uint16))


def test_append_leaves_out_what_has_no_place(kern):
    """Pages outside the cache, places in front of the first and beyond the table: not written; queries are turned."""
    p = Paged([(2, 20), (3, 2), (2, 40), (1, 16)], 2, 2, 64, 16, seed=30)
    rng = np.random.default_rng(31)
    key, value = dev(f16(rng, p.rows, 2, 64)), dev(f16(rng, p.rows, 2, 64))
    table = p.table.copy()
    table[0, 1], table[2] = -1, p.k.shape[0]
    lengths = np.array([20, 2, 40, table.shape[1] * 16 + 1], np.int32)
    batch = PagedBatch(ints(p.row_offsets), ints(lengths), ints(table))
    k0 = p.k_t.cpu().numpy()
    kern.append_f16(p.cache, batch, heads_view(key), heads_view(value), Rotary.new(64), heads_view(p.out_t), heads_view(p.q_t))
    n = p.row_offsets[-1]
    positions = np.array([18, 19, -1, 0, 1, 38, 39, lengths[3] - 1])
    want = ref.rotate(p.q[:n].transpose(1, 0, 2), positions, *rotary_frequencies(64), False).transpose(1, 0, 2)
    assert turned_close(p.out_t.cpu().numpy()[:n], want)
    got = p.k_t.cpu().numpy()
    changed = ~((got == k0) | (np.isnan(got) & np.isnan(k0))).all(axis=(1, 3))  # [pages, slots]
    expected = np.zeros_like(changed)
    expected[table[1, 0], :2] = True
    assert np.array_equal(changed, expected)


# ---- together -------------------------------------------------------------------------------------------

def test_a_prompt_and_the_tokens_behind_it(shared_keys):
    """Two sequences: a prompt into the cache in pieces, then token by token, each step rotated, appended and attended to;
    every step's result is that of the whole sequence packed, and of the definition."""
    heads, kv, d, page, k = 4, 2, 64, 16, shared_keys
    rng = np.random.default_rng(40)
    total = [83, 41]
    x = [f16(rng, n, heads + 2 * kv, d) for n in total]
    rotary, freq, scale = Rotary.new(d), rotary_frequencies(d), 1.0 / np.sqrt(d)
    turned = [np.concatenate([ref.rotate(a[:, :heads + kv].transpose(1, 0, 2), np.arange(len(a)), *freq, False)
                              .transpose(1, 0, 2).astype(np.float16), a[:, heads + kv:]], axis=1) for a in x]
    want = [ref.attention(t[:, :heads].transpose(1, 0, 2), t[:, heads:heads + kv].transpose(1, 0, 2),
                          t[:, heads + kv:].transpose(1, 0, 2), scale).transpose(1, 0, 2) for t in turned]
    pool = torch.full((2, 12, page, kv, d), np.nan, dtype=torch.float16, device="cuda")
    cache = PagedCache(*(TensorView.of(t.permute(0, 2, 1, 3)) for t in pool))
    table = ints(np.stack([rng.permutation(12)[:6] for _ in range(2)]))
    table[1] = ints([p for p in range(12) if p not in table[0].tolist()][:6])
    done, top = [0, 0], max(np.abs(a).max() for a in x)
    for step in ([50, 20], [1, 1], [0, 1], [17, 4], [1, 0], [14, 15]):
        rows = np.concatenate([a[s:s + n] for a, s, n in zip(x, done, step)])
        done = [s + n for s, n in zip(done, step)]
        qkv = TensorView.of(dev(rows)).permute([1, 0, 2])
        q, key, value = qkv.take([heads, -1, -1]), qkv.skip([heads, 0, 0]).take([kv, -1, -1]), qkv.skip([heads + kv, 0, 0])
        batch = PagedBatch(ints(ref.offsets(step)), ints(done), table, max(step), max(done))
        out = torch.zeros(len(rows), heads, d, dtype=torch.float16, device="cuda")
        k.append_f16(cache, batch, key, value, rotary, q, q)
        k.attention_paged_f16(heads_view(out), q, cache, batch, scale)
        got = out.cpu().numpy()
        expect = np.concatenate([w[s - n:s] for w, s, n in zip(want, done, step)])
        # (rotated values may round the other way here and there: one step of fp16, 2^-10, in a score's terms, which the
        # tests' scores, below 2^5 in absolute terms, turn into at most 2^5 2^-10 of the values)
        assert np.abs(got - expect).max() <= top * 2.0 ** -5
        assert np.sqrt(((got - expect) ** 2).mean()) <= top * 2.0 ** -10
    assert done == total
    # the same in one packed call, on the rotated values themselves
    whole = torch.from_numpy(np.concatenate(turned)).cuda()
    out = torch.zeros(sum(total), heads, d, dtype=torch.float16, device="cuda")
    view = TensorView.of(whole).permute([1, 0, 2])
    starts = ints(ref.offsets(total))
    k.attention_packed_f16(heads_view(out), view.take([heads, -1, -1]), view.skip([heads, 0, 0]).take([kv, -1, -1]),
                           view.skip([heads + kv, 0, 0]), PackedBatch(starts, starts), scale)
    assert ref.close_enough(out.cpu().numpy(), np.concatenate(want), top, max(total))


def test_a_captured_step_serves_later_ones():
    """One graph of append and attention, replayed while lengths, pages and values change under it."""
    heads, kv, d, page, n = 8, 2, 128, 16, 3
    k = GpuKernels(workspace_bytes=64 << 20)
    rng = np.random.default_rng(50)
    lengths_now = [5, 900, 16]
    pages, table = ref.pages_of([64, 1024, 64], page, rng)
    pool = dev(f16(rng, 2, pages, kv, page, d))
    cache = PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1]))
    lengths, tab = ints(lengths_now), ints(table)
    batch = PagedBatch(ints([0, 1, 2, 3]), lengths, tab, 1, 1024)
    qkv = torch.zeros(n, heads + 2 * kv, d, dtype=torch.float16, device="cuda")
    turned, out = (torch.zeros(n, heads, d, dtype=torch.float16, device="cuda") for _ in range(2))
    rotary, scale = Rotary.new(d), 1.0 / np.sqrt(d)
    view = TensorView.of(qkv).permute([1, 0, 2])
    q, key, value = view.take([heads, -1, -1]), view.skip([heads, 0, 0]).take([kv, -1, -1]), view.skip([heads + kv, 0, 0])

    def step():
        k.append_f16(cache, batch, key, value, rotary, heads_view(turned), q)
        k.attention_paged_f16(heads_view(out), heads_view(turned), cache, batch, scale)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(5):
        lengths_now = [a + 1 for a in lengths_now]
        lengths.copy_(ints(lengths_now))
        qkv.copy_(dev(f16(rng, n, heads + 2 * kv, d)))
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed, cached = out.clone(), pool.clone()
        out.zero_()
        pool.copy_(before)
        step()
        assert torch.equal(out, replayed) and torch.equal(pool, cached)
        k_np, v_np, q_np = pool[0].cpu().numpy(), pool[1].cpu().numpy(), turned.cpu().numpy()
        for s in range(n):
            kk, vv = (ref.gathered(t, table[s], lengths_now[s]) for t in (k_np, v_np))
            want = ref.attention(q_np[s][:, None], kk, vv, scale)[:, 0]
            assert ref.close_enough(replayed[s].cpu().numpy(), want, np.abs(vv).max(), lengths_now[s])


@pytest.mark.parametrize("seqs", [[(1, 3000), (1, 70)], [(60, 3000)], [(300, 1900), (1, 1700)]])
def test_workspace_bytes(kern, seqs):
    """What is reported is what is used: the same bits with it as through the pool; with less, or none, still right."""
    p = Paged(seqs, 8, 2, 128, 16, seed=66)
    batch = PagedBatch(p.batch.row_offsets, p.batch.lengths, p.batch.table, max(r for r, _ in seqs), 3000)
    keys = [torch.from_numpy(np.concatenate([ref.gathered(x, p.table[i], n) for i, (_, n) in enumerate(seqs)], 1)).cuda()
            for x in (p.k, p.v)]
    packed = PackedBatch(batch.row_offsets, ints(ref.offsets(p.lengths)), batch.longest_rows, 3000)
    paged_bytes = attention_paged_workspace_bytes(p.cache, batch, 8, p.rows)
    packed_bytes = attention_packed_workspace_bytes(packed, 8, 2, p.rows, sum(p.lengths), 128)
    assert paged_bytes > 0 and packed_bytes > 0

    def run(k, paged):
        p.out_t.fill_(SENTINEL)
        if paged:
            k.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, batch, 0.1)
        else:
            k.attention_packed_f16(heads_view(p.out_t), heads_view(p.q_t), *map(TensorView.of, keys), packed, 0.1)
        p.check(0.1, CAUSAL)
        return p.out_t.clone()
    lib = _ffi.lib()
    for paged, nbytes in ((True, paged_bytes), (False, packed_bytes)):
        lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES)
        pool = run(kern, paged)
        lib.adr_set_held_workspace_limit(0)
        n = p.row_offsets[-1]
        assert torch.equal(run(GpuKernels(workspace_bytes=nbytes), paged)[:n], pool[:n])
        for part in (nbytes // 2, nbytes // 7, 64):
            run(GpuKernels(workspace_bytes=part), paged)
    with pytest.raises(AdrasteaError):
        attention_paged_workspace_bytes(p.cache, batch, 7, p.rows)     # (7 heads, 2 key heads)
    with pytest.raises(AdrasteaError):
        attention_packed_workspace_bytes(packed, 8, 2, -1, 5, 128)


def test_offsets_that_decrease(shared_keys):
    """Rows that only one sequence claims are right; the others hold some result, and nothing else is written."""
    p = Paged([(10, 300), (0, 40), (10, 500)], 4, 2, 64, 16, seed=65)
    want = p.want(0.125, CAUSAL)
    # (sequence 1 ends before it begins; sequence 2 begins among the rows of sequence 0)
    p.seqs = [(10, 300), (0, 40), (15, 500)]
    batch = PagedBatch(ints([0, 10, 5, 20]), p.batch.lengths, p.batch.table)
    shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, batch, 0.125)
    got = p.out_t.cpu().numpy()
    k, v = (ref.gathered(x, p.table[2], 500) for x in (p.k, p.v))
    behind = ref.attention(p.q[5:20].transpose(1, 0, 2), k, v, 0.125).transpose(1, 0, 2)
    top = np.nanmax(np.abs(p.v.astype(np.float64)))
    assert ref.close_enough(got[:5], want[:5], top, 300) and ref.close_enough(got[10:20], behind[5:], top, 500)
    assert np.isfinite(got[5:10]).all() and (got[20:] == SENTINEL).all()


def test_two_streams_at_once(shared_keys):
    """Calls that run beside each other on two streams, each with its own part of the library's pool."""
    if shared_keys._workspace is not None:
        pytest.skip("an instance with a workspace serves one stream")
    ps = [Paged([(1, 3000), (1, 70)], 4, 2, 128, 16, seed=61), Paged([(90, 2000), (1, 5)], 4, 2, 64, 16, seed=62)]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip(ps, streams):
            with torch.cuda.stream(s):
                shared_keys.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.1)
    torch.cuda.synchronize()
    for p in ps:
        p.check(0.1, CAUSAL)


def test_two_graphs_share_a_workspace():
    """Two captured calls with one instance's buffer, replayed by turns on a stream."""
    k = GpuKernels(workspace_bytes=64 << 20)
    ps = [Paged([(1, 3000), (1, 70)], 4, 2, 128, 16, seed=63), Paged([(90, 2000), (1, 5)], 4, 2, 64, 16, seed=64)]
    graphs = []
    for p in ps:
        k.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.1)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            k.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.1)
    for _ in range(4):
        for p, g in zip(ps, graphs):
            p.out_t[:p.row_offsets[-1]] = 0
            g.replay()
    torch.cuda.synchronize()
    for p in ps:
        p.check(0.1, CAUSAL)


def test_another_stream(kern):
    p = Paged([(1, 200), (30, 60)], 4, 2, 64, 16, seed=60)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kern.attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.125)
    s.synchronize()
    p.check(0.125, CAUSAL)


def test_refusals_of_the_python_interface(kern):
    p = Paged([(2, 20)], 4, 2, 64, 16)
    out, q = heads_view(p.out_t), heads_view(p.q_t)
    b = p.batch
    for bad in ((b.row_offsets.long(), b.lengths, b.table), (b.row_offsets[:1], b.lengths, b.table),
                (b.row_offsets, b.lengths, b.table.t())):
        with pytest.raises(AssertionError):
            PagedBatch(*bad)
    for elsewhere in (PagedBatch(b.row_offsets.cpu(), b.lengths, b.table), PagedBatch(b.row_offsets, b.lengths, b.table.cpu())):
        with pytest.raises(AssertionError):
            kern.attention_paged_f16(out, q, p.cache, elsewhere, 0.1)
    with pytest.raises(AssertionError):
        kern.attention_paged_f16(out, heads_view(p.q_t.cpu()), p.cache, b, 0.1)
    with pytest.raises(AssertionError):
        kern.attention_paged_f16(heads_view(p.out_t[:, :2]), q, p.cache, p.batch, 0.1)
    with pytest.raises(AdrasteaError) as e:
        kern.attention_paged_f16(heads_view(p.out_t[:, :3]), heads_view(p.q_t[:, :3]), p.cache, p.batch, 0.1)
    assert e.value.code == _ffi.ADR_EINVAL_SHAPE
    with pytest.raises(AdrasteaError) as e:
        kern.attention_paged_f16(out, q, p.cache, p.batch, -0.1)
    assert e.value.code == _ffi.ADR_EUNSUPPORTED_LAYOUT
    with pytest.raises(AssertionError):
        kern.append_f16(p.cache, p.batch, q, q, None)
    with pytest.raises(AssertionError):
        kern.rotary_f16(out, q, ints([0]), Rotary.new(64))
    with pytest.raises(AssertionError):
        kern.attention_packed_f16(out, q, q, heads_view(p.q_t[:2]), PackedBatch(ints([0, 1]), ints([0, 1])), 0.1)


def test_the_tracer_forwards(kern):
    p = Paged([(3, 20)], 4, 2, 64, 16)
    MatmulTracer(kern).attention_paged_f16(heads_view(p.out_t), heads_view(p.q_t), p.cache, p.batch, 0.125)
    p.check(0.125, CAUSAL)
    x = dev(f16(np.random.default_rng(1), 3, 2, 64))
    a, b = torch.zeros_like(x), torch.zeros_like(x)
    MatmulTracer(kern).rotary_f16(heads_view(a), heads_view(x), ints([1, 2, 3]), Rotary.new(64))
    kern.rotary_f16(heads_view(b), heads_view(x), ints([1, 2, 3]), Rotary.new(64))
    assert torch.equal(a, b)

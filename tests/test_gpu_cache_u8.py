"""The paged cache in 8 bits on the GPU: quantised as it is written, read back, and attention over it, against plain 64-bit
definitions (step_reference.py, which also derives the tolerances).  Codes and scales have to be those of 64 bits."""
import numpy as np
import pytest
import torch

from adrastea_amd import (AdrasteaError, attention_paged_u8_workspace_bytes, GpuKernels, HeadNorm, MatmulMask, MatmulTracer, PagedBatch,
                          PagedCacheU8, RotaryAxes, RotaryLayout, TensorLayout, TensorView, _ffi, rotary_frequencies)
import sequences_reference as ref
import step_reference as step

pytestmark = pytest.mark.gpu

CAUSAL, NONE = MatmulMask.CAUSAL, MatmulMask.NONE
SENTINEL = 777.0
EPS = 1e-6
FORMS = ["a row to a wavefront", "few rows, 2 waves", "few rows, 8 waves", "few rows, shared", "many rows", "many rows, 2 groups", "many rows, shared",
         "many rows, 2 groups, shared"]
KNOBS = [1, 2, 3, 4, 5, 6, 7, 8]


@pytest.fixture(scope="module")
def kern():
    return GpuKernels()


@pytest.fixture(params=["unshared", "pool", "workspace", *FORMS])
def shared_keys(request):
    """Kernels whose keys are not shared over workgroups, shared through the library's pool, or through their own buffer;
    and each form of the kernels by itself, whatever the sizes are."""
    lib = _ffi.lib()
    forced = KNOBS[FORMS.index(request.param)] if request.param in FORMS else 0
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
    return TensorView.of(t.permute(1, 0, 2))


def sections_of(pairs, axes):
    return [pairs - (axes - 1) * (pairs // axes)] + [pairs // axes] * (axes - 1)


def axis_of(sections):
    return [a for a, n in enumerate(sections) for _ in range(n)]


def pool_of(codes, scales, order):
    """Views of [pages, kv, page, ...] arrays, kept head by head or token by token."""
    if order == "heads":
        return TensorView.of(codes), TensorView.of(scales)
    return (TensorView.of(codes.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)),
            TensorView.of(scales.permute(0, 2, 1).contiguous().permute(0, 2, 1)))


class Cache:
    """Codes and scales in pages, everything that no row may read a code of 0 and a scale of NaN."""

    def __init__(self, lengths, kv, d, page, rng, order="heads"):
        pages, self.table = ref.pages_of(lengths, page, rng)
        self.codes = np.zeros((2, pages, kv, page, d), np.uint8)
        self.scales = np.full((2, pages, kv, page), np.nan, np.float16)
        for i, n in enumerate(lengths):
            for x0 in range(0, n, page):
                m, at = min(page, n - x0), self.table[i, x0 // page]
                self.codes[:, at, :, :m] = np.clip(rng.standard_normal((2, kv, m, d)) * 40 + 127.5, 0, 255).astype(np.uint8)
                self.scales[:, at, :, :m] = rng.uniform(0.01, 0.03, (2, kv, m)).astype(np.float16)
        self.order = order
        self.upload()

    def upload(self):
        k, ks = pool_of(dev(self.codes[0]), dev(self.scales[0]), self.order)
        v, vs = pool_of(dev(self.codes[1]), dev(self.scales[1]), self.order)
        self.handle = PagedCacheU8(k, ks, v, vs)

    def values(self, i, n):
        """Keys and values [kv, n, d] of sequence i."""
        out = []
        for t in (0, 1):
            codes = ref.gathered(self.codes[t], self.table[i], n)
            scales = ref.gathered(self.scales[t][..., None], self.table[i], n)[..., 0]
            out.append(step.value_of(codes, scales))
        return out


class Paged:
    def __init__(self, seqs, heads, kv, d, page, seed=0, order="heads", spare=3):
        rng = np.random.default_rng(seed)
        self.seqs, self.heads, self.d = seqs, heads, d
        self.rows = sum(r for r, _ in seqs) + spare
        self.row_offsets = ref.offsets([r for r, _ in seqs])
        self.lengths = [n for _, n in seqs]
        self.cache = Cache(self.lengths, kv, d, page, rng, order)
        self.q = f16(rng, self.rows, heads, d)
        self.q[self.row_offsets[-1]:] = np.nan
        self.q_t = dev(self.q)
        self.out_t = torch.full((self.rows, heads, d), SENTINEL, dtype=torch.float16, device="cuda")
        self.batch = PagedBatch(ints(self.row_offsets), ints(self.lengths), ints(self.cache.table))

    def want(self, scale, mask, temp=1.0):
        out = np.full((self.rows, self.heads, self.d), SENTINEL)
        for i, (r, n) in enumerate(self.seqs):
            a = self.row_offsets[i]
            k, v = self.cache.values(i, n)
            out[a:a + r] = ref.attention(self.q[a:a + r].transpose(1, 0, 2), k, v, scale, temp, mask == CAUSAL).transpose(1, 0, 2)
        return out

    def cache_scale(self, which, i, h, n):
        return ref.gathered(self.cache.scales[which][..., None], self.cache.table[i], n)[h, :, 0].astype(np.float64)

    def check(self, scale, mask, temp=1.0):
        want, got = self.want(scale, mask, temp), self.out_t.cpu().numpy()
        n = self.row_offsets[-1]
        assert np.array_equal(got[n:], want[n:].astype(np.float16)), "rows behind the last sequence"
        top = 127.5 * np.nanmax(self.cache.scales[1].astype(np.float64), initial=0.0)
        assert step.close_enough(got[:n], want[:n], top, max([n for _, n in self.seqs] + [1]), True)
        return got


# ---- written and read back -----------------------------------------------------------------------------------

# (sequences of (rows, keys), heads, kv heads, d, page, rotated values, axes, pairs)
APPENDS = [([(1, 1)], 4, 4, 64, 16, 64, 1, False), ([(1, 37), (0, 5), (3, 3), (5, 70)], 8, 2, 128, 16, 128, 3, False),
           ([(1, i + 1) for i in range(70)], 4, 1, 64, 32, 32, 1, True), ([(40, 41), (4, 2)], 6, 2, 80, 16, 80, 2, False),
           ([(3, 9), (4, 30)], 2, 1, 7, 5, 6, 2, True), ([(200, 260), (0, 0), (1, 64)], 5, 5, 96, 64, 96, 3, False),
           ([(2, 5)] * 130, 2, 2, 64, 16, 64, 2, True), ([(700, 700), (300, 301)], 2, 8, 128, 16, 128, 1, False),
           ([(5, 9)], 1, 1, 256, 16, 256, 1, False), ([(3, 3)], 2, 2, 8, 16, 0, 1, False)]
APPENDS = [c for c in APPENDS if c[1] % c[2] == 0 or c[1] == 5]


@pytest.mark.parametrize("norm", [True, False], ids=["normed", "plain"])
@pytest.mark.parametrize("case", APPENDS, ids=["s%d_h%d_%d_d%d_p%d" % (len(c[0]), *c[1:5]) for c in APPENDS])
def test_codes_are_those_of_64_bits(kern, case, norm):
    seqs, heads, kv, d, page, rot, axes, pairs = case
    rng = np.random.default_rng(len(seqs) + d)
    rows, lengths = [r for r, _ in seqs], [n for _, n in seqs]
    starts, total = ref.offsets(rows), sum(rows) + 2
    n = int(starts[-1])
    qkv, weight = f16(rng, total, heads + 2 * kv, d, std=2.0), f16(rng, d)
    packed = dev(qkv)
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    cache = Cache(lengths, kv, d, page, rng, "tokens" if len(seqs) % 2 else "heads")
    out = torch.full((total, heads, d), SENTINEL, dtype=torch.float16, device="cuda")
    sections = sections_of(rot // 2, axes)
    positions = rng.integers(0, 100000, (axes, total))
    rotary = RotaryAxes.new(rot, sections, layout=RotaryLayout.PAIRS if pairs else RotaryLayout.HALVES)
    batch = PagedBatch(ints(starts), ints(lengths), ints(cache.table))
    head_norm = HeadNorm(dev(weight), EPS) if norm else None
    kern.append_u8(cache.handle, batch, heads_view(k), heads_view(v), rotary, heads_view(out), heads_view(q), ints(positions),
                   head_norm, head_norm)
    x = [step.normed(t, weight, EPS) if norm else t.astype(np.float64) for t in (qkv[:n, :heads], qkv[:n, heads:heads + kv])]
    frequencies = rotary_frequencies(rot)[0]
    want_q, want_k = (step.turned(t.transpose(1, 0, 2), positions[:, :n], axis_of(sections), frequencies, 1.0, pairs) for t in x)
    got_q = out.cpu().numpy()
    assert (got_q[n:] == SENTINEL).all()
    assert (np.abs(got_q[:n].transpose(1, 0, 2) - want_q) <= step.turned_bound(want_q, x[0].transpose(1, 0, 2), rot // 2, 1.0, pairs)).all()
    codes, scales = cache.codes.copy(), cache.scales.copy()
    place = [(i, length - r + j) for i, (r, length) in enumerate(seqs) for j in range(r)]
    for t, y in ((0, want_k.transpose(1, 0, 2)), (1, qkv[:n, heads + kv:].astype(np.float64))):
        c, s = step.quantised(y)
        for row, (i, at) in enumerate(place):
            if at >= 0:
                codes[t, cache.table[i, at // page], :, at % page] = c[row]
                scales[t, cache.table[i, at // page], :, at % page] = s[row]
    h = cache.handle
    got = [[view.storage.cpu().numpy() for view in pair] for pair in ((h.key, h.key_scale), (h.value, h.value_scale))]
    for t in (0, 1):
        assert np.array_equal(got[t][0], codes[t]), "codes"
        assert np.array_equal(got[t][1], scales[t], equal_nan=True), "scales"
    # the way back: half a scale from what was written, at most
    read = [torch.full((total, kv, d), SENTINEL, dtype=torch.float16, device="cuda") for _ in range(2)]
    kern.read_u8(heads_view(read[0]), heads_view(read[1]), cache.handle, batch)
    for t, y in ((0, want_k.transpose(1, 0, 2)), (1, qkv[:n, heads + kv:].astype(np.float64))):
        got_t = read[t].cpu().numpy()
        assert (got_t[n:] == SENTINEL).all()
        for row, (i, at) in enumerate(place):
            if at < 0:
                assert np.isnan(got_t[row]).all()
                continue
            slot = (t, cache.table[i, at // page], slice(None), at % page)
            want = ((codes[slot].astype(np.float32) - np.float32(127.5)) * scales[slot].astype(np.float32)[:, None]).astype(np.float16)
            assert np.array_equal(got_t[row], want)
            s = scales[slot].astype(np.float64)[:, None]
            assert (np.abs(step.value_of(codes[slot], scales[slot]) - y[row]) <= s / 2 * (1 + 2.0 ** -40)).all()


@pytest.mark.parametrize("d", [64, 7], ids=["d64", "any layout"])
def test_heads_at_the_ends_of_the_format(kern, d):
    """Zeros, the smallest numbers of fp16, the largest, one step's borders, infinities and NaN: codes, scales, and values that
    do not reach other heads."""
    kinds = np.zeros((9, d), np.float16)
    kinds[1, 0], kinds[2], kinds[3], kinds[4] = 2.0 ** -24, 65504.0, -65504.0, np.arange(d) * 2.0 ** -24
    kinds[5] = np.float16(0.5) * (np.arange(d) % 3 - 1)
    kinds[5, 0] = 63.75          # the scale is 0.5, and the others lie on borders of its steps
    kinds[6, 1], kinds[7, 2], kinds[8, 3] = np.nan, np.inf, -np.inf
    rows = len(kinds)
    both = np.stack([kinds, np.ones_like(kinds)], axis=1)  # a head of ones beside each
    cache = Cache([rows], 2, d, 16, np.random.default_rng(0))
    batch = PagedBatch(ints([0, rows]), ints([rows]), ints(cache.table))
    x = heads_view(dev(both))
    kern.append_u8(cache.handle, batch, x, x)
    want_codes, want_scales = step.quantised(both.astype(np.float64))
    page = cache.table[0, 0]
    for codes, scales in ((cache.handle.key, cache.handle.key_scale), (cache.handle.value, cache.handle.value_scale)):
        assert np.array_equal(codes.storage.cpu().numpy()[page, :, :rows].transpose(1, 0, 2), want_codes)
        assert np.array_equal(scales.storage.cpu().numpy()[page, :, :rows].T, want_scales, equal_nan=True)
    assert want_scales[0, 0] == 0 and want_scales[1, 0] == 2.0 ** -24 and want_scales[2, 0] == 513.5 and want_scales[5, 0] == 0.5
    assert np.isnan(want_scales[6:, 0]).all() and (want_scales[:, 1] == want_scales[0, 1]).all()
    out = [torch.zeros(rows, 2, d, dtype=torch.float16, device="cuda") for _ in range(2)]
    kern.read_u8(heads_view(out[0]), heads_view(out[1]), cache.handle, batch)
    for t in out:
        t = t.cpu().numpy()
        assert (t[0, 0] == 0).all() and np.isnan(t[6:, 0]).all() and np.isfinite(t[:6]).all()
        assert (np.abs(t[:6, 0].astype(np.float64) - kinds[:6]) <= want_scales[:6, :1].astype(np.float64) / 2 + np.abs(kinds[:6]) * 2.0 ** -11
                + 2.0 ** -25).all()


def test_keys_beyond_the_format_and_slots_that_are_not_there(kern):
    """A weight makes keys of more than 65504, which are stored as the largest; rows on pages of -1, beyond the table or in front of
    the first key are written nowhere, and read as NaN."""
    rng = np.random.default_rng(1)
    cache = Cache([8, 40], 2, 64, 16, rng)
    before = cache.codes.copy()
    table = cache.table.copy()
    table[1, 1] = -1
    k = f16(rng, 20, 2, 64)
    weight = np.full(64, 60000.0, np.float16)
    # sequence 0 has 8 keys and 10 rows (two in front of the first), sequence 1 has 10 rows on its second and third page
    batch = PagedBatch(ints([0, 10, 20]), ints([8, 36]), ints(table[:, :2]))
    kern.append_u8(cache.handle, batch, heads_view(dev(k)), heads_view(dev(k)), key_norm=HeadNorm(dev(weight), EPS))
    c, s = step.quantised(step.normed(k, weight, EPS))
    assert (s == np.float16(513.5)).any()
    got, scale = (t.storage.cpu().numpy() for t in (cache.handle.key, cache.handle.key_scale))
    page = table[0, 0]
    assert np.array_equal(got[page, :, :8].transpose(1, 0, 2), c[2:10]) and np.array_equal(scale[page, :, :8].T, s[2:10])
    others = np.ones(got.shape[0], bool)
    others[page] = False
    assert np.array_equal(got[others], before[0][others]), "rows without a slot"
    out = [torch.full((20, 2, 64), SENTINEL, dtype=torch.float16, device="cuda") for _ in range(2)]
    kern.read_u8(heads_view(out[0]), heads_view(out[1]), cache.handle, batch)
    nowhere = np.ones(20, bool)
    nowhere[2:10] = False
    for t in out:
        t = t.cpu().numpy()
        assert np.isnan(t[nowhere]).all() and np.isfinite(t[~nowhere]).all()


# ---- attention -------------------------------------------------------------------------------------------------

PAGED = [
    ([(1, 1)], 1, 1, 64, 16), ([(1, 37)], 4, 4, 128, 16), ([(1, 300), (1, 1), (0, 0), (1, 64), (1, 65), (0, 9)], 8, 2, 128, 16),
    ([(5, 5), (3, 130), (0, 20), (2, 2)], 6, 2, 64, 32), ([(4, 2), (3, 0), (1, 0)], 4, 4, 64, 16),
    ([(70, 200), (1, 513), (129, 129)], 4, 1, 128, 64), ([(33, 140)], 5, 1, 128, 16), ([(17, 17), (16, 600)], 7, 7, 64, 128),
    ([(2, 75), (40, 41)], 3, 1, 48, 16), ([(3, 90)], 2, 2, 16, 32), ([(9, 100), (1, 260)], 4, 2, 80, 16), ([(1, 2100)], 16, 2, 96, 16),
    ([(3, 50)], 2, 1, 7, 4), ([(3, 70), (1, 5)], 2, 2, 160, 16), ([(2, 40)], 2, 1, 256, 16), ([(3, 21), (1, 64)], 4, 2, 64, 1),
    ([(3, 50), (1, 49)], 4, 2, 128, 5), ([(2, 100), (65, 300)], 4, 4, 64, 48), ([(1, 4000), (2, 3)], 2, 2, 128, 16),
    ([(200, 1500)], 4, 2, 128, 32), ([(300, 300), (40, 900)], 2, 1, 64, 16),
]
IDS = ["%s_h%d_%d_d%d_p%d" % ("-".join("%dx%d" % s for s in c[0]), *c[1:]) for c in PAGED]


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("case", PAGED, ids=IDS)
def test_attention(shared_keys, case, mask):
    p = Paged(*case, seed=len(case[0]) * 100 + case[3], order="tokens" if case[4] == 16 else "heads")
    scale = 1.0 / np.sqrt(p.d)
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, scale, 1.3, mask)
    p.check(scale, mask, 1.3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows,keys", [(2, 9), (7, 200), (40, 40), (200, 330)])
def test_what_a_row_does_not_see_never_reaches_it(shared_keys, rows, keys, d):
    """A scale of the last key that is no finite number, or larger than codes have values for, makes NaN of the last row alone."""
    p = Paged([(rows, keys), (3, 3)], 4, 2, d, 16, seed=rows)
    scale = 1.0 / np.sqrt(d)
    place = (p.cache.table[0, (keys - 1) // 16], slice(None), (keys - 1) % 16)
    clean = p.cache.scales.copy()
    for which, bad in ((0, np.nan), (0, np.inf), (0, 514.0), (1, np.nan), (1, -np.inf), (1, 600.0)):
        p.cache.scales[:] = clean
        p.cache.scales[(which, *place)] = bad
        p.cache.upload()
        shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, scale)
        got = p.out_t.cpu().numpy()
        p.cache.scales[(which, *place)] = clean[(which, *place)]  # (the others do not see it)
        want = p.want(scale, CAUSAL)
        seen = np.ones(p.row_offsets[-1], bool)
        seen[rows - 1] = False
        top = 127.5 * 0.03
        assert np.isnan(got[rows - 1]).all()
        assert step.close_enough(got[:p.row_offsets[-1]][seen], want[:p.row_offsets[-1]][seen], top, keys, True)


def test_queries_that_are_no_numbers(shared_keys):
    """NaN for their rows, where those see a key."""
    p = Paged([(2, 50), (1, 0), (1, 30)], 4, 2, 64, 16, seed=1)
    p.q[0, 1, 5], p.q[2], p.q[3, 2, 0] = np.inf, np.nan, -np.inf
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(dev(p.q)), p.cache.handle, p.batch, 0.125)
    got = p.out_t.cpu().numpy()
    assert np.isnan(got[0, 1]).all() and np.isnan(got[3, 2]).all() and (got[2] == 0).all()
    assert np.isfinite(got[0, [0, 2, 3]]).all() and np.isfinite(got[1]).all() and np.isfinite(got[3, [0, 1, 3]]).all()


def test_pages_outside_the_cache_are_nan_and_never_read(shared_keys):
    p = Paged([(1, 40), (3, 40), (1, 100), (1, 20)], 4, 2, 64, 16, seed=5)
    for bad in (-1, 1 << 20, p.cache.codes.shape[1], -2 ** 31):
        table = p.cache.table.copy()
        table[1, 2] = bad         # keys 32 .. 39 of sequence 1, of which its rows see 6, 7 and 8
        table[2, 7:] = bad        # behind the last key
        p.batch = PagedBatch(ints(p.row_offsets), ints(p.lengths), ints(table))
        shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125)
        got, want = p.out_t.cpu().numpy(), p.want(0.125, CAUSAL)
        assert np.isnan(got[1:4]).all()
        rest = [0, 4, 5]
        assert step.close_enough(got[rest], want[rest], 127.5 * 0.03, 100, True)


def test_values_of_very_different_sizes(shared_keys):
    """A key with most of the weight whose values are tiny, or zero, beside keys of large values and little weight, and the other way
    round: each as exact as the rest of the row allows.  Bounds: sums of the weights' roundings, 2^-11 of each |w v| and 2^-32 of the
    row's largest |w v|'s scale a key, over the 32-bit sums' (keys + 127) 2^-23 of what they add up to, and the result's own."""
    d, n = 64, 600
    for first, rest, near in ((2.0 ** -24, 513.5, 8.0), (0.0, 513.5, 20.0), (513.5, 2.0 ** -24, -30.0), (0.01, 1e-6, -16.0), (1e-6, 0.01, 16.0),
                              (0.0, 0.0, 1.0), (513.5, 2.0 ** -20, -60.0)):
        p = Paged([(1, n), (2, n)], 2, 2, d, 16, seed=3)
        for i in range(2):
            for x in range(n):
                at = (slice(None), p.cache.table[i, x // 16], slice(None), x % 16)
                p.cache.scales[1][at[1:]] = first if x == 77 else rest
                p.cache.scales[0][at[1:]] = 0.02
                p.cache.codes[0][at[1:]] = 128 if x != 77 else 255
        p.cache.upload()
        p.q[:p.row_offsets[-1]] = 1.0
        # the score of key 77 is `near` log2 units above the others'
        step_of = 64 * 127 * float(np.float16(0.02))
        scale = abs(near) * np.log(2) / step_of
        if near < 0:
            p.q[:p.row_offsets[-1]] = -1.0
        shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(dev(p.q)), p.cache.handle, p.batch, scale)
        got = p.out_t.cpu().numpy()
        for i, (r, m) in enumerate(p.seqs):
            k, v = p.cache.values(i, m)
            for j in range(r):
                row, end = p.row_offsets[i] + j, j + m - r + 1
                for h in range(2):
                    s = k[h, :end] @ p.q[row, h].astype(np.float64) * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    want = w @ v[h, :end]
                    each = (w[:, None] * np.abs(v[h, :end])).sum(0)
                    sizes = w * p.cache_scale(1, i, h, end)
                    bound = (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + each * 2.0 ** -11 + 127.5 * sizes.max() * end * 2.0 ** -32 +
                             127.5 * sizes.sum() * (end + 127) * 2.0 ** -23 + each * 2.0 ** -11)
                    assert (np.abs(got[row, h] - want) <= bound).all(), (first, rest, near, row, h)


def test_scores_of_any_size_and_values_near_the_largest(shared_keys):
    """Queries and scales with which scores pass 2^24 in log2 units: the largest one's value; a mean of values at the end of the
    format is finite."""
    p = Paged([(3, 70), (2, 33)], 2, 2, 64, 16, seed=7)
    p.q[:p.row_offsets[-1]] = np.sign(p.q[:p.row_offsets[-1]]) * 30000
    p.cache.scales[0][~np.isnan(p.cache.scales[0])] = 200.0
    p.cache.codes[1][:] = 255
    p.cache.scales[1][~np.isnan(p.cache.scales[1])] = 513.5
    p.cache.upload()
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(dev(p.q)), p.cache.handle, p.batch, 1.0)
    got = p.out_t.cpu().numpy()[:p.row_offsets[-1]].astype(np.float64)
    assert np.isfinite(got).all() and (np.abs(got - 127.5 * 513.5) <= 65504 * 2.0 ** -9).all()
    p.cache.codes[1] = np.random.default_rng(3).integers(0, 256, p.cache.codes[1].shape)
    p.cache.scales[1][~np.isnan(p.cache.scales[1])] = 0.02
    p.cache.upload()
    shared_keys.attention_paged_u8(heads_view(p.out_t), heads_view(dev(p.q)), p.cache.handle, p.batch, 1.0)
    p.check(1.0, CAUSAL)


@pytest.mark.parametrize("odd", ["query row pitch", "column stride", "code start", "overlapping slots", "negative page stride"])
def test_other_layouts(shared_keys, odd):
    p = Paged([(2, 50), (5, 20)], 4, 2, 64, 16, seed=9)
    out, q, h = heads_view(p.out_t), heads_view(p.q_t), p.cache.handle
    if odd == "query row pitch":
        wide = torch.zeros(p.rows, 4, 67, dtype=torch.float16, device="cuda")
        wide[:, :, :64] = p.q_t
        q = TensorView(wide, TensorLayout((4, p.rows, 64), (67, 4 * 67, 1)))
    elif odd == "column stride":
        wide = torch.zeros(p.rows, 4, 128, dtype=torch.float16, device="cuda")
        wide[:, :, ::2] = SENTINEL
        out = TensorView(wide, TensorLayout((4, p.rows, 64), (128, 4 * 128, 2)))
    elif odd == "code start":
        codes = dev(p.cache.codes[0])
        store = torch.zeros(codes.numel() + 16, dtype=torch.uint8, device="cuda")
        store[5:5 + codes.numel()] = codes.flatten()
        h = PagedCacheU8(TensorView(store, TensorLayout.row_major(codes.shape), 5), h.key_scale, h.value, h.value_scale)
    elif odd == "overlapping slots":
        p.cache.scales[1][:] = 0.01  # (every value the same 64 codes, and one scale)
        flat = dev(p.cache.codes[1][0, 0, 0])
        one = torch.full((1,), 0.01, dtype=torch.float16, device="cuda")
        dims = p.cache.codes[1].shape
        h = PagedCacheU8(h.key, h.key_scale, TensorView(flat, TensorLayout._of_checked(dims, (0, 0, 0, 1))),
                         TensorView(one, TensorLayout._of_checked(dims[:3], (0, 0, 0))))
        p.cache.codes[1][:] = p.cache.codes[1][0, 0, 0]
        p.cache.scales[1][:] = np.float16(0.01)
    else:
        codes, pages = dev(p.cache.codes[0][::-1]), p.cache.codes.shape[1]
        s = codes.stride()
        h = PagedCacheU8(TensorView(codes, TensorLayout(tuple(codes.shape), (-s[0], *s[1:])), (pages - 1) * s[0]), h.key_scale, h.value,
                         h.value_scale)
    shared_keys.attention_paged_u8(out, q, h, p.batch, 0.125)
    if odd == "column stride":
        p.out_t.copy_(wide[:, :, ::2])
    p.check(0.125, CAUSAL)


def test_a_captured_step_replays(kern):
    """Append, read and attention of one token each, captured with their own buffer and replayed over lengths that grow, beside the
    program's eager work."""
    rng = np.random.default_rng(11)
    heads, kv, d, page, seqs = 8, 2, 64, 16, 5
    cache = Cache([200] * seqs, kv, d, page, rng)
    lengths = ints([3, 30, 15, 16, 99])
    batch = PagedBatch(ints(range(seqs + 1)), lengths, ints(cache.table), 1, 200)
    qkv = torch.zeros(seqs, heads + 2 * kv, d, dtype=torch.float16, device="cuda")
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    weight = HeadNorm(dev(f16(rng, d)), EPS)
    rotary = RotaryAxes.new(d, [d // 2])
    kern = GpuKernels(workspace_bytes=max(attention_paged_u8_workspace_bytes(cache.handle, batch, heads, seqs), 16))
    tensors = [torch.zeros(seqs, n, d, dtype=torch.float16, device="cuda") for n in (heads, heads, kv, kv)]

    def work():
        turned, out, read_k, read_v = (heads_view(t) for t in tensors)
        kern.append_u8(cache.handle, batch, heads_view(k), heads_view(v), rotary, turned, heads_view(q), None, weight, weight)
        kern.read_u8(read_k, read_v, cache.handle, batch)
        kern.attention_paged_u8(out, turned, cache.handle, batch, 0.125)
    work()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        work()
    for _ in range(4):
        lengths += 1
        qkv.copy_(dev(f16(rng, *qkv.shape)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in tensors]
        for t in tensors:
            t.zero_()
        work()
        for a, b in zip(got, tensors):
            assert torch.equal(a, b) and a.abs().max() > 0


def test_on_another_stream(kern):
    p = Paged([(1, 500), (1, 40)], 4, 2, 64, 16, seed=3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        kern.attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125)
    stream.synchronize()
    p.check(0.125, CAUSAL)


def test_refusals_through_python(kern):
    p = Paged([(2, 20)], 4, 2, 64, 16)
    h, out, q = p.cache.handle, heads_view(p.out_t), heads_view(p.q_t)
    halves = torch.zeros(*p.cache.codes[0].shape, dtype=torch.float16, device="cuda")
    for bad in (lambda: PagedCacheU8(TensorView.of(halves), h.key_scale, h.value, h.value_scale),
                lambda: PagedCacheU8(h.key, TensorView.of(halves[..., 0].float()), h.value, h.value_scale),
                lambda: kern.attention_paged_u8(TensorView.of(p.out_t.float().permute(1, 0, 2)), q, h, p.batch, 0.1)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: PagedCacheU8(h.key, h.key, h.value, h.value_scale),
                lambda: PagedCacheU8(h.key, h.key_scale, h.key_scale, h.value_scale),
                lambda: kern.attention_paged_u8(out, heads_view(p.q_t[:, :, :32]), h, p.batch, 0.1),
                lambda: kern.read_u8(out, out, h, p.batch),
                lambda: kern.append_u8(h, p.batch, q, q),
                lambda: kern.attention_paged_u8(TensorView.of(p.out_t.cpu().permute(1, 0, 2)), q, h, p.batch, 0.1)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(AdrasteaError):
        kern.attention_paged_u8(out, q, h, p.batch, 0.1, 1.0, 2)
    with pytest.raises(AdrasteaError):
        kern.attention_paged_u8(out, q, h, p.batch, -0.1)
    assert (p.out_t == SENTINEL).all()


def test_the_tracer_forwards(kern):
    p = Paged([(2, 20)], 4, 2, 64, 16)
    MatmulTracer(kern).attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, 0.125)
    p.check(0.125, CAUSAL)

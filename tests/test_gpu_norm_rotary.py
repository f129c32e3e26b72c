"""Heads normed and turned in one pass, by positions on several axes, alone and into the paged cache, on the GPU, against plain
64-bit definitions (step_reference.py, which also derives the tolerance)."""
import numpy as np
import pytest
import torch

from adrastea_amd import (AdrasteaError, GpuKernels, HeadNorm, MatmulTracer, PagedBatch, PagedCache, Rotary, RotaryAxes, RotaryLayout,
                          TensorLayout, TensorView, rotary_frequencies)
import sequences_reference as ref
import step_reference as step

pytestmark = pytest.mark.gpu

SENTINEL = 777.0
EPS = 1e-5


@pytest.fixture(scope="module")
def kern():
    return GpuKernels()


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


# (heads, rows, d, rotated values, axes, pairs): whole heads and parts, odd chunk counts, sizes off the vector path
TURNS = [(32, 1, 128, 128, 1, False), (3, 5, 64, 64, 2, False), (2, 33, 128, 64, 3, True), (16, 7, 80, 80, 2, False), (1, 1, 8, 8, 1, True),
         (4, 9, 96, 48, 3, False), (5, 3, 80, 40, 2, False), (2, 4, 7, 6, 1, False), (1, 2, 1, 0, 1, False), (3, 6, 256, 128, 4, True),
         (2, 3, 512, 512, 8, False), (2, 3, 600, 500, 2, True), (7, 300, 64, 32, 1, False), (2, 5, 128, 0, 1, False), (1, 3000, 128, 128, 3, True),
         (3, 5, 72, 64, 1, False), (3, 5, 72, 8, 1, True)]


@pytest.mark.parametrize("norm", [True, False], ids=["normed", "plain"])
@pytest.mark.parametrize("case", TURNS, ids=["h%d_r%d_d%d_%d_a%d_%s" % (*c[:5], "pairs" if c[5] else "halves") for c in TURNS])
def test_norm_and_rotation(kern, case, norm):
    heads, rows, d, rot, axes, pairs = case
    rng = np.random.default_rng(rows * 1000 + d)
    x, weight = f16(rng, rows, heads, d, std=3.0), f16(rng, d)
    sections = sections_of(rot // 2, axes)
    positions = rng.integers(-500, 200000, (axes, rows))
    layout = RotaryLayout.PAIRS if pairs else RotaryLayout.HALVES
    rotary = RotaryAxes.new(rot, sections, layout=layout)
    out = torch.full((rows, heads, d), SENTINEL, dtype=torch.float16, device="cuda")
    kern.norm_rotary_f16(heads_view(out), heads_view(dev(x)), ints(positions), rotary, HeadNorm(dev(weight), EPS) if norm else None)
    y = step.normed(x, weight, EPS) if norm else x.astype(np.float64)
    y = y.transpose(1, 0, 2)
    want = step.turned(y, positions, axis_of(sections), rotary_frequencies(rot)[0], 1.0, pairs)
    got = out.cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(got - want) <= step.turned_bound(want, y, rot // 2, 1.0, pairs)).all()


def test_one_axis_without_a_norm_is_the_plain_rotation(kern):
    """What rotary_f16 computes, for positions of rank 1 and 2, a Rotary or a RotaryAxes, and in place.  Not its bits: which of two
    products is fused into their sum is the compiler's choice for each kernel, a rounding of 2^-24 of a partner either way.  So
    both are held to the definition, and the forms of the call to each other's bits."""
    rng = np.random.default_rng(1)
    x, positions = dev(f16(rng, 40, 6, 128)), ints(rng.integers(0, 1 << 20, 40))
    y = x.cpu().numpy().transpose(1, 0, 2)
    want = step.turned(y, positions.cpu().numpy()[None], [0] * 64, rotary_frequencies(128)[0], 1.0, False)
    bound = step.turned_bound(want, y.astype(np.float64), 64, 1.0, False)
    got, first = torch.empty_like(x), torch.empty_like(x)
    plain = Rotary.new(128)
    kern.rotary_f16(heads_view(got), heads_view(x), positions, plain)
    assert (np.abs(got.cpu().numpy().transpose(1, 0, 2) - want) <= bound).all()
    kern.norm_rotary_f16(heads_view(first), heads_view(x), positions, plain)
    assert (np.abs(first.cpu().numpy().transpose(1, 0, 2) - want) <= bound).all()
    for p in (positions, positions[None]):
        got.zero_()
        kern.norm_rotary_f16(heads_view(got), heads_view(x), p, RotaryAxes.new(128, [64]))
        assert torch.equal(got, first)
    kern.norm_rotary_f16(heads_view(x), heads_view(x), positions, plain)
    assert torch.equal(x, first)


def test_frequencies_of_each_axis():
    own = RotaryAxes.new(80, [20, 20], own_frequencies=True)
    assert torch.equal(own.turns[:20], own.turns[20:]) and torch.equal(own.turns[:20], Rotary.new(40).turns)
    assert own.axis.tolist() == [0] * 20 + [1] * 20


def test_an_axis_out_of_range_counts_as_the_first(kern):
    rng = np.random.default_rng(2)
    x, positions = dev(f16(rng, 9, 2, 64)), ints(rng.integers(0, 1000, (2, 9)))
    good = RotaryAxes.new(64, [32, 0])
    bad = RotaryAxes(good.turns, ints([7, -1, 2, 1 << 30] * 8), 2)
    want, got = torch.empty_like(x), torch.empty_like(x)
    kern.norm_rotary_f16(heads_view(want), heads_view(x), positions, good)
    kern.norm_rotary_f16(heads_view(got), heads_view(x), positions, bad)
    assert torch.equal(got, want)


@pytest.mark.parametrize("d", [64, 80, 7], ids=["d64", "d80", "any layout"])
def test_heads_that_are_zero_huge_or_no_numbers(kern, d):
    """A head of zeros stays one under a positive eps and is NaN under none; the largest numbers of fp16 and the smallest are
    normed as others; a NaN stays in its head, and what passes is not mixed with what is turned."""
    rot = d // 4 * 2 if d == 7 else 16
    x = np.ones((6, 2, d), np.float16)
    x[0], x[1], x[2], x[3, 0, 0], x[4, 0, 0], x[4, 0, -1] = 0.0, 65504.0, 2.0 ** -24, np.nan, np.inf, 1.0
    weight = np.ones(d, np.float16)
    positions, rotary = ints(np.zeros(6)), Rotary.new(rot)

    def run(eps):
        out = torch.zeros(6, 2, d, dtype=torch.float16, device="cuda")
        kern.norm_rotary_f16(heads_view(out), heads_view(dev(x)), positions, rotary, HeadNorm(dev(weight), eps))
        return out.cpu().numpy()
    got, bare = run(1e-6), run(0.0)
    assert (got[0] == 0).all() and np.isnan(bare[0]).all()
    assert (np.abs(got[1] - 1) <= 2.0 ** -10).all() and (np.abs(bare[2] - 1) <= 2.0 ** -10).all()
    assert np.isnan(got[3, 0]).all() and (np.abs(got[3, 1] - 1) < 2.0 ** -10).all()
    assert np.isnan(got[4, 0, 0]) and got[4, 0, -1] == 0 and (np.abs(got[5] - 1) <= 2.0 ** -10).all()
    out = torch.zeros(6, 2, d, dtype=torch.float16, device="cuda")
    kern.norm_rotary_f16(heads_view(out), heads_view(dev(x)), positions, rotary)
    assert (out[4, 0, rot:].cpu().numpy() == 1).all()


@pytest.mark.parametrize("odd", ["d", "column stride", "row pitch", "start"])
def test_other_layouts(kern, odd):
    rng = np.random.default_rng(3)
    d, rows, heads = (66 if odd == "d" else 64), 11, 3
    x, weight = f16(rng, rows, heads, d), f16(rng, d)
    store = torch.full((rows * heads * d * 3 + 64,), SENTINEL, dtype=torch.float16, device="cuda")
    strides = {"d": (heads * d, d, 1), "column stride": (heads * d * 2, d * 2, 2), "row pitch": (heads * d + 1, d, 1),
               "start": (heads * d, d, 1)}[odd]
    start = 3 if odd == "start" else 0
    at = store.as_strided((rows, heads, d), strides, start)
    at.copy_(dev(x))
    positions = ints(rng.integers(0, 5000, (2, rows)))
    sections = sections_of(d // 2, 2)
    view = TensorView(store, TensorLayout((heads, rows, d), (strides[1], strides[0], strides[2])), start)
    kern.norm_rotary_f16(view, view, positions, RotaryAxes.new(d // 2 * 2, sections), HeadNorm(dev(weight), EPS))
    y = step.normed(x, weight, EPS).transpose(1, 0, 2)
    want = step.turned(y, positions.cpu().numpy(), axis_of(sections), rotary_frequencies(d // 2 * 2)[0], 1.0, False)
    got = at.cpu().numpy().transpose(1, 0, 2)
    assert (np.abs(got - want) <= step.turned_bound(want, y, d // 2, 1.0, False)).all()
    at.fill_(SENTINEL)
    assert (store == SENTINEL).all(), "values between the rows"


# (sequences of (rows, keys), heads, kv heads, d, page, rotated values, axes, pairs)
APPENDS = [([(1, 1)], 4, 4, 64, 16, 64, 1, False), ([(1, 37), (0, 5), (3, 3), (5, 70)], 8, 2, 128, 16, 128, 3, False),
           ([(1, i + 1) for i in range(70)], 4, 1, 64, 32, 32, 1, True), ([(40, 41), (2, 1)], 6, 2, 80, 16, 80, 2, False),
           ([(3, 9), (4, 30)], 2, 1, 7, 5, 6, 2, True), ([(200, 260), (0, 0), (1, 64)], 5, 5, 96, 64, 96, 3, False),
           ([(2, 5)] * 130, 2, 2, 64, 16, 64, 2, True)]


@pytest.mark.parametrize("own_positions", [True, False], ids=["positions", "places"])
@pytest.mark.parametrize("norm", ["both", "keys", "none"])
@pytest.mark.parametrize("case", APPENDS, ids=["s%d_h%d_%d_d%d_p%d" % (len(c[0]), *c[1:5]) for c in APPENDS])
def test_append(kern, case, norm, own_positions):
    seqs, heads, kv, d, page, rot, axes, pairs = case
    rng = np.random.default_rng(len(seqs) + d)
    rows, lengths = [r for r, _ in seqs], [n for _, n in seqs]
    starts, total = ref.offsets(rows), sum(rows) + 3
    pages, table = ref.pages_of(lengths, page, rng)
    qkv, q_weight, k_weight = f16(rng, total, heads + 2 * kv, d, std=2.0), f16(rng, d), f16(rng, d)
    packed = dev(qkv)
    q, k, v = packed[:, :heads], packed[:, heads:heads + kv], packed[:, heads + kv:]
    pool = torch.full((2, pages, kv, page, d), SENTINEL, dtype=torch.float16, device="cuda")
    out = torch.full((total, heads, d), SENTINEL, dtype=torch.float16, device="cuda")
    sections = sections_of(rot // 2, axes)
    places = np.concatenate([np.arange(n - r, n) for r, n in seqs])
    positions = rng.integers(0, 3000, (axes, total)) if own_positions else np.tile(np.concatenate([places, np.zeros(3, int)]), (axes, 1))
    rotary = RotaryAxes.new(rot, sections, layout=RotaryLayout.PAIRS if pairs else RotaryLayout.HALVES)
    kern.append_norm_f16(PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1])), PagedBatch(ints(starts), ints(lengths), ints(table)),
                         heads_view(k), heads_view(v), rotary, heads_view(out), heads_view(q), ints(positions) if own_positions else None,
                         HeadNorm(dev(q_weight), EPS) if norm == "both" else None,
                         HeadNorm(dev(k_weight), EPS) if norm != "none" else None)
    n, frequencies = starts[-1], rotary_frequencies(rot)[0]

    def check(got, x, weight):
        y = (step.normed(x, weight, EPS) if weight is not None else x.astype(np.float64)).transpose(1, 0, 2)
        want = step.turned(y, positions[:, :n], axis_of(sections), frequencies, 1.0, pairs)
        assert (np.abs(got.transpose(1, 0, 2) - want) <= step.turned_bound(want, y, rot // 2, 1.0, pairs)).all()
    got = out.cpu().numpy()
    assert (got[n:] == SENTINEL).all()
    check(got[:n], qkv[:n, :heads], q_weight if norm == "both" else None)
    pool = pool.cpu().numpy()
    written = np.zeros((pages, page), bool)
    key, value = np.zeros((n, kv, d)), np.zeros((n, kv, d))
    for i, (r, length) in enumerate(seqs):
        for j in range(r):
            x, row = length - r + j, starts[i] + j
            if x < 0:
                key[row], value[row] = np.nan, qkv[row, heads + kv:]  # (not in the cache)
                continue
            at = table[i, x // page], x % page
            written[at] = True
            key[row], value[row] = pool[0, at[0], :, at[1]], pool[1, at[0], :, at[1]]
    assert np.array_equal(value, qkv[:n, heads + kv:])
    kept = ~np.isnan(key).any((1, 2))
    keep = np.flatnonzero(kept)
    y = step.normed(qkv[:n, heads:heads + kv], k_weight, EPS) if norm != "none" else qkv[:n, heads:heads + kv].astype(np.float64)
    y = y[keep].transpose(1, 0, 2)
    want = step.turned(y, positions[:, :n][:, keep], axis_of(sections), frequencies, 1.0, pairs)
    assert (np.abs(key[keep].transpose(1, 0, 2) - want) <= step.turned_bound(want, y, rot // 2, 1.0, pairs)).all()
    assert (pool.transpose(0, 1, 3, 2, 4)[:, ~written] == SENTINEL).all(), "slots of no row"


def test_append_is_refused_through_python(kern):
    pool = torch.zeros(2, 4, 2, 16, 64, dtype=torch.float16, device="cuda")
    cache = PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1]))
    batch = PagedBatch(ints([0, 3]), ints([3]), ints([[0]]))
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    weight = torch.ones(64, dtype=torch.float16, device="cuda")
    v = heads_view(x)
    two = RotaryAxes.new(64, [16, 16])
    for bad in (lambda: kern.append_norm_f16(cache, batch, v, v, two, positions=ints([0, 1, 2])),
                lambda: kern.append_norm_f16(cache, batch, v, v, two, positions=ints([[0, 1, 2]])),
                lambda: kern.append_norm_f16(cache, batch, v, v, key_norm=HeadNorm(weight[:32])),
                lambda: kern.append_norm_f16(cache, batch, v, v, query=v),
                lambda: kern.append_norm_f16(cache, batch, v, v, key_norm=HeadNorm(weight.cpu())),
                lambda: HeadNorm(weight.float()), lambda: RotaryAxes(two.turns, two.axis, 9),
                lambda: RotaryAxes(two.turns, two.axis[:5], 2)):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: RotaryAxes.new(64, [16, 15]), lambda: RotaryAxes.new(64, [33, -1]), lambda: RotaryAxes.new(64, [32] + [0] * 8),
                lambda: HeadNorm(weight, -1.0), lambda: HeadNorm(weight, float("nan")), lambda: RotaryAxes.new(64, [])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(AdrasteaError):
        kern.norm_rotary_f16(v, v, None, two)


def test_the_tracer_forwards(kern):
    rng = np.random.default_rng(5)
    x, weight = dev(f16(rng, 4, 2, 64)), HeadNorm(dev(f16(rng, 64)))
    a, b = torch.zeros_like(x), torch.zeros_like(x)
    kern.norm_rotary_f16(heads_view(a), heads_view(x), ints([1, 2, 3, 4]), Rotary.new(64), weight)
    MatmulTracer(kern).norm_rotary_f16(heads_view(b), heads_view(x), ints([1, 2, 3, 4]), Rotary.new(64), weight)
    assert torch.equal(a, b) and a.abs().max() > 0

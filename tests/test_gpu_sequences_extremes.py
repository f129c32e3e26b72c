"""Attention over several sequences where numbers are large, small or not finite, through every form of the kernels, against
what the definition gives in 64 bits."""
import numpy as np
import pytest
import torch

from adrastea_amd import PackedBatch, Rotary, _ffi
import sequences_reference as ref
from test_gpu_sequences import CAUSAL, NONE, Packed, Paged, dev, heads_view, kern, shared_keys  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def packed_call(k, p, scale, mask=CAUSAL, temp=1.0):
    p.q_t, p.k_t, p.v_t = dev(p.q), dev(p.k), dev(p.v)
    k.attention_packed_f16(heads_view(p.out_t), heads_view(p.q_t), heads_view(p.k_t), heads_view(p.v_t), p.batch, scale, temp, mask)
    return p.out_t.cpu().numpy()[:p.row_offsets[-1]]


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["high", "low", "rising"])
def test_scores_of_any_size(shared_keys, kind, d, mask):
    """Scores of 2^29 to 2^32 in log2 units, where a step of 32 bits is 2^6 to 2^9: keys differ by 2^20 d / 64 and more, so that
    each row's result is the value of its largest key.  (Scores are exact: 2^14 times d integers of 11 bits.)  `rising`: the
    first keys far below zero, the others near it."""
    p = Packed([(1, 700), (40, 300), (1, 3), (200, 330), (2, 75)], 4, 2, d, seed=d)
    rng = np.random.default_rng(90)
    p.q[:p.row_offsets[-1]] = 2.0 ** 14
    height = np.empty((p.keys, p.kv))
    for i, (_, n) in enumerate(p.seqs):
        for h in range(p.kv):
            some = rng.permutation(np.arange(700, 700 + n))
            height[p.key_offsets[i]:p.key_offsets[i + 1], h] = some
            if kind == "low":
                height[p.key_offsets[i]:p.key_offsets[i + 1], h] *= -1
            elif kind == "rising" and n > 100:
                height[p.key_offsets[i]:p.key_offsets[i + 1], h] = np.sort(some) - (700 + n - 3)
    height[-1] = np.nan
    p.k[:] = height[:, :, None]
    got = packed_call(shared_keys, p, 1.0, mask)
    for i, (r, n) in enumerate(p.seqs):
        for j in range(r):
            end = j + n - r + 1 if mask == CAUSAL else n
            best = p.key_offsets[i] + height[p.key_offsets[i]:p.key_offsets[i] + end].argmax(0)   # of each key head
            want = p.v[best, np.arange(p.kv)].repeat(2, 0).astype(np.float64)
            # (one weight, rounded to fp16 against its unrounded self, and the result's rounding: half a step each, with
            # their product and the 32-bit quotient's 2^-22)
            assert (np.abs(got[p.row_offsets[i] + j] - want) <= np.abs(want) * (2.0 ** -10 + 2.0 ** -20) + 2.0 ** -24).all(), (i, j)


@pytest.mark.parametrize("rows,keys", [(1, 6000), (70, 6000)])
@pytest.mark.parametrize("depth", [18.0, 25.5, 30.0])
def test_many_keys_of_little_weight(shared_keys, rows, keys, depth):
    """One key that outweighs each of the others by 2^depth, and whose value is zero: what is left is the others'."""
    p = Packed([(rows, keys)], 2, 1, 64, seed=7)
    p.q[:rows], p.k[:keys] = 0.0, 0.0
    p.q[:rows, :, 0], p.k[1:keys, :, 0] = 1.0, -1.0
    p.v[0], p.v[1:keys] = 0.0, 1.0
    got = packed_call(shared_keys, p, depth * np.log(2.0)).astype(np.float64)
    others = np.arange(keys - rows, keys, dtype=np.float64) * 2.0 ** -depth     # keys behind the first that each row sees
    want = others / (1.0 + others)
    # Weights below fp16's normal numbers are off by half of their step, 2^-25, where the largest is at least 2^7: 2^-32 of it
    # for each key; above, 2^-11 of each.  32-bit sums of at most 6000 terms: 6000 2^-24 of themselves.  The exponent (5 bits, 32-bit
    # scale): 2^-18.  The result's rounding.
    bound = others * (2.0 ** -11 + 6000 * 2.0 ** -23 + 2.0 ** -18) + np.arange(keys - rows, keys) * 2.0 ** -32 + want * 2.0 ** -11 + 2.0 ** -25
    assert (np.abs(got - want[:, None, None]) <= bound[:, None, None]).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows", [1, 70])
def test_the_largest_values_stay_finite(shared_keys, sign, rows):
    """Values that are all the largest number of fp16: every weighted mean of them is that number.  One weight, in a later
    tile than the row's first key, is a little more than half a step above a number of fp16, and the only large one."""
    keys = 300
    p = Packed([(rows, keys), (60, 62), (140, 300)], 2, 1, 64, seed=8)
    p.v[:] = sign * 65504.0
    p.q[:rows], p.k[:keys] = 0.0, 0.0
    p.q[:rows, :, 0], p.k[1:keys, :, 0], p.k[128, :, 0] = 1.0, -100.0, 1.0
    for mask in (CAUSAL, NONE):
        got = packed_call(shared_keys, p, (7.0 + np.log2(1.0 + 2.0 ** -11 + 2.0 ** -13)) * np.log(2.0), mask).astype(np.float64)
        # (weights rounded to fp16 against their unrounded sum, 2^-11, then the result's rounding)
        assert np.isfinite(got).all() and (np.abs(got - sign * 65504.0) <= 65504.0 * (2.0 ** -10 + 2.0 ** -20)).all()


def test_more_sequences_than_a_launch_has_workgroups(kern):  # noqa: F811
    """Many sequences of one row that sees one key: each row's result is its value, to the bit."""
    n, heads, d = 280000, 32, 8
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = torch.randn(3, n, heads, d, dtype=torch.float16, device="cuda", generator=gen)
    out = torch.zeros_like(q)
    at = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    kern.attention_packed_f16(*(heads_view(t) for t in (out, q, k, v)), PackedBatch(at, at), 0.3)
    assert torch.equal(out, v)


@pytest.mark.parametrize("seen,hidden", [(3, None), (None, 1), (3, 1), (None, 2), (5, 2)])
@pytest.mark.parametrize("rows,keys", [(9, 200), (150, 150), (70, 400)])
def test_no_numbers_before_and_behind_a_row(shared_keys, rows, keys, seen, hidden):
    """Values that are no numbers, in columns of their own: at a key that all rows see, and at one of the last, which only the
    rows behind it see.  Every row has them in exactly these columns, and numbers in the others."""
    p = Packed([(3, 3), (rows, keys), (2, 9)], 4, 2, 128, seed=rows)
    first = p.key_offsets[1]
    gone = np.zeros((rows, p.d), bool)
    clean = p.v.copy()
    if seen is not None:
        p.v[first + keys - rows - (0 if rows == keys else seen), :, 5] = np.inf
        gone[:, 5] = True
    if hidden is not None:
        p.v[first + keys - hidden, :, 70] = -np.inf
        gone[rows - hidden:, 70] = True
    got = packed_call(shared_keys, p, 0.1)
    a = p.row_offsets[1]
    assert (np.isfinite(got[a:a + rows]) == ~gone[:, None, :]).all()
    assert np.isfinite(got[:a]).all() and np.isfinite(got[a + rows:]).all()
    p.v = clean
    want = p.want(0.1, CAUSAL)[:p.row_offsets[-1]]
    got[a:a + rows] = np.where(gone[:, None, :], want[a:a + rows], got[a:a + rows])
    assert ref.close_enough(got, want, np.abs(clean[:-1].astype(np.float64)).max(), keys)


@pytest.mark.parametrize("what", ["key", "value", "score"])
def test_a_prompt_of_no_numbers_takes_no_longer(kern, what):  # noqa: F811
    """Rows that come out as NaN because they see one are not computed twice: 500 times the time when they were."""
    n, heads, kv, d = 4096, 32, 8, 128
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, out = torch.randn(2, n, heads, d, dtype=torch.float16, device="cuda", generator=gen)
    k, v = torch.randn(2, n, kv, d, dtype=torch.float16, device="cuda", generator=gen)
    at = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    batch = PackedBatch(at, at, n, n)

    def fastest():
        times = []
        for _ in range(4):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            kern.attention_packed_f16(*(heads_view(t) for t in (out, q, k, v)), batch, 0.1)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)
    numbers = fastest()
    if what == "score":   # (infinite, of every row)
        q[:, :, 0] = q[:, :, 0].abs() + 1.0
        k[7, :, 0] = float("inf")
    else:
        (k if what == "key" else v)[7] = float("nan")
    assert fastest() < 20 * numbers
    assert out[7:].isnan().all() and out[:7].isfinite().all()


def test_append_of_no_query_heads():
    """With addresses of queries, but no heads of them, the keys and values go to their pages as without."""
    p = Paged([(3, 20), (1, 17)], 4, 2, 64, 16, seed=21)
    key, value = torch.randn(2, p.rows, 2, 64, dtype=torch.float16, device="cuda")
    rotary = Rotary.new(64)
    rows = (1, 128, 64)  # strides of key and value
    written = []
    for q in (None, p.q_t.data_ptr()):
        p.k_t.zero_(), p.v_t.zero_()
        rc = _ffi.lib().adr_append_f16(torch.cuda.current_stream().cuda_stream, p.cache._desc, p.batch._desc, key.data_ptr(),
                                       value.data_ptr(), q, q, None, rotary._desc, 0, p.rows, *rows, *rows, 1, 256, 64, 1, 256, 64)
        assert rc == 0
        written.append((p.k_t.clone(), p.v_t.clone()))
    for without, with_address in zip(*written):
        assert torch.equal(without, with_address) and without.any()


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("rows,keys", [(1, 300), (40, 300), (200, 210)])
def test_infinite_scores(shared_keys, rows, keys, mask):
    """A score of +inf leaves no number in the rows that see it; one of -inf is a key that weighs nothing."""
    p = Packed([(rows, keys), (3, 50)], 4, 2, 64, seed=keys)
    p.q[:, :, 0] = np.abs(p.q[:, :, 0]) + np.float16(1.0)
    at = keys - rows + rows // 2      # (which half of the rows see)
    p.k[at, :, 0], p.k[3, :, 0] = np.inf, -np.inf
    got = packed_call(shared_keys, p, 0.125, mask)
    seen = np.zeros(p.row_offsets[-1], bool)
    seen[rows // 2 if mask == CAUSAL else 0:rows] = True
    assert np.isnan(got[seen]).all() and np.isfinite(got[~seen]).all()
    want = p.want(0.125, mask)[:p.row_offsets[-1]]
    assert ref.close_enough(got[~seen], want[~seen], np.abs(p.v[:-1].astype(np.float64)).max(), keys)

"""The checker of sequences_long.py on the CPU: what a kernel may round passes it, and what it may lose does not."""
import pytest
import torch

from sequences_long import TILE, Definition, marked_keys, matrix_steps, row_steps, sequence

CASES = [(1, 40011, 2, 1, 64), (3, 9001, 2, 2, 128), (2, 100017, 1, 1, 128)]


@pytest.fixture(scope="module", params=CASES, ids=lambda c: "%dx%d" % c[:2])
def case(request):
    rows, n, heads, kv, d = request.param
    q, k, v, scale = sequence(rows, n, heads, kv, d, torch.Generator().manual_seed(n), "cpu")
    return q, k, v, scale, Definition(q, k, v, scale)


def refused(case, got):
    """By the widest of the bounds."""
    whole = case[-1]
    return not whole.agrees(got, row_steps(whole.n))


def test_the_roundings_pass(case):
    """The definition with its weights in fp16, between 2^7 and 2^15, and the sum of the unrounded ones; the result in fp16."""
    q, k, v, scale, whole = case
    heads, rows, _ = q.shape
    kv, n, _ = k.shape
    hidden = torch.arange(n)[None] > torch.arange(n - rows, n)[:, None]
    for top in (7.0, 14.9):
        out = []
        for h in range(heads):
            g = h // (heads // kv)
            s = (q[h].float() @ k[g].float().t() * scale).masked_fill(hidden, -torch.inf)
            w = torch.exp2((s - s.amax(-1, keepdim=True)) * 1.4426950408889634 + top)
            out.append((w.half().float() @ v[g].float() / w.sum(-1, keepdim=True)).half())
        assert whole.agrees(torch.stack(out), matrix_steps(n))


def test_zeros_and_halves_are_refused(case):
    q, k, v, scale, whole = case
    n = whole.n
    first = torch.arange(n) < n // 2
    assert refused(case, torch.zeros_like(whole.out))
    for keep in (first, ~first, torch.arange(n) % 2 == 0, torch.arange(n) >= n // 16):
        assert refused(case, Definition(q, k, v, scale, keep=keep).out)


def test_a_lost_tile_or_page_or_key_is_refused(case):
    q, k, v, scale, whole = case
    n, keys = whole.n, torch.arange(whole.n)
    lost = [keys < TILE, keys < 32, keys >= n - TILE, keys >= (n - 1) // TILE * TILE, keys >= (n - 1) // 32 * 32, keys >= (n - 1) // 16 * 16,
            keys == n - 1, (keys >= n // 2) & (keys < n // 2 + 16), (keys >= TILE) & (keys < 2 * TILE)]
    lost += [keys == x for x in marked_keys(n) if x < n - q.shape[1] + 1]
    for gone in lost:
        assert refused(case, Definition(q, k, v, scale, keep=~gone).out), gone.nonzero().flatten()[:2]


def test_a_tile_counted_twice_is_refused(case):
    """As by two parts that overlap: the marked key's weight doubled."""
    q, k, v, scale, whole = case
    n = whole.n
    for x in (0, n // 2, n - 17):
        kk, vv = torch.cat((k[:, x:x + 1], k), 1), torch.cat((v[:, x:x + 1], v), 1)
        assert refused(case, Definition(q, kk, vv, scale).out)


def test_marked_keys_are_keys():
    for n in (1, 2, 17, 33, 64, 65, 100, 127, 128, 129, 9001):
        at = marked_keys(n)
        assert at == sorted(set(at)) and at[0] == 0 and at[-1] == n - 1
        assert torch.isfinite(sequence(1, n, 2, 1, 64, torch.Generator().manual_seed(n), "cpu")[1]).all()

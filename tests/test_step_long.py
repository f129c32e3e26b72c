"""The bound of step_long.py on the CPU: what a kernel over codes may round passes it, and what it may lose does not."""
import pytest
import torch

from sequences_long import TILE, marked_keys, matrix_steps, sequence
from step_long import Codes, quantised

CASES = [(1, 40011, 2, 1, 64), (3, 9001, 2, 2, 128), (1, 131073, 1, 1, 128)]


@pytest.fixture(scope="module", params=CASES, ids=lambda c: "%dx%d" % c[:2])
def case(request):
    rows, n, heads, kv, d = request.param
    q, k, v, scale = sequence(rows, n, heads, kv, d, torch.Generator().manual_seed(n), "cpu")
    keys, values = quantised(k), quantised(v)
    return q, keys, values, scale, Codes(q, keys, values, scale)


def test_a_code_is_within_half_a_scale():
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(1)).half()
    codes, scales = quantised(x)
    off = ((codes.double() - 127.5) * scales.double()[:, None] - x.double()).abs()
    assert (off <= scales.double()[:, None] / 2 * (1 + 2.0 ** -40)).all()


def test_the_roundings_pass(case):
    """Probabilities times the values' scales in fp16, between 2^6 and 2^15 at the top, times codes in 32 bits."""
    q, keys, values, scale, whole = case
    heads, rows, _ = q.shape
    kv, n, _ = keys[0].shape
    hidden = torch.arange(n)[None] > torch.arange(n - rows, n)[:, None]
    for top in (6.0, 14.5):
        out = []
        for h in range(heads):
            g = h // (heads // kv)
            s = -127.5 * q[h].float().sum(-1, keepdim=True) + q[h].float() @ keys[0][g].float().t()
            s = (s * (keys[1][g].float() * scale * 1.4426950408889634)).masked_fill(hidden, -torch.inf)
            scales = values[1][g].float()
            m = (s + scales.log2()).amax(-1, keepdim=True) - top
            w = torch.exp2(s - m)
            p = (w * scales).half().float()
            out.append(((p @ values[0][g].float() - 127.5 * p.sum(-1, keepdim=True)) / w.sum(-1, keepdim=True)).half())
        assert whole.matrix_agrees(torch.stack(out), matrix_steps(n))


def test_a_lost_half_tile_page_or_key_is_refused(case):
    q, keys, values, scale, whole = case
    n, at = whole.n, torch.arange(whole.n)
    lost = [at < n // 2, at >= n // 2, at < TILE, at < 32, at >= n - TILE, at >= (n - 1) // 32 * 32, at >= (n - 1) // 16 * 16, at == n - 1]
    lost += [at == x for x in marked_keys(n) if x < n - q.shape[1] + 1]
    for gone in lost:
        assert not whole.matrix_agrees(Codes(q, keys, values, scale, keep=~gone).out, matrix_steps(n)), gone.nonzero().flatten()[:2]
    assert not whole.matrix_agrees(torch.zeros_like(whole.out), matrix_steps(n))

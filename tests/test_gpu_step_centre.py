"""Attention over codes of values that lie close to the middle of their format, as where one large value of a head sets its scale, and of queries
with a large common part: what the offset of 127.5 makes sums hold beside them is no more than a rounding or two of the result, over long
contexts as well.

The offset is in the sums of some keys only, 512 of few rows and 1024 of many, and taken off them: 2^-24 of 127.5 times as many weights, over
sqrt(3) in the mean, at each of n / 16 additions at most of independent sign, is 2^-24 * 127.5 * 512 / sqrt(3) * sqrt(n / 16) = 0.00056 sqrt(n)
weights, or twice that.  Values of -7.5 to 7.5 steps (4.6 in the mean) of either sign sum to 4.6 sqrt(n): 1.2 or 2.4 in 10000 of it, where the last
rounding is 2.1: sqrt(1 + 0.33) = 1.16 times that, and of many rows, whose probabilities have 11 bits, sqrt(2 + 1.3) = 1.82.  Left in the
sums of all of n = 24000 keys it is 24000 / 512 times as much.
"""
import numpy as np
import pytest
import torch

from adrastea_amd import GpuKernels, PagedBatch, PagedCacheU8, TensorView, _ffi
from sequences_long import Definition
from step_rounding import times_the_last
from test_gpu_cache_u8 import FORMS, KNOBS, heads_view, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("knob", KNOBS[1:], ids=FORMS[1:])
@pytest.mark.parametrize("rows,n,heads,kv,d", [(4, 24000, 32, 4, 64), (3, 8000, 24, 3, 128), (40, 24011, 8, 2, 64)])
def test_values_around_the_middle(rows, n, heads, kv, d, knob):
    gen = torch.Generator(device="cuda").manual_seed(n + d)
    pages = (n + 15) // 16
    k = torch.randint(90, 166, (pages, kv, 16, d), generator=gen, device="cuda", dtype=torch.uint8)
    v = torch.randint(120, 136, (pages, kv, 16, d), generator=gen, device="cuda", dtype=torch.uint8)
    scales = [(torch.rand(pages, kv, 16, generator=gen, device="cuda") * 0.01 + 0.02).half() for _ in range(2)]
    q = torch.randn(rows, heads, d, generator=gen, device="cuda").half()
    out = torch.zeros_like(q)
    cache = PagedCacheU8(TensorView.of(k), TensorView.of(scales[0]), TensorView.of(v), TensorView.of(scales[1]))
    batch = PagedBatch(ints([0, rows]), ints([n]), ints(np.arange(pages)[None]))
    whole = [((c.double() - 127.5) * s.double()[..., None]).transpose(0, 1).flatten(1, 2)[:, :n] for c, s in ((k, scales[0]), (v, scales[1]))]
    want = Definition(q.transpose(0, 1), *whole, d ** -0.5).out.transpose(0, 1)
    lib = _ffi.lib()
    lib.adr_debug_knob(2, knob)
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES)
    try:
        GpuKernels().attention_paged_u8(heads_view(out), heads_view(q), cache, batch, d ** -0.5)
    finally:
        lib.adr_set_held_workspace_limit(0)
        lib.adr_debug_knob(2, 0)
    assert times_the_last(out.cpu().numpy(), want.cpu().numpy()) < (1.16 * 1.04 if knob <= 4 else 1.82 * 1.04)

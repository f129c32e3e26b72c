"""Attention over codes is no further from the definition than its roundings (step_rounding.py): few rows have none but the last one, many
rows that of the probabilities."""
import numpy as np
import pytest

from adrastea_amd import GpuKernels, _ffi
from step_rounding import ROUNDED, WHOLE, times_the_last
from test_gpu_cache_u8 import CAUSAL, FORMS, KNOBS, Paged, heads_view
from test_gpu_draft_tree import Drafts, random_parents

pytestmark = pytest.mark.gpu


@pytest.fixture(params=FORMS[1:])
def form(request):
    lib = _ffi.lib()
    knob = KNOBS[FORMS.index(request.param)]
    assert lib.adr_debug_knob(2, knob) == 0
    lib.adr_set_held_workspace_limit(_ffi.HELD_WORKSPACE_DEFAULT_BYTES)
    yield WHOLE if knob <= 4 else ROUNDED
    lib.adr_set_held_workspace_limit(0)
    lib.adr_debug_knob(2, 0)


# (sequences of (rows, keys), heads, kv heads, d)
CASES = [([(1, n) for n in range(200, 520, 20)], 8, 2, 64), ([(1, 300 + n) for n in range(12)], 16, 1, 128), ([(5, 411), (16, 300), (7, 350)], 6, 2, 96),
         ([(1, 333)] * 13, 8, 8, 80)]


@pytest.mark.parametrize("case", CASES, ids=["h%d_%d_d%d" % c[1:] for c in CASES])
def test_rows(form, case):
    p = Paged(*case, 16, seed=case[3])
    GpuKernels().attention_paged_u8(heads_view(p.out_t), heads_view(p.q_t), p.cache.handle, p.batch, case[3] ** -0.5)
    n = p.row_offsets[-1]
    assert n * case[1] * case[3] > 6000
    assert times_the_last(p.out_t.cpu().numpy()[:n], p.want(case[3] ** -0.5, CAUSAL)[:n]) < form


@pytest.mark.parametrize("rows,heads,kv,d", [([5, 3, 9], 8, 2, 64), ([30], 4, 1, 128)])
def test_drafts(form, rows, heads, kv, d):
    rng = np.random.default_rng(d)
    t = Drafts([random_parents(r, rng) for r in rows], [400 + 31 * i for i in range(len(rows))], heads, kv, d, 16, 8, seed=d)
    n = t.starts[-1]
    assert n * heads * d > 6000
    assert times_the_last(t.run(GpuKernels(), d ** -0.5)[:n], t.want(d ** -0.5)[:n]) < form

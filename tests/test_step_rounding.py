"""What the bounds of step_rounding.py let pass and what they refuse, on the CPU."""
import numpy as np
import pytest

import step_reference as step
from step_rounding import ROUNDED, WHOLE, rounded, times_the_last


@pytest.mark.parametrize("d,top", [(64, 7.0), (128, 9.3), (64, 14.0)])
def test_what_passes(d, top):
    rng = np.random.default_rng(d)
    got = {w: [] for w in ("two halves", "half", "values too", "values")}
    want = []
    for _ in range(16):
        n, rows = 300, 16
        q = rng.standard_normal((rows, d)).astype(np.float16)
        codes = [np.clip(rng.standard_normal((n, d)) * 40 + 127.5, 0, 255).astype(np.uint8) for _ in range(2)]
        scales = [rng.uniform(0.01, 0.03, n).astype(np.float16) for _ in range(2)]
        seen = step.causal(rows, n)
        k, v = (step.value_of(codes[t], scales[t])[None] for t in (0, 1))
        want.append(step.attention(q[None], k, v, d ** -0.5, 1.0, seen)[0])
        for what, w, values in (("two halves", "two halves", False), ("half", "half", False), ("values too", "half", True), ("values", "two halves", True)):
            got[what].append(rounded(q, codes, scales, d ** -0.5, seen, w, values, top))
    times = {what: times_the_last(np.stack(x), np.stack(want)) for what, x in got.items()}
    assert times["two halves"] < 1.005
    assert WHOLE < 1.25 < times["half"] < ROUNDED and WHOLE < times["values"]
    assert times["values too"] > ROUNDED

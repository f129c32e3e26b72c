"""Refusals of the heads' norms with rotation, the cache in 8 bits and drafted trees; no device needed."""
import math

import pytest
import torch

from adrastea_amd import DraftTree, HeadNorm, RotaryAxes, _ffi

P = 4096  # an aligned address that is never read: every call here is refused, or has nothing to do
SHAPE, ENUM, NULL, LAYOUT = (_ffi.ADR_EINVAL_SHAPE, _ffi.ADR_EINVAL_ENUM, _ffi.ADR_ENULL, _ffi.ADR_EUNSUPPORTED_LAYOUT)
THREE = (1, 64, 320)


def cache(**change):
    c = dict(key=P, value=P, pages=4, kv_heads=2, page_size=16, d=64)
    c.update(change)
    return _ffi.PagedCacheDesc(c["key"], c["value"], c["pages"], c["kv_heads"], c["page_size"], c["d"], *((1, 64, 1024, 2048) * 2))


def codes(**change):
    c = dict(key=P, key_scale=P, value=P, value_scale=P, pages=4, kv_heads=2, page_size=16, d=64)
    c.update(change)
    return _ffi.PagedCacheU8Desc(*c.values(), *((1, 64, 1024, 2048) * 2), *((1, 16, 32) * 2))


def batch(**change):
    b = dict(row_offsets=P, lengths=P, table=P, sequences=3, table_width=2, table_pitch=2)
    b.update(change)
    return _ffi.PagedBatchDesc(*b.values(), 0, 0)


def axes(**change):
    r = dict(turns=P, axis=P, dims=64, layout=0, magnitude=1.0, axes=2)
    r.update(change)
    return _ffi.RotaryAxesDesc(*r.values())


def norm(weight=P, eps=1e-6):
    return _ffi.HeadNormDesc(weight, eps)


AXES = [(dict(dims=63), SHAPE), (dict(dims=66), SHAPE), (dict(dims=-2), SHAPE), (dict(layout=2), ENUM), (dict(axes=0), SHAPE),
        (dict(axes=9), SHAPE), (dict(axes=-1), SHAPE), (dict(turns=None), NULL), (dict(turns=P + 4), LAYOUT), (dict(axis=P + 2), LAYOUT)]
NORMS = [norm(eps=-1e-6), norm(eps=math.nan), norm(eps=math.inf)]


def test_norm_and_rotation_refuse():
    def call(r=None, n=None, out=P, x=P, positions=P, pitch=5, heads=2, rows=5, d=64):
        return _ffi.lib().adr_norm_rotary_f16(None, out, x, positions, pitch, r or axes(), n or norm(), heads, rows, d, *THREE, *THREE)
    for kw, code in AXES:
        assert call(r=axes(**kw)) == code, kw
    for n in NORMS:
        assert call(n=n) == SHAPE
    for kw, code in [(dict(pitch=4), SHAPE), (dict(rows=-1), SHAPE), (dict(heads=-1), SHAPE), (dict(d=-1), SHAPE), (dict(out=None), NULL),
                     (dict(x=None), NULL), (dict(positions=None), NULL), (dict(positions=P + 1), LAYOUT),
                     (dict(heads=1 << 16, rows=1 << 16, pitch=1 << 16), SHAPE)]:
        assert call(**kw) == code, kw
    assert call(rows=0, out=None) == 0 and call(heads=0, x=None) == 0


@pytest.mark.parametrize("name,make", [("adr_append_norm_f16", cache), ("adr_append_u8", codes)])
def test_append_refuses(name, make):
    def call(c=None, b=None, key=P, value=P, qo=P, q=P, positions=P, pitch=5, r=None, qn=None, kn=None, heads=4, rows=5):
        return getattr(_ffi.lib(), name)(None, c or make(), b or batch(), key, value, qo, q, positions, pitch, r or axes(), qn or norm(),
                                         kn or norm(), heads, rows, *(THREE * 4))
    for kw, code in AXES:
        assert call(r=axes(**kw)) == code, kw
    for n in NORMS:
        assert call(qn=n) == SHAPE and call(kn=n) == SHAPE
    for kw, code in [(dict(key=None), NULL), (dict(value=None), NULL), (dict(q=None), NULL), (dict(qo=None), NULL), (dict(heads=3), SHAPE),
                     (dict(rows=-1), SHAPE), (dict(pitch=4), SHAPE), (dict(c=make(key=None)), NULL), (dict(c=make(value=None)), NULL),
                     (dict(c=make(kv_heads=0)), SHAPE), (dict(c=make(page_size=0)), SHAPE), (dict(c=make(pages=-1)), SHAPE),
                     (dict(b=batch(lengths=None)), NULL), (dict(b=batch(row_offsets=None)), NULL), (dict(b=batch(table=None)), NULL),
                     (dict(b=batch(table_pitch=0)), SHAPE), (dict(b=batch(table=P + 1)), LAYOUT), (dict(b=batch(sequences=-1)), SHAPE),
                     (dict(positions=P + 2), LAYOUT)]:
        assert call(**kw) == code, kw
    if make is codes:
        assert call(c=codes(key_scale=None)) == NULL and call(c=codes(value_scale=None)) == NULL
    assert call(rows=0, key=None) == 0 and call(b=batch(sequences=0)) == 0


def test_read_refuses():
    def call(c=None, b=None, key=P, value=P, rows=5):
        return _ffi.lib().adr_read_u8(None, key, value, c or codes(), b or batch(), rows, *THREE, *THREE)
    for kw, code in [(dict(key=None), NULL), (dict(value=None), NULL), (dict(rows=-1), SHAPE), (dict(c=codes(key_scale=None)), NULL),
                     (dict(c=codes(value=None)), NULL), (dict(c=codes(kv_heads=-1)), SHAPE), (dict(c=codes(page_size=-1)), SHAPE),
                     (dict(b=batch(table_width=-1)), SHAPE), (dict(b=batch(lengths=P + 2)), LAYOUT), (dict(b=batch(table=None)), NULL)]:
        assert call(**kw) == code, kw
    assert call(rows=0, key=None) == 0 and call(c=codes(kv_heads=0), value=None) == 0


ATTENTION = [
    (dict(rows=-1), SHAPE), (dict(heads=-4), SHAPE), (dict(heads=3), SHAPE), (dict(out=None), NULL), (dict(q=None), NULL),
    (dict(b=batch(sequences=-1)), SHAPE), (dict(b=batch(table_width=-1)), SHAPE), (dict(b=batch(table_pitch=1)), SHAPE),
    (dict(b=batch(row_offsets=None)), NULL), (dict(b=batch(lengths=None)), NULL), (dict(b=batch(table=None)), NULL),
    (dict(b=batch(lengths=P + 2)), LAYOUT), (dict(scale=0.0), LAYOUT), (dict(scale=-1.0), LAYOUT), (dict(scale=math.nan), LAYOUT),
    (dict(temp=0.0), LAYOUT), (dict(temp=math.nan), LAYOUT), (dict(scale=math.inf), LAYOUT), (dict(scale=1e30), LAYOUT)]


def test_attention_over_codes_refuses():
    def call(c=None, b=None, heads=4, rows=5, scale=0.1, temp=1.0, mask=1, out=P, q=P):
        return _ffi.lib().adr_attention_paged_u8(None, out, q, c or codes(), b or batch(), heads, rows, *THREE, *THREE, scale, temp, mask)
    for kw, code in ATTENTION + [(dict(mask=2), ENUM), (dict(c=codes(d=257)), LAYOUT), (dict(c=codes(key_scale=None)), NULL),
                                 (dict(c=codes(value_scale=None)), NULL), (dict(c=codes(key=None)), NULL), (dict(c=codes(pages=-1)), SHAPE),
                                 (dict(c=codes(page_size=0)), SHAPE), (dict(c=codes(d=-1)), SHAPE)]:
        assert call(**kw) == code, kw
    for kw in (dict(rows=0), dict(heads=0), dict(b=batch(sequences=0)), dict(c=codes(d=0))):
        assert call(out=None, q=None, **kw) == 0, kw


@pytest.mark.parametrize("suffix,make", [("f16", cache), ("u8", codes)])
def test_trees_refuse(suffix, make):
    lib = _ffi.lib()

    def tree(bits=P, words=1, pitch=1):
        return _ffi.DraftTreeDesc(bits, words, pitch)

    def call(c=None, b=None, t=None, heads=4, rows=5, scale=0.1, temp=1.0, out=P, q=P):
        return getattr(lib, "adr_attention_tree_" + suffix)(None, out, q, c or make(), b or batch(), t or tree(), heads, rows, *THREE, *THREE,
                                                            scale, temp)
    for kw, code in ATTENTION + [(dict(t=tree(words=-1)), SHAPE), (dict(t=tree(words=2)), SHAPE), (dict(t=tree(bits=None)), NULL),
                                 (dict(t=tree(bits=P + 1)), LAYOUT)]:
        assert call(**kw) == code, kw
    assert call(rows=0, out=None) == 0
    args = (None, P, P, make(), batch(), tree(), 4, 5, *THREE, *THREE, 0.1, 1.0)
    ws = getattr(lib, "adr_attention_tree_" + suffix + "_ws")
    assert ws(*args, None, 64) == NULL and ws(*args, P, -1) == NULL and ws(*args, P + 8, 64) == SHAPE


def test_workspace_arguments_are_checked():
    lib = _ffi.lib()
    args = (None, P, P, codes(), batch(), 4, 5, *THREE, *THREE, 0.1, 1.0, 1)
    assert lib.adr_attention_paged_u8_ws(*args, None, 64) == NULL
    assert lib.adr_attention_paged_u8_ws(*args, P, -1) == NULL
    assert lib.adr_attention_paged_u8_ws(*args, P + 8, 64) == SHAPE
    assert lib.adr_attention_paged_u8_workspace_bytes(codes(), batch(), 3, 5) == SHAPE
    assert lib.adr_attention_paged_u8_workspace_bytes(codes(), batch(), 4, 0) == 0
    for heads, rows, sequences, width in ((32, 1, 1, 500), (32, 16, 16, 250), (32, 256, 1, 600), (8, 5, 3, 2)):
        sizes = dict(sequences=sequences, table_width=width, table_pitch=width)
        want = lib.adr_attention_paged_u8_workspace_bytes(codes(pages=10000), batch(**sizes), heads, rows)
        none = dict(key=None, key_scale=None, value=None, value_scale=None)
        unknown = batch(row_offsets=None, lengths=None, table=None, **sizes)
        assert want >= 0 and lib.adr_attention_paged_u8_workspace_bytes(codes(pages=10000, **none), unknown, heads, rows) == want


def test_workspaces_of_trees():
    lib = _ffi.lib()
    for call, c in ((lib.adr_attention_tree_f16_workspace_bytes, cache), (lib.adr_attention_tree_u8_workspace_bytes, codes)):
        assert call(c(), batch(), 3, 5) == SHAPE and call(c(kv_heads=-2), batch(), 4, 5) == SHAPE and call(c(), batch(), 4, 0) == 0
        wide = dict(sequences=1, table_width=2000, table_pitch=2000)
        assert call(c(pages=10000), batch(**wide), 32, 8) > 0          # (a long context's keys are shared)
        assert call(c(pages=10000), batch(sequences=1, table_width=1, table_pitch=1), 32, 8) == 0


def test_handles_check_types():
    with pytest.raises(AssertionError):
        HeadNorm(torch.ones(4))
    with pytest.raises(AssertionError):
        HeadNorm(torch.ones(4, 4, dtype=torch.float16))
    with pytest.raises(AssertionError):
        HeadNorm(torch.ones(8, dtype=torch.float16)[::2])
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            HeadNorm(torch.ones(4, dtype=torch.float16), eps)
    turns = torch.zeros(4, dtype=torch.float64)
    with pytest.raises(AssertionError):
        RotaryAxes(turns, torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(AssertionError):
        RotaryAxes(turns, torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(AssertionError):
        RotaryAxes(turns, torch.zeros(4, dtype=torch.int32), 0)
    for sections in ([2, 1], [5, -1], []):
        with pytest.raises(ValueError):
            RotaryAxes.new(8, sections)
    with pytest.raises(AssertionError):
        DraftTree(torch.zeros(4, 2, dtype=torch.int64))
    for parents in ([[0]], [[-1, 1]], [[-1, -2]]):
        with pytest.raises(ValueError):
            DraftTree.of(parents)

"""Refusals of the operators over several sequences, and the frequencies of rotary scalings; no device needed."""
import math

import pytest
import torch

from adrastea_amd import RotaryScaling, _ffi, rotary_frequencies
from sequences_reference import yarn_reference

P = 4096  # an aligned address that is never read: every call here is refused, or has nothing to do


def cache(**change):
    c = dict(key=P, value=P, pages=4, kv_heads=2, page_size=16, d=64, kx=1, ky=64, kz=1024, kp=2048)
    c.update(change)
    s = (c["kx"], c["ky"], c["kz"], c["kp"])
    return _ffi.PagedCacheDesc(c["key"], c["value"], c["pages"], c["kv_heads"], c["page_size"], c["d"], *s, *s)


def batch(**change):
    b = dict(row_offsets=P, lengths=P, table=P, sequences=3, table_width=2, table_pitch=2)
    b.update(change)
    return _ffi.PagedBatchDesc(b["row_offsets"], b["lengths"], b["table"], b["sequences"], b["table_width"],
                               b["table_pitch"], 0, 0)


def paged(c=None, b=None, heads=4, rows=5, scale=0.1, temp=1.0, mask=1, out=P, q=P):
    return _ffi.lib().adr_attention_paged_f16(None, out, q, c or cache(), b or batch(), heads, rows, 1, 64, 320, 1, 64, 320,
                                              scale, temp, mask)


SHAPE, ENUM, NULL, LAYOUT = (_ffi.ADR_EINVAL_SHAPE, _ffi.ADR_EINVAL_ENUM, _ffi.ADR_ENULL, _ffi.ADR_EUNSUPPORTED_LAYOUT)


def test_paged_attention_refuses():
    for kw, code in [
            (dict(rows=-1), SHAPE), (dict(heads=-4), SHAPE), (dict(heads=3), SHAPE), (dict(c=cache(kv_heads=0)), SHAPE),
            (dict(c=cache(kv_heads=-1)), SHAPE), (dict(c=cache(pages=-1)), SHAPE), (dict(c=cache(page_size=0)), SHAPE),
            (dict(c=cache(page_size=-16)), SHAPE), (dict(c=cache(d=-1)), SHAPE), (dict(b=batch(sequences=-1)), SHAPE),
            (dict(b=batch(table_width=-1)), SHAPE), (dict(b=batch(table_pitch=1)), SHAPE),
            (dict(heads=1 << 20, c=cache(kv_heads=1), rows=1 << 12), SHAPE), (dict(mask=2), ENUM),
            (dict(out=None), NULL), (dict(q=None), NULL), (dict(c=cache(key=None)), NULL), (dict(c=cache(value=None)), NULL),
            (dict(b=batch(row_offsets=None)), NULL), (dict(b=batch(lengths=None)), NULL), (dict(b=batch(table=None)), NULL),
            (dict(b=batch(lengths=P + 2)), LAYOUT), (dict(c=cache(d=257)), LAYOUT), (dict(scale=0.0), LAYOUT),
            (dict(scale=-1.0), LAYOUT), (dict(scale=math.nan), LAYOUT), (dict(temp=0.0), LAYOUT),
            (dict(temp=math.nan), LAYOUT), (dict(scale=math.inf), LAYOUT)]:
        assert paged(**kw) == code, kw
    for kw in (dict(rows=0), dict(heads=0), dict(b=batch(sequences=0)), dict(c=cache(d=0))):
        assert paged(out=None, q=None, **kw) == 0, kw  # nothing to do, whatever the pointers


def test_workspace_arguments_are_checked():
    lib = _ffi.lib()
    args = (None, P, P, cache(), batch(), 4, 5, 1, 64, 320, 1, 64, 320, 0.1, 1.0, 1)
    assert lib.adr_attention_paged_f16_ws(*args, None, 64) == NULL
    assert lib.adr_attention_paged_f16_ws(*args, P, -1) == NULL
    assert lib.adr_attention_paged_f16_ws(*args, P + 8, 64) == SHAPE
    assert lib.adr_attention_paged_f16_workspace_bytes(cache(), batch(), 4, 5) >= 0
    assert lib.adr_attention_paged_f16_workspace_bytes(cache(), batch(), 3, 5) == SHAPE
    assert lib.adr_attention_paged_f16_workspace_bytes(cache(), batch(), 4, 0) == 0
    packed = _ffi.PackedBatchDesc(P, P, 3, 0, 0)
    assert lib.adr_attention_packed_f16_workspace_bytes(packed, 4, 2, 50, 50, 64) >= 0
    assert lib.adr_attention_packed_f16_workspace_bytes(packed, 4, 2, 50, -1, 64) == SHAPE


def packed(heads=4, kv=2, rows=5, keys=5, d=64, scale=0.1, temp=1.0, mask=1, out=P, q=P, k=P, v=P, ro=P, ko=P, sequences=2):
    b = _ffi.PackedBatchDesc(ro, ko, sequences, 0, 0)
    return _ffi.lib().adr_attention_packed_f16(None, out, q, k, v, b, heads, kv, rows, keys, d, *((1, 64, 320) * 4), scale,
                                               temp, mask)


def test_packed_attention_refuses():
    for kw, code in [(dict(keys=-1), SHAPE), (dict(heads=5), SHAPE), (dict(kv=0), SHAPE), (dict(sequences=-2), SHAPE),
                     (dict(mask=7), ENUM), (dict(k=None), NULL), (dict(v=None), NULL), (dict(ko=None), NULL),
                     (dict(ro=None), NULL), (dict(out=None), NULL), (dict(d=300), LAYOUT), (dict(ko=P + 1), LAYOUT),
                     (dict(temp=-1.0), LAYOUT)]:
        assert packed(**kw) == code, kw
    assert packed(rows=0, out=None) == 0 and packed(sequences=0, out=None) == 0


def test_rotary_and_append_refuse():
    lib = _ffi.lib()

    def rot(dims=64, layout=0, turns=P, heads=2, rows=3, d=64, out=P, x=P, pos=P):
        r = _ffi.RotaryDesc(turns, dims, layout, 1.0)
        return lib.adr_rotary_f16(None, out, x, pos, r, heads, rows, d, 1, 64, 192, 1, 64, 192)
    for kw, code in [(dict(dims=63), SHAPE), (dict(dims=66), SHAPE), (dict(dims=-2), SHAPE), (dict(d=2048, dims=514), SHAPE),
                     (dict(layout=2), ENUM), (dict(turns=None), NULL), (dict(pos=None), NULL), (dict(out=None), NULL),
                     (dict(x=None), NULL), (dict(rows=-1), SHAPE), (dict(pos=P + 2), LAYOUT), (dict(turns=P + 4), LAYOUT)]:
        assert rot(**kw) == code, kw
    assert rot(rows=0, out=None) == 0 and rot(heads=0, out=None) == 0

    def append(c=None, b=None, key=P, value=P, qo=P, q=P, dims=64, heads=4, rows=5):
        r = _ffi.RotaryDesc(P, dims, 0, 1.0)
        return lib.adr_append_f16(None, c or cache(), b or batch(), key, value, qo, q, None, r, heads, rows,
                                  *((1, 64, 320) * 4))
    for kw, code in [(dict(key=None), NULL), (dict(value=None), NULL), (dict(q=None), NULL), (dict(qo=None), NULL),
                     (dict(heads=3), SHAPE), (dict(dims=80), SHAPE), (dict(rows=-1), SHAPE), (dict(c=cache(key=None)), NULL),
                     (dict(b=batch(lengths=None)), NULL), (dict(b=batch(table_pitch=0)), SHAPE),
                     (dict(c=cache(page_size=0)), SHAPE), (dict(b=batch(table=P + 1)), LAYOUT)]:
        assert append(**kw) == code, kw
    assert append(rows=0, key=None) == 0


def test_plain_frequencies():
    f, magnitude = rotary_frequencies(8, 10000.0)
    assert magnitude == 1.0
    assert f == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-15)
    assert rotary_frequencies(0) == ([], 1.0)
    assert rotary_frequencies(2)[0] == [1.0]


def test_scaled_frequencies():
    base, dims = 500000.0, 64
    plain, _ = rotary_frequencies(dims, base)
    assert rotary_frequencies(dims, base, RotaryScaling.Linear(4.0))[0] == pytest.approx([x / 4 for x in plain], rel=1e-15)
    grown, _ = rotary_frequencies(dims, base, RotaryScaling.Base(4.0))
    assert grown[0] == plain[0] and grown[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    waves, magnitude = rotary_frequencies(dims, base, RotaryScaling.Wavelength(8.0, 1.0, 4.0, 8192))
    assert magnitude == 1.0
    for w, x in zip(waves, plain):
        length = 2 * math.pi / x
        if length < 8192 / 4.0:
            assert w == x
        elif length > 8192 / 1.0:
            assert w == pytest.approx(x / 8, rel=1e-15)
        else:
            blend = (8192 / length - 1.0) / (4.0 - 1.0)
            assert w == pytest.approx((1 - blend) * x / 8 + blend * x, rel=1e-14)
    yarn, magnitude = rotary_frequencies(dims, base, RotaryScaling.Yarn(16.0, 4096))
    assert yarn == pytest.approx(yarn_reference(dims, base, 16.0, 4096, 32.0, 1.0), rel=1e-14)
    assert magnitude == pytest.approx(0.1 * math.log(16.0) + 1)
    assert rotary_frequencies(dims, base, RotaryScaling.Yarn(16.0, 4096, magnitude=1.0))[1] == 1.0
    assert rotary_frequencies(dims, base, RotaryScaling.Yarn(1.0, 4096)) == (pytest.approx(plain, rel=1e-15), 1.0)


def test_scalings_that_make_no_sense_are_refused():
    for bad in (lambda: rotary_frequencies(7), lambda: rotary_frequencies(-2), lambda: rotary_frequencies(8, 0.0),
                lambda: rotary_frequencies(8, scaling=RotaryScaling.Linear(0.0)),
                lambda: rotary_frequencies(8, scaling=RotaryScaling.Wavelength(8.0, 4.0, 4.0, 100)),
                lambda: rotary_frequencies(8, scaling=RotaryScaling("cubic", (1.0,)))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("scale,temp", [(1.0, math.inf), (1e-20, 1e20), (2.0 ** -126, 1.5), (2.0 ** -140, 1.0), (2.0 ** 59, 1.0), (1e29, 1.0),
                                        (2.0 ** 30, 2.0 ** -30), (1e38, 1e-38), (math.inf, math.inf)])
def test_a_factor_of_the_scores_out_of_range(scale, temp):
    """Where scale / temp is no normal number in 32 bits, hidden scores would not stay -inf; where it is huge, finite ones would
    pass the kernels' mark for none."""
    assert paged(scale=scale, temp=temp) == LAYOUT and packed(scale=scale, temp=temp) == LAYOUT


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not real")
@pytest.mark.parametrize("scale,temp", [(2.0 ** -126, 1.0), (2.0 ** 58, 1.0), (1.0, 1e30), (2.0 ** -149, 2.0 ** -60)])
def test_the_ends_of_its_range(scale, temp):
    """Accepted as far as the arguments go: without a GPU, what is refused is the device."""
    assert paged(scale=scale, temp=temp) not in (0, LAYOUT) and packed(scale=scale, temp=temp) not in (0, LAYOUT)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not real")
def test_append_of_no_query_heads_is_no_call_of_nothing():
    """Keys and values are there to be written: without a GPU, that is an error of the device and not a success."""
    lib = _ffi.lib()
    r = _ffi.RotaryDesc(P, 64, 0, 1.0)
    strides = (1, 64, 320) * 4
    without = lib.adr_append_f16(None, cache(), batch(), P, P, None, None, None, r, 0, 5, *strides)
    assert without not in (0, SHAPE, NULL) and lib.adr_append_f16(None, cache(), batch(), P, P, P, P, None, r, 0, 5, *strides) == without
    assert lib.adr_append_f16(None, cache(kv_heads=0), batch(), P, P, P, P, None, r, 0, 5, *strides) == 0


def test_workspace_bytes_before_there_is_a_table():
    """Sizes are enough to ask: the addresses of a batch that is yet to be allocated change nothing."""
    lib = _ffi.lib()
    for heads, rows, sequences, width in ((32, 1, 1, 500), (32, 16, 16, 250), (32, 256, 1, 600), (8, 5, 3, 2)):
        c = cache(pages=10000, kv_heads=8 if heads == 32 else 2, d=128, ky=128, kz=2048, kp=16384)
        sizes = dict(sequences=sequences, table_width=width, table_pitch=width)
        want = lib.adr_attention_paged_f16_workspace_bytes(c, batch(**sizes), heads, rows)
        unknown = batch(row_offsets=None, lengths=None, table=None, **sizes)
        assert lib.adr_attention_paged_f16_workspace_bytes(c, unknown, heads, rows) == want
        assert want > 0 or heads == 8

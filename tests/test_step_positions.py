"""Positions that are the same on every axis (a pitch of 0, what expand makes): taken by the C interface and by both ways from Python; no
device needed."""
import pytest
import torch

from adrastea_amd import _ffi
from test_native_step import batch, both, cache, codes, norm, recorders, rotary, rows  # noqa: F401
from test_step_host import NULL, P, SHAPE, THREE, axes
from test_step_host import batch as batch_desc, cache as cache_desc, codes as codes_desc, norm as norm_desc


def test_a_pitch_of_0_is_no_refusal():
    """A call that is refused for its missing output, which is looked at behind the pitch."""
    lib = _ffi.lib()

    def turn(pitch, out=None):
        return lib.adr_norm_rotary_f16(None, out, P, P, pitch, axes(), norm_desc(), 2, 5, 64, *THREE, *THREE)
    assert turn(0) == NULL and turn(5) == NULL and turn(4) == SHAPE and turn(1) == SHAPE and turn(-1) == SHAPE
    for name, make in (("adr_append_norm_f16", cache_desc), ("adr_append_u8", codes_desc)):
        def append(pitch):
            return getattr(lib, name)(None, make(), batch_desc(), None, P, P, P, P, pitch, axes(), norm_desc(), norm_desc(), 4, 5, *(THREE * 4))
        assert append(0) == NULL and append(5) == NULL and append(4) == SHAPE and append(-1) == SHAPE


@pytest.mark.parametrize("n", [9, 1])
def test_both_ways_pass_a_pitch_of_0(both, n):  # noqa: F811
    shared = torch.zeros(n, dtype=torch.int32).expand(3, -1)
    assert shared.stride(0) == 0
    k, q, o = rows(2, n, 64), rows(8, n, 64), rows(8, n, 64)
    for name, *args in (("norm_rotary_f16", o, q, shared, rotary(3), norm()),
                        ("append_norm_f16", cache(), batch(), k, k, rotary(3), o, q, shared, norm(), None),
                        ("append_u8", codes(), batch(), k, k, rotary(3), o, q, shared, norm(), norm())):
        native, general = both(name, *args)
        assert native == general and native is not None

"""Workgroups that share the keys of few rows over codes are no more than a card of 256 units holds at once: with equal stretches, those that
start when others end are a second round.  Told by the workspace, which has two slots of 16 rows and a seam for each; no device needed."""
import pytest

from adrastea_amd import _ffi
from test_step_host import P

SEAM = 32          # bytes: parts, slot, block, and a sequence's five numbers
# of heads up to 64: three wavefronts a SIMD by their registers, two to a workgroup; beyond: 38912 bytes of 160 KiB
AT_ONCE = {64: 6, 128: 4}


@pytest.mark.parametrize("d", [64, 128, 48, 80])
@pytest.mark.parametrize("heads,kv", [(32, 4), (20, 20), (16, 1), (12, 12)])
def test_stretches_are_one_round(heads, kv, d):
    width = 4000  # pages of 16: 64000 keys
    wide = 64 if d <= 64 else 128
    strides = (1, 128, 16 * 128, kv * 16 * 128) * 2
    codes = _ffi.PagedCacheU8Desc(P, P, P, P, 1 << 20, kv, 16, d, *strides, *((1, 16, kv * 16) * 2))
    batch = _ffi.PagedBatchDesc(P, P, P, 8, width, width, 1, 0)  # (eight sequences of one row: all of a sequence's rows in a block)
    nbytes = _ffi.lib().adr_attention_paged_u8_workspace_bytes(codes, batch, heads, 8)
    slots = nbytes / (2 * 16 * (wide * 4 + 8) + SEAM)
    assert slots == int(slots) and 256 <= slots <= 256 * AT_ONCE[wide]

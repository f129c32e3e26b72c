"""Positions that are expanded over the axes give the bits of their copy, through both ways from Python."""
import numpy as np
import pytest
import torch

from adrastea_amd import GpuKernels, HeadNorm, PagedBatch, PagedCache, RotaryAxes, TensorView, kernels
from test_gpu_cache_u8 import Cache, dev, f16, heads_view, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("way", ["native", "general"])
@pytest.mark.parametrize("d", [64, 20], ids=["d64", "any layout"])
@pytest.mark.parametrize("rows", [37, 1])
def test_expanded_positions(rows, d, way, monkeypatch):
    kern = GpuKernels()
    if way == "general":
        monkeypatch.setattr(kernels, "_native", None)
    rng = np.random.default_rng(rows + d)
    qkv, weight = dev(f16(rng, rows, 8, d)), HeadNorm(dev(f16(rng, d)), 1e-6)
    q, k, v = (heads_view(t) for t in (qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]))
    one = ints(rng.integers(0, 100000, rows))
    rotary = RotaryAxes.new(d, [d // 4, d // 8, d // 2 - d // 4 - d // 8])

    def run(positions):
        codes = Cache([rows], 2, d, 16, np.random.default_rng(1))
        pool = torch.zeros(2, *codes.handle.key.storage.shape, dtype=torch.float16, device="cuda")
        batch = PagedBatch(ints([0, rows]), ints([rows]), ints(codes.table))
        outs = [torch.zeros(rows, 4, d, dtype=torch.float16, device="cuda") for _ in range(3)]
        kern.norm_rotary_f16(heads_view(outs[0]), q, positions, rotary, weight)
        kern.append_norm_f16(PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1])), batch, k, v, rotary, heads_view(outs[1]), q, positions,
                             weight, weight)
        kern.append_u8(codes.handle, batch, k, v, rotary, heads_view(outs[2]), q, positions, weight, weight)
        return [*outs, pool, codes.handle.key.storage, codes.handle.key_scale.storage]
    want, got = run(one.expand(3, -1).contiguous()), run(one.expand(3, -1))
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b)
        assert a.float().nan_to_num(0.0).abs().max() > 0

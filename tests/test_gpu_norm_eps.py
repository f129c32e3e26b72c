"""The smallest eps of a head's norm: a head of zeros stays one under any that is positive, below the normal numbers of 32 bits as well."""
import numpy as np
import pytest
import torch

from adrastea_amd import GpuKernels, HeadNorm, PagedBatch, PagedCache, TensorView
from test_gpu_cache_u8 import Cache, dev, heads_view, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 7], ids=["d64", "any layout"])
@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1.1e-38, 1e-37])
def test_heads_of_zeros(eps, d):
    kern, x = GpuKernels(), np.zeros((3, 4, d), np.float16)
    x[1], x[2, 1] = 2.0 ** -24, 1.0            # (the smallest numbers of fp16, and some)
    want = np.sign(x)
    q, weight = dev(x), HeadNorm(torch.ones(d, dtype=torch.float16, device="cuda"), eps)
    outs = [torch.full((3, 4, d), 9.0, dtype=torch.float16, device="cuda") for _ in range(3)]
    kern.norm_rotary_f16(heads_view(outs[0]), heads_view(q), norm=weight)
    codes = Cache([3], 2, d, 16, np.random.default_rng(0))
    batch = PagedBatch(ints([0, 3]), ints([3]), ints(codes.table))
    pool = torch.zeros(2, *codes.codes.shape[1:], dtype=torch.float16, device="cuda")
    args = heads_view(q[:, :2]), heads_view(q[:, 2:])
    kern.append_norm_f16(PagedCache(TensorView.of(pool[0]), TensorView.of(pool[1])), batch, *args, None, heads_view(outs[1]), heads_view(q), None, weight,
                         weight)
    kern.append_u8(codes.handle, batch, *args, None, heads_view(outs[2]), heads_view(q), None, weight, weight)
    for t in outs:
        assert (np.abs(t.cpu().numpy() - want) <= 2.0 ** -10).all()
    page = codes.table[0, 0]
    assert (np.abs(pool[0, page, :, :3].cpu().numpy().transpose(1, 0, 2) - want[:, :2]) <= 2.0 ** -10).all()
    scales = codes.handle.key_scale.storage[page, :, :3].cpu().numpy().T
    assert (scales[0] == 0).all() and (np.abs(scales[1] * 127.5 - 1) < 2.0 ** -9).all()

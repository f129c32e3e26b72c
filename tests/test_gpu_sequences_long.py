"""Long contexts on the GPU, through every form of the kernels, by the bound of sequences_long.py: the result depends on the keys
at borders of tiles, pieces and pages, and on the last one (test_sequences_long.py shows what the bound refuses)."""
import numpy as np
import pytest
import torch

from adrastea_amd import PackedBatch, PagedBatch, PagedCache, TensorView
import sequences_reference as ref
from sequences_long import Definition, matrix_steps, row_steps, sequence
from test_gpu_sequences import CAUSAL, FORMS, NONE, heads_view, ints, shared_keys  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

# (sequences of (rows, keys), heads, kv heads, d, page size)
LONG = [([(1, 40011)], 16, 2, 64, 16), ([(3, 70017), (1, 20001)], 8, 4, 128, 32), ([(300, 20011)], 8, 2, 128, 64),
        ([(1, 1500 * i + 1) for i in range(1, 20)], 4, 4, 64, 16), ([(40, 30033), (1, 50000), (0, 100), (1, 9001)], 6, 2, 128, 128),
        ([(2, 131073)], 4, 1, 128, 16)]


@pytest.mark.parametrize("mask", [CAUSAL, NONE], ids=["causal", "full"])
@pytest.mark.parametrize("case", LONG, ids=["%dx_%dx%d_h%d_%d_d%d" % (len(c[0]), *c[0][0], *c[1:4]) for c in LONG])
def test_long_contexts(shared_keys, request, case, mask):  # noqa: F811
    seqs, heads, kv, d, page = case
    gen = torch.Generator(device="cuda").manual_seed(len(seqs) + d)
    data = [sequence(max(r, 1), n, heads, kv, d, gen, "cuda") for r, n in seqs]
    scale = data[0][3]
    rows = [r for r, _ in seqs]
    q = torch.cat([s[0][:, :r] for s, r in zip(data, rows)], 1).permute(1, 0, 2).contiguous()
    k, v = (torch.cat([s[i] for s in data], 1).permute(1, 0, 2).contiguous() for i in (1, 2))
    pages, table = ref.pages_of([n for _, n in seqs], page, np.random.default_rng(3))
    pools = torch.full((2, pages, page, kv, d), float("nan"), dtype=torch.float16, device="cuda")
    starts = ref.offsets([n for _, n in seqs])
    for i, (_, n) in enumerate(seqs):
        for pool, x in zip(pools, (k, v)):
            whole = torch.full((-(-n // page) * page, kv, d), float("nan"), dtype=torch.float16, device="cuda")
            whole[:n] = x[starts[i]:starts[i + 1]]
            pool[ints(table[i, :-(-n // page)]).long()] = whole.view(-1, page, kv, d)
    cache = PagedCache(*(TensorView.of(t.permute(0, 2, 1, 3)) for t in pools))
    offsets, longest = ints(ref.offsets(rows)), max(n for _, n in seqs)
    from_pages, from_packed = torch.empty_like(q), torch.empty_like(q)
    shared_keys.attention_paged_f16(heads_view(from_pages), heads_view(q), cache,
                                    PagedBatch(offsets, ints([n for _, n in seqs]), ints(table), max(rows), longest), scale, 1.0, mask)
    shared_keys.attention_packed_f16(heads_view(from_packed), heads_view(q), heads_view(k), heads_view(v),
                                     PackedBatch(offsets, ints(starts), max(rows), longest), scale, 1.0, mask)
    steps = row_steps if request.node.callspec.params["shared_keys"] == FORMS[0] else matrix_steps
    for i, (r, n) in enumerate(seqs):
        if r == 0:
            continue
        want = Definition(*data[i], causal=mask == CAUSAL)
        at = int(offsets[i])
        for got in (from_pages, from_packed):
            assert want.agrees(got[at:at + r].permute(1, 0, 2), steps(n)), (i, r, n)

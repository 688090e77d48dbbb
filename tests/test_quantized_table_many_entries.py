"""8-bit tables with more entries than the workgroups of a launch take at once: every one of the entries that a
lane group holds together, a last group that is partly filled, and a second step of the loops."""
import numpy as np
import pytest
import torch

import embiggen_amd as E
from embiggen_amd.embedding_transformers import METHODS
from test_quantized_table import CODES, check_table, expand, quantise

# width, entries: four rows a workgroup and 128 of them; four entries a lane group, the last ones partly filled
MANY = [(600, 9_001), (7, 200_003)]


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,entries", MANY)
def test_many_entries_written_and_read(width, entries, dtype, id_type, codes):
    rows = entries // 3
    gen = torch.Generator().manual_seed(width)
    first = torch.randn(rows, width, generator=gen).to(dtype)
    values = torch.randn(entries, width, generator=gen).to(dtype)
    ids = torch.randint(-20, rows + 20, (entries,), generator=gen)  # many rows several times, some outside
    table = E.QuantizedTable.from_table(first.cuda(), codes, 32)
    check_table(table, first.double().numpy())
    table.write(values.cuda(), ids.to(id_type).cuda())
    want = first.clone()
    inside = ((ids >= 0) & (ids < rows)).nonzero().squeeze(1).tolist()
    last = {int(ids[i]): i for i in inside}  # the last entry of a row
    want[list(last)] = values[list(last.values())]
    check_table(table, want.double().numpy())
    # read back in another order, rows outside among them
    whole = expand(*quantise(want.double().numpy(), codes, 32), 32)
    whole = torch.from_numpy(np.concatenate([whole, np.zeros((1, width), np.float32)]))
    at = torch.randint(-20, rows + 20, (entries,), generator=gen)
    place = torch.where((at >= 0) & (at < rows), at, torch.tensor(rows))
    assert torch.equal(table.read(at.to(id_type).cuda()).cpu(), whole[place])
    assert torch.equal(table.read(at.to(id_type).cuda(), torch.bfloat16).cpu(), whole[place].bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
@pytest.mark.parametrize("width,edges", MANY)
@pytest.mark.parametrize("method", list(METHODS))
def test_many_edges_are_what_few_of_them_are(method, width, edges, codes):
    """An edge's result has nothing to do with the edges beside it: the same bits as in calls of 300 edges, where every
    lane group has one edge."""
    gen = torch.Generator().manual_seed(width)
    table = E.QuantizedTable.from_table(torch.randn(800, width, generator=gen).cuda(), codes, 32)
    other = E.QuantizedTable.from_table(torch.randn(300, width, generator=gen).cuda(), codes, 64)
    src, dst = torch.randint(-5, 805, (edges,), generator=gen), torch.randint(-5, 305, (edges,), generator=gen)
    for id_type in (torch.int32, torch.int64):
        u, v = src.to(id_type).cuda(), dst.to(id_type).cuda()
        got = E.edge_embedding(table, u, v, method, destination_table=other)
        places = list(range(0, edges, 300)) if edges < 10_000 else [0, 65_300, 65_400, 130_900, 131_000, 196_500, edges - 300]
        for i in places:
            few = E.edge_embedding(table, u[i:i + 300], v[i:i + 300], method, destination_table=other)
            assert torch.equal(got[i:i + 300], few), (id_type, i)


@pytest.mark.gpu
def test_more_edges_than_one_step_of_the_largest_launch():
    """2^22 workgroups of four lane groups and four edges each: behind them a second step begins."""
    edges, width = (1 << 26) + 5, 1000
    gen = torch.Generator().manual_seed(0)
    table = E.QuantizedTable.from_table(torch.randn(500, width, generator=gen).cuda(), group_size=128)
    src, dst = (torch.randint(0, 500, (edges,), device="cuda", dtype=torch.int32) for _ in range(2))
    got = E.edge_embedding(table, src, dst, "CosineSimilarity")
    # all pairs of rows, looked up
    rows = torch.arange(500, device="cuda", dtype=torch.int32)
    pairs = E.edge_embedding(table, rows.repeat_interleave(500), rows.repeat(500), "CosineSimilarity").view(500, 500)
    for first in range(0, edges, 1 << 24):
        at = slice(first, first + (1 << 24))
        assert torch.equal(got[at, 0], pairs[src[at].long(), dst[at].long()]), first

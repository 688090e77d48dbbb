"""8-bit tables as objects: copied, stored and taken up again, and where they are refused."""
import copy
import io
import pickle

import pytest
import torch

import embiggen_amd as E
from embiggen_amd import _lib


def on_the_cpu(rows=4, width=20):
    """A table that no device holds (the class refuses to make one)."""
    table = E.QuantizedTable.__new__(E.QuantizedTable)
    table._codes, table._scales = torch.zeros(rows, 32, dtype=torch.int8), torch.zeros(rows, 1)
    table.embedding_size, table.group_size = width, 64
    table._io = _lib.Table8(table._codes.data_ptr(), table._scales.data_ptr(), rows, width, 32, 64, 0)
    table._taken = table._where()
    return table


def test_a_table_is_stored_by_its_tensors_and_checked_when_it_is_taken_up():
    table = on_the_cpu()
    stored = pickle.dumps(table)
    for again in (lambda: pickle.loads(stored), lambda: copy.copy(table), lambda: copy.deepcopy(table)):
        with pytest.raises(ValueError, match="no CPU execution path"):
            again()


def test_tensors_that_moved_are_checked_again():
    table = on_the_cpu()
    assert table._table() is table._io
    for change in (lambda: setattr(table.codes, "data", torch.zeros(4, 32, dtype=torch.int8)),
                   lambda: setattr(table.scales, "data", torch.zeros(4, 1)),
                   lambda: table.codes.resize_(2, 32)):
        change()
        with pytest.raises(ValueError, match="no CPU execution path|The scales should be"):
            table._table()
        table._taken = table._where()


@pytest.mark.parametrize("transformer", [E.GraphTransformer, E.EdgePredictionTransformer, E.EdgeLabelPredictionTransformer])
def test_transformers_of_graphs_refuse_a_table(transformer):
    for features in (on_the_cpu(), [on_the_cpu()], (on_the_cpu(), on_the_cpu())):
        with pytest.raises(ValueError, match="8 bits"):
            transformer("Hadamard", aligned_mapping=True).fit(features)


@pytest.mark.parametrize("transformer", [E.NodeTransformer, E.NodeLabelPredictionTransformer])
def test_transformers_of_nodes_refuse_a_table(transformer):
    with pytest.raises(ValueError, match="neither a pandas DataFrame nor a numpy array"):
        transformer(aligned_mapping=True).fit(on_the_cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
def test_copies_of_a_table_and_of_a_transformer(codes):
    gen = torch.Generator().manual_seed(0)
    table = E.QuantizedTable.from_table(torch.randn(30, 37, generator=gen).cuda(), codes, 16)
    values = table.read()
    transformer = E.EdgeTransformer(["Hadamard", "CosineSimilarity"]).fit(table)
    ids = torch.arange(30, device="cuda")
    features = transformer.transform(ids, ids.flip(0))
    file = io.BytesIO()
    torch.save(table, file)
    file.seek(0)
    deep = [copy.deepcopy(table), pickle.loads(pickle.dumps(table)), torch.load(file, weights_only=False)]
    shared = copy.copy(table)
    transformers = [copy.deepcopy(transformer), pickle.loads(pickle.dumps(transformer))]
    assert shared.codes is table.codes and shared.scales is table.scales
    table.write(torch.zeros(30, 37).cuda())
    for other in deep:
        assert other.codes.dtype == codes and (other.shape, other.group_size) == (table.shape, 16)
        assert torch.equal(other.read(), values)
    for other in transformers:
        assert torch.equal(other.transform(ids, ids.flip(0)), features)
    assert bool((shared.read() == 0).all())


@pytest.mark.gpu
def test_tensors_that_moved_are_the_table():
    gen = torch.Generator().manual_seed(0)
    table, other = (E.QuantizedTable.from_table(torch.randn(n, 40, generator=gen).cuda(), group_size=16) for n in (30, 12))
    want, ids = other.read(), torch.arange(30, device="cuda")
    table.codes.data, table.scales.data = other.codes.clone(), other.scales.clone()
    got = table.read(ids)
    assert table.shape == (12, 40) and torch.equal(got[:12], want) and bool((got[12:] == 0).all())
    table.write(torch.zeros(30, 40).cuda(), ids)  # the rows behind the last one are left out
    assert bool((table.read() == 0).all()) and torch.equal(other.read(), want)
    table.scales.data = other.scales[:5].clone()
    for call in (table.read, lambda: table.write(want), lambda: E.edge_embedding(other, ids, ids, destination_table=table)):
        with pytest.raises(ValueError, match="The scales should be"):
            call()

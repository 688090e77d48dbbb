"""Embedding tables in 8 bits against their definition: codes, scales and values read back are exact;
the edge operators' sums are within (d + 8) 2^-24 of their terms' magnitudes."""
import ctypes as C

import numpy as np
import pytest
import torch

import embiggen_amd as E
from embiggen_amd import _lib
from embiggen_amd.embedding_transformers import METHODS

CODES = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
E4M3 = None


def e4m3_values():
    """The non-negative finite values of the format, by their codes."""
    global E4M3
    if E4M3 is None:
        code = np.arange(127)
        exponent, mantissa = code >> 3, code & 7
        E4M3 = np.where(exponent == 0, mantissa * 2.0 ** -9,
                        (1 + mantissa / 8) * 2.0 ** (exponent - 7.0))
    return E4M3


def scale_of(top, dtype):
    """The scale of groups whose largest magnitudes are the float32 numbers `top`."""
    inverse = np.float32(1) / np.float32(CODES[dtype])
    return np.maximum(np.asarray(top).astype(np.float32) * inverse, np.float32(2.0 ** -90))


def quantise(values, dtype, group):
    """(codes as the values they stand for, scales) in 64 bits, by the definition."""
    values = np.asarray(values, dtype=np.float64)
    n, d = values.shape
    groups = -(-d // group)
    codes, scales = np.zeros((n, d)), np.zeros((n, groups), dtype=np.float32)
    for g in range(groups):
        part = values[:, g * group:(g + 1) * group]
        top = np.abs(part).max(1)
        with np.errstate(invalid="ignore"):
            scale = scale_of(top, dtype)
        scale[~np.isfinite(top)] = np.nan
        scales[:, g] = scale
        with np.errstate(invalid="ignore"):
            q = part / scale.astype(np.float64)[:, None]
        if dtype == torch.int8:
            c = np.round(q)
        else:
            table = e4m3_values()
            above = np.clip(np.searchsorted(table, np.abs(q)), 1, 126)
            lo, hi = table[above - 1], table[above]
            up = (np.abs(q) - lo > hi - np.abs(q)) | ((np.abs(q) - lo == hi - np.abs(q)) & (above % 2 == 0))
            c = np.where(up, hi, lo) * np.sign(q)
        c[~np.isfinite(top)] = 0
        codes[:, g * group:(g + 1) * group] = c
    return codes, scales


def stored(table):
    codes = table.codes[:, :table.embedding_size].float().cpu().numpy().astype(np.float64)
    return codes, table.scales.cpu().numpy()


def expand(codes, scales, group):
    with np.errstate(invalid="ignore"):
        return (codes.astype(np.float32) * np.repeat(scales, group, 1)[:, :codes.shape[1]])


def check_table(table, values):
    codes, scales = stored(table)
    want, want_scales = quantise(values, table.codes.dtype, table.group_size)
    assert np.array_equal(scales, want_scales, equal_nan=True)
    assert np.array_equal(codes, want), np.argwhere(codes != want)[:5]
    assert np.array_equal(table.read().cpu().numpy(), expand(want, want_scales, table.group_size),
                          equal_nan=True)
    pad = table.codes.view(torch.uint8)[:, table.embedding_size:]
    assert bool((pad == 0).all())


# ------------------------------------------------------------------------------ refusals (CPU)
def test_the_definition_rounds_like_the_format():
    """The oracle's e4m3 rounding against torch's conversion (float32 inputs, exact quotients)."""
    x = torch.linspace(-448, 448, 100_001)
    table = e4m3_values()
    a = x.abs().double().numpy()
    above = np.clip(np.searchsorted(table, a), 1, 126)
    lo, hi = table[above - 1], table[above]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (above % 2 == 0))
    assert np.array_equal(np.where(up, hi, lo) * np.sign(x.numpy()),
                          x.to(torch.float8_e4m3fn).float().numpy())


def test_refusals():
    codes, scales = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1)
    T = E.QuantizedTable
    for bad, text in (
            (lambda: T(codes.float(), scales), "int8 or float8"),
            (lambda: T(codes[0], scales), "two-dimensional"),
            (lambda: T(codes, scales, group_size=48), "group size"),
            (lambda: T(codes[:, :31], scales), "multiple of 16"),
            (lambda: T(codes, scales, embedding_size=33), "multiple of 16"),
            (lambda: T(codes, scales, embedding_size=0), "multiple of 16"),
            (lambda: T(codes, torch.zeros(4, 2)), "scales"),
            (lambda: T(codes, scales.double()), "scales"),
            (lambda: T(codes, scales), "no CPU execution path"),
            (lambda: T.empty(4, 0), "at least one column"),
            (lambda: T.empty(4, 8, torch.uint8), "int8 or float8"),
            (lambda: T.empty(4, 8, group_size=8), "group size"),
            (lambda: T.from_table(torch.zeros(4, 8)), "no CPU execution path"),
            (lambda: T.from_table(torch.zeros(4, 8).half()), "float32 or bfloat16"),
            (lambda: T.from_table(torch.zeros(8)), "two-dimensional")):
        with pytest.raises(ValueError, match=text):
            bad()


def test_refusals_at_the_c_boundary():
    L = _lib.lib()
    good = dict(d_codes=64, d_scales=64, rows=4, d=20, stride=32, group=64, code=0)
    for change, text in ((dict(code=2), b"code"), (dict(group=8), b"group"), (dict(stride=24), b"stride"),
                         (dict(d=0), b"stride"), (dict(d=33), b"stride"), (dict(d_codes=None), b"NULL"),
                         (dict(d_codes=8), b"aligned")):
        t = _lib.Table8(**{**good, **change})
        for status in (L.gn2v_table_write(C.byref(t), None, 0, 20, None, 0, 0, None, None),
                       L.gn2v_table_read(C.byref(t), None, 0, 0, None, 0, 20, None),
                       L.gn2v_table_edge_embedding(C.byref(t), C.byref(t), None, None, 4, 0, 0, None,
                                                   20, None)):
            assert status == 1 and text in L.gn2v_last_error()
    t = _lib.Table8(**good)
    assert L.gn2v_table_write(C.byref(t), None, 5, 20, None, 0, 0, None, None) == 1
    assert L.gn2v_table_write(C.byref(t), None, 0, 19, None, 0, 0, None, None) == 1
    assert L.gn2v_table_write(C.byref(t), None, 0, 20, None, 0, 5, None, None) == 1
    assert L.gn2v_table_write(C.byref(t), None, 0, 20, 64, 2, 1, None, None) == 1
    assert L.gn2v_table_write(C.byref(t), 64, 0, 20, 64, 4, 5000, None, None) == 1  # no scratch
    assert L.gn2v_table_write(None, None, 0, 20, None, 0, 0, None, None) == 1
    assert L.gn2v_table_read(C.byref(t), None, 0, 3, None, 0, 20, None) == 1
    assert L.gn2v_table_edge_embedding(C.byref(t), C.byref(t), None, None, 4, 0, 99, None, 20, None) == 1
    assert L.gn2v_table_edge_embedding(C.byref(t), C.byref(t), None, None, 4, 0, 7, None, 39, None) == 1
    other = _lib.Table8(**{**good, "code": 1})
    assert L.gn2v_table_edge_embedding(C.byref(t), C.byref(other), None, None, 4, 0, 0, None, 20, None) == 1


# ----------------------------------------------------------------------------- write and read
@pytest.mark.gpu
@pytest.mark.parametrize("group", [16, 32, 64, 128])
@pytest.mark.parametrize("width", [1, 7, 16, 33, 100, 128, 130, 520])
@pytest.mark.parametrize("codes", list(CODES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_written_rows_are_the_definition(dtype, codes, width, group):
    gen = torch.Generator().manual_seed(width + group)
    values = (torch.randn(70, width, generator=gen)
              * torch.exp(torch.randn(70, 1, generator=gen) * 5)).to(dtype)
    values[3] = 0
    values[4] = -0.0
    values[5] *= 1e-38
    table = E.QuantizedTable.from_table(values.cuda(), codes, group)
    assert table.shape == (70, width) and len(table) == 70
    check_table(table, values.double().numpy())
    assert torch.equal(table.read(dtype=torch.bfloat16), table.read().bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
def test_values_next_to_the_borders_of_the_codes(codes):
    """Quotients at, just above and just below the midpoint between two codes, for scales whose
    division is inexact: one rounding, never two."""
    rng = np.random.RandomState(1)
    rows = []
    for _ in range(400):
        top = np.float32(rng.uniform(0.5, 2) * 2.0 ** rng.randint(-60, 60))
        scale = np.float64(scale_of(top, codes))
        if codes == torch.int8:
            middle = rng.randint(0, 126, 15) + 0.5
        else:
            t = e4m3_values()
            i = rng.randint(0, 126, 15)
            middle = (t[i] + t[i + 1]) / 2
        x = (middle * scale).astype(np.float32)
        step = rng.randint(-1, 2, 15)
        x = np.where(step < 0, np.nextafter(x, np.float32(0)),
                     np.where(step > 0, np.nextafter(x, np.float32(np.inf)), x))
        rows.append(np.concatenate([[top], np.minimum(x, top) * rng.choice([-1, 1], 15)]))
    values = np.array(rows, dtype=np.float32)
    table = E.QuantizedTable.from_table(torch.from_numpy(values).cuda(), codes, 16)
    check_table(table, values)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
def test_every_code_reads_back_as_its_value(codes):
    raw = torch.arange(256, dtype=torch.uint8).view(codes).view(8, 32)
    scales = torch.rand(8, 2) + 0.5
    table = E.QuantizedTable(raw.cuda(), scales.cuda(), group_size=16)
    want = raw.float() * scales.repeat_interleave(16, 1)
    assert torch.equal(torch.nan_to_num(table.read().cpu(), nan=7.0), torch.nan_to_num(want, nan=7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
def test_infinities_and_nans_stay_in_their_group(codes):
    values = torch.randn(6, 96, generator=torch.Generator().manual_seed(0))
    values[0, 3], values[1, 40], values[2, 95] = float("inf"), float("nan"), float("-inf")
    values[3, 0] = 3.4e38
    table = E.QuantizedTable.from_table(values.cuda(), codes, 32)
    check_table(table, values.numpy())
    back = table.read().cpu()
    assert bool(back[0, :32].isnan().all()) and not back[0, 32:].isnan().any()
    assert not back[3].isnan().any() and not back[4].isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("entries", [1, 300, 512, 513, 1024, 1025, 6000])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_the_last_entry_of_a_row_is_kept(entries, id_type):
    rows, width = 500, 40
    gen = torch.Generator().manual_seed(entries)
    first = torch.randn(rows, width, generator=gen)
    values = torch.randn(entries, width, generator=gen)
    ids = torch.randint(0, 60, (entries,), generator=gen) * 7  # many times the same rows
    ids[torch.rand(entries, generator=gen) < 0.1] = -1
    ids[torch.rand(entries, generator=gen) < 0.1] = rows
    table = E.QuantizedTable.from_table(first.cuda(), group_size=32)
    untouched = table.read()
    table.write(values.cuda(), ids.to(id_type).cuda())
    want = first.clone()
    for i in range(entries):
        if 0 <= ids[i] < rows:
            want[ids[i]] = values[i]
    check_table(table, want.numpy())
    outside = torch.ones(rows, dtype=torch.bool)
    outside[ids[(ids >= 0) & (ids < rows)]] = False
    assert torch.equal(table.read()[outside.cuda()], untouched[outside.cuda()])


@pytest.mark.gpu
def test_reading_some_rows_and_rows_outside():
    values = torch.randn(50, 33, generator=torch.Generator().manual_seed(0))
    table = E.QuantizedTable.from_table(values.cuda(), torch.float8_e4m3fn, 16)
    whole = table.read()
    ids = torch.tensor([4, -1, 49, 50, 4, 2 ** 31 - 1, 0])
    for id_type in (torch.int32, torch.int64):
        got = table.read(ids.to(id_type).cuda())
        want = torch.zeros(7, 33).cuda()
        for i, r in enumerate(ids.tolist()):
            if 0 <= r < 50:
                want[i] = whole[r]
        assert torch.equal(got, want)
    far = torch.tensor([2 ** 32, -2 ** 40]).cuda()
    assert bool((table.read(far) == 0).all())
    assert table.read(ids[:0].cuda()).shape == (0, 33)
    table.write(values[:0].cuda(), ids[:0].cuda())
    table.write(values[:3].cuda() * 2)  # the first rows
    assert torch.equal(table.read()[3:], whole[3:])
    for bad, text in ((lambda: table.write(values[:2].cuda(), ids.cuda()), "rows for 7"),
                      (lambda: table.write(values[:2]), "on cuda"),
                      (lambda: table.write(values[:2, :32].cuda()), "33 columns"),
                      (lambda: table.write(torch.zeros(51, 33).cuda()), "do not fit"),
                      (lambda: table.write(values.double().cuda()), "float32 or bfloat16"),
                      (lambda: table.read(ids), "on cpu"),
                      (lambda: table.read(ids.float().cuda()), "int32 or int64"),
                      (lambda: table.read(dtype=torch.float16), "float32 or bfloat16")):
        with pytest.raises(ValueError, match=text):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_values(dtype):
    wide = torch.randn(40, 61, generator=torch.Generator().manual_seed(0)).to(dtype)
    device = wide.cuda()
    views = [device[:, :37], device[:, 1:38], device[::2, 3:40], device.t()[:37].t(),
             device[:1, :37].expand(40, 37)]
    for v in views:
        table = E.QuantizedTable.from_table(v, group_size=16)
        check_table(table, v.cpu().double().numpy())
    table = E.QuantizedTable.from_table(device, group_size=16, embedding_size=20)
    check_table(table, wide[:, :20].double().numpy())
    empty = E.QuantizedTable.empty(0, 20)
    assert empty.read().shape == (0, 20)
    assert bool((E.QuantizedTable.empty(3, 20).read() == 0).all())


# ------------------------------------------------------------------------------ edge operators
@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
@pytest.mark.parametrize("width", [1, 30, 100, 128, 600])
@pytest.mark.parametrize("method", list(METHODS))
def test_edge_operators_on_8_bit_rows(method, width, codes):
    gen = torch.Generator().manual_seed(width)
    table = E.QuantizedTable.from_table(torch.randn(80, width, generator=gen).cuda(), codes, 32)
    other = E.QuantizedTable.from_table(torch.randn(30, width, generator=gen).cuda(), codes, 64)
    src = torch.randint(0, 80, (301,), generator=gen)
    dst = torch.randint(0, 30, (301,), generator=gen)
    dst[7], src[9] = -1, 80  # rows of zeros
    a = torch.cat([table.read(), torch.zeros(1, width).cuda()]).cpu().double()[src]
    b = torch.cat([other.read(), torch.zeros(1, width).cuda()]).cpu().double()[dst]
    want, tolerance = {
        "Hadamard": lambda: (a * b, 0), "Sum": lambda: (a + b, 0), "Average": lambda: ((a + b) / 2, 0),
        "L1": lambda: (a - b, 0), "AbsoluteL1": lambda: ((a - b).abs(), 0),
        "SquaredL2": lambda: ((a - b) ** 2, 3 * 2.0 ** -24), "L2": lambda: ((a - b).abs(), 6 * 2.0 ** -24),
        "Concatenate": lambda: (torch.cat([a, b], 1), 0), "Min": lambda: (torch.minimum(a, b), 0),
        "Max": lambda: (torch.maximum(a, b), 0),
        "L2Distance": lambda: ((a - b).square().sum(1, keepdim=True).sqrt(), (width + 8) * 2.0 ** -24),
        "CosineSimilarity": lambda: (
            (a * b).sum(1, keepdim=True)
            / (a.norm(dim=1) * b.norm(dim=1)).clamp(min=1e-6)[:, None], None),
    }[method]()
    got = E.edge_embedding(table, src.cuda(), dst.int().cuda() if width == 30 else dst.cuda(), method,
                           destination_table=other).cpu().double()
    assert got.shape == want.shape
    if tolerance is None:
        size = (a * b).abs().sum(1, keepdim=True) / (a.norm(dim=1) * b.norm(dim=1)).clamp(min=1e-6)[:, None]
        assert bool(((got - want).abs() <= (2 * width + 16) * 2.0 ** -24 * size).all())
    else:  # one float32 operation more than the values: half a step of the result each
        assert bool(((got - want).abs() <= (2.0 ** -24 + tolerance) * want.abs()).all())


@pytest.mark.gpu
def test_edge_transformer_on_an_8_bit_table():
    gen = torch.Generator().manual_seed(0)
    rows = torch.randn(60, 48, generator=gen).cuda()
    table = E.QuantizedTable.from_table(rows)
    src, dst = (torch.randint(0, 60, (200,), generator=gen).cuda() for _ in range(2))
    t = E.EdgeTransformer(["Hadamard", "CosineSimilarity"]).fit(table)
    out = t.transform(src, dst)
    exact = E.EdgeTransformer(["Hadamard", "CosineSimilarity"]).fit(table.read()).transform(src, dst)
    assert out.shape == (200, 49) and float((out - exact).abs().max()) <= 60 * 2.0 ** -24 * 16
    # within the codes' rounding of the table's own values: half a step of 1 / 127 of the largest
    near = E.edge_embedding(rows, src, dst, "Sum")
    assert float((E.edge_embedding(table, src, dst, "Sum") - near).abs().max()) <= float(
        rows.abs().max()) / 127 * 1.001
    same = E.edge_embedding(table, src, src, "L1")
    assert bool((same == 0).all())
    for bad in (lambda: E.EdgeTransformer().fit([table, table]),
                lambda: E.EdgeTransformer().fit(table, node_type_feature=np.zeros((2, 2))),
                lambda: E.edge_embedding(table, src, dst, destination_table=rows),
                lambda: E.edge_embedding(rows, src, dst, destination_table=table),
                lambda: E.edge_embedding(table, src, dst, embedding_size=47),
                lambda: E.edge_embedding(table, src, dst[:5]),
                lambda: E.edge_embedding(table, src, dst.cpu()),
                lambda: E.edge_embedding(
                    table, src, dst, destination_table=E.QuantizedTable.empty(60, 48, torch.float8_e4m3fn))):
        with pytest.raises(ValueError):
            bad()
    # the float path is what it was
    t = E.EdgeTransformer("Hadamard").fit(rows)
    assert torch.equal(t.transform(src, dst), rows[src] * rows[dst])


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets():
    """A table of more than 2^32 bytes of codes: its last rows are written, read and used by edges."""
    rows, width = 34_000_000, 128
    table = E.QuantizedTable.empty(rows, width, group_size=128)
    values = torch.randn(3, width, generator=torch.Generator().manual_seed(0))
    ids = torch.tensor([rows - 1, 5, rows - 2]).cuda()
    table.write(values.cuda(), ids)
    want, scales = quantise(values.double().numpy(), torch.int8, 128)
    assert np.array_equal(table.read(ids).cpu().numpy(), expand(want, scales, 128))
    last = table.read(ids)
    assert torch.equal(E.edge_embedding(table, ids[:1], ids[2:], "Hadamard"), last[:1] * last[2:])
    assert bool((table.read(torch.tensor([rows - 3, 4, 6]).cuda()) == 0).all())


@pytest.mark.gpu
def test_captured_writes_and_reads():
    table = E.QuantizedTable.empty(4000, 64)
    values, ids = torch.zeros(2000, 64).cuda(), torch.zeros(2000, dtype=torch.int64).cuda()

    def step():
        table.write(values, ids)
        return table.read(ids), E.edge_embedding(table, ids[:-1], ids[1:], "CosineSimilarity")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        read, cosine = step()
    for seed in (1, 2, 3):
        gen = torch.Generator().manual_seed(seed)
        values.copy_(torch.randn(2000, 64, generator=gen))
        ids.copy_(torch.randint(0, 4000, (2000,), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        own = E.QuantizedTable.empty(4000, 64)
        own.write(values, ids)
        assert torch.equal(read, own.read(ids))
        assert torch.equal(cosine, E.edge_embedding(own, ids[:-1], ids[1:], "CosineSimilarity"))

"""Scales of 8-bit tables at the ends of float32, and how far the stored scale is from the quotient."""
import numpy as np
import pytest
import torch

import embiggen_amd as E
from test_quantized_table import CODES


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
def test_cosines_of_rows_whose_scales_multiply_past_float32(codes):
    """The sums over a row's zeros stay zero whatever its scale; what the float32 rows give is the definition."""
    a, b = torch.ones(7, 64), torch.ones(7, 64)
    a[0], b[0] = 0, 1
    a[0, 0] = 1e22  # the square is infinite, of the zeros beside it zero: 1e22 / infinity
    a[1], b[1] = 0, 0
    a[1, 0], b[1, 40] = 1e22, 1e22  # no column in common: 0 / infinity
    a[2], b[2] = 0, 0
    a[2, 0], b[2, 0] = 3e38, 1e-30  # the square of 1e-30 is zero, and zero times infinity is no number
    a[3], b[3] = 0, 0
    a[3, 0], b[3, 0] = 1e19, 1e-12  # inside float32: one
    a[4, 5] = float("nan")
    a[6], b[6] = 0, 0
    a[6, 0], b[6, 0] = 3e38, 1e-20  # 3e18 / infinity
    table, other = (E.QuantizedTable.from_table(v.cuda(), codes, 32) for v in (a, b))
    ids = torch.arange(7, device="cuda")
    got = E.edge_embedding(table, ids, ids, "CosineSimilarity", destination_table=other).cpu().squeeze(1)
    want = E.edge_embedding(table.read(), ids, ids, "CosineSimilarity", destination_table=other.read()).cpu().squeeze(1)
    for i, value in ((0, 0.0), (1, 0.0), (2, float("nan")), (4, float("nan")), (6, 0.0)):
        assert np.array_equal([float(got[i]), float(want[i])], [value, value], equal_nan=True), i
    # at most 64 products, 8 operations more: (64 + 8) 2^-24 of the terms each, as of the other sums
    for i in (3, 5):
        assert abs(float(got[i]) - 1) <= 2 * 72 * 2.0 ** -24, i


@pytest.mark.gpu
@pytest.mark.parametrize("codes", list(CODES))
def test_the_scale_is_next_to_the_quotient(codes):
    """The scale is the largest magnitude times the float32 inverse of the largest code value: two roundings, 2^-24 of
    it each, of the quotient; so a value read back is within the code's half step, 2^-23 of a step per step more."""
    gen = torch.Generator().manual_seed(0)
    values = torch.randn(4000, 64, generator=gen) * torch.exp(torch.randn(4000, 1, generator=gen) * 3)
    table = E.QuantizedTable.from_table(values.cuda(), codes, 64)
    top = values.abs().amax(1).double()
    quotient = top / CODES[codes]
    scale = table.scales.cpu().double().squeeze(1)
    assert bool(((scale - quotient).abs() <= 2 * 2.0 ** -24 * (1 + 2.0 ** -24) * quotient).all())
    off = (table.read().cpu().double() - values.double()).abs()
    size = values.abs().double()
    # int8: half a step.  e4m3: 2^-4 of the value, at least half of the smallest step, 2^-9.  The value read back is
    # rounded to float32, and the largest one may lie 2^-23 outside the codes.
    half = 0.5 * quotient[:, None] if codes == torch.int8 else torch.maximum(2.0 ** -4 * size, 2.0 ** -10 * quotient[:, None])
    assert bool((off <= half * (1 + 2.0 ** -22) + 2.0 ** -22 * top[:, None]).all())

"""Projections of rows by their type against their definitions in 64 bits.

Tolerances, element by element.  A sum of n products in float32, in any order, is off by at most
(n + 2) 2^-24 times the sum of the products' magnitudes (first order; 8 more for the terms a formula
adds); a result in bfloat16 is rounded once more, 2^-8 of it.  The low-rank rows enter bfloat16 products
as a high and a low part: what is left out is 2^-8 of 2^-8 of them."""
import ctypes as C

import numpy as np
import pytest
import torch

import embiggen_amd as E
from embiggen_amd import _lib
from embiggen_amd.embedding_transformers import projections as module

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def rounding(dtype):
    return 0.0 if dtype == torch.float32 else 2.0 ** -8


def close(got, want, tolerance, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs() - tolerance
    assert not torch.isnan(got).any() and bool((off <= 0).all()), (
        what, float(off.max()), float((got - want).abs().max()))


def make(rows, types, *shapes, dtype, seed=0, unknown=0.1, skew=False):
    gen = torch.Generator().manual_seed(seed)
    if skew:
        ids = (torch.rand(rows, generator=gen) ** 4 * types).long().clamp_(max=types - 1)
    else:
        ids = torch.randint(0, types, (rows,), generator=gen)
    ids[torch.rand(rows, generator=gen) < unknown] = -1
    return ids, [torch.randn(*s, generator=gen).to(dtype) for s in shapes]


def typed_reference(x, w, ids, b, dy=None, dtype=torch.float32):
    """(values, tolerances) of y, and with dy of dx, dw, db."""
    x, w, b = x.double(), w.double(), b.double()
    k, n = w.shape[1:]
    eps = rounding(dtype)
    names = {"y": (x.shape[0], n)}
    if dy is not None:
        dy = dy.double()
        names.update(dx=x.shape, dw=w.shape, db=b.shape)
    value = {name: torch.zeros(shape, dtype=torch.float64) for name, shape in names.items()}
    size = {name: v.clone() for name, v in value.items()}
    for t in range(w.shape[0]):
        at = (ids == t).nonzero().squeeze(1)
        m = len(at)
        for out, f in ((value, lambda v: v), (size, torch.abs)):
            scale = U if out is size else 1
            out["y"][at] = (f(x[at]) @ f(w[t]) + f(b[t])) * (scale * (k + 8) if scale == U else 1)
            if dy is not None:
                out["dx"][at] = f(dy[at]) @ f(w[t]).T * (scale * (n + 8) if scale == U else 1)
                out["dw"][t] = f(x[at]).T @ f(dy[at]) * (scale * (m + 8) if scale == U else 1)
                out["db"][t] = f(dy[at]).sum(0) * (scale * (m + 8) if scale == U else 1)
    return value, {name: size[name] + eps * value[name].abs() for name in value}


def adapted_reference(x, w, down, up, ids, b, scale, dy=None, dtype=torch.float32):
    x, w, down, up, b = (v.double() for v in (x, w, down, up, b))
    rows, k = x.shape
    n, r = w.shape[1], down.shape[2]
    eps = rounding(dtype)
    split = 0.0 if dtype == torch.float32 else 2.0 ** -16
    names = {"y": (rows, n)}
    if dy is not None:
        dy = dy.double()
        names.update(dx=x.shape, dw=w.shape, d_down=down.shape, d_up=up.shape, db=b.shape)
    value = {name: torch.zeros(shape, dtype=torch.float64) for name, shape in names.items()}
    size = {name: v.clone() for name, v in value.items()}
    for out, f in ((value, lambda v: v), (size, torch.abs)):
        first = out is value
        c = (lambda terms: 1.0) if first else (lambda terms: U * terms)
        low = (lambda terms: 1.0) if first else (lambda terms: U * terms + split)
        s = f(torch.tensor(scale, dtype=torch.float64))
        out["y"] += (f(x) @ f(w) + f(b)) * c(k + r + 8)
        if dy is not None:
            out["dx"] += f(dy) @ f(w).T * c(n + r + 8)
            out["dw"] += f(x).T @ f(dy) * c(rows + 8)
            out["db"] += f(dy).sum(0) * c(rows + 8)
        for t in range(down.shape[0]):
            at = (ids == t).nonzero().squeeze(1)
            m = len(at)
            out["y"][at] += s * (f(x[at]) @ f(down[t])) @ f(up[t]) * low(k + r + 8)
            if dy is not None:
                back = s * f(dy[at]) @ f(up[t]).T
                out["dx"][at] += back @ f(down[t]).T * low(n + r + 8)
                out["d_down"][t] = f(x[at]).T @ back * low(m + n + 8)
                out["d_up"][t] = s * (f(x[at]) @ f(down[t])).T @ f(dy[at]) * low(m + k + 8)
    return value, {name: size[name] + eps * value[name].abs() for name in value}


def run_typed(x, w, types, b, dy=None):
    leaves = [v.cuda().requires_grad_(dy is not None) for v in (x, w, b)]
    y = E.typed_projection(leaves[0], leaves[1], types, bias=leaves[2])
    out = {"y": y}
    if dy is not None:
        out.update(zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy.cuda())))
    return out


# ------------------------------------------------------------------------------ refusals (CPU)
def test_refusals_of_the_rows_and_weights():
    x, w, ids = torch.zeros(4, 3), torch.zeros(2, 3, 5), torch.zeros(4, dtype=torch.int64)
    for bad, text in (
            (lambda: E.typed_projection([1], w, ids), "tensor"),
            (lambda: E.typed_projection(x[0], w, ids), "dimensions"),
            (lambda: E.typed_projection(x.double(), w, ids), "float32 or bfloat16"),
            (lambda: E.typed_projection(x.half(), w.half(), ids), "float32 or bfloat16"),
            (lambda: E.typed_projection(x, w[:, :2], ids), "shape"),
            (lambda: E.typed_projection(x, w[:, :, :0], ids), "empty"),
            (lambda: E.typed_projection(x, w.bfloat16(), ids), "type and device"),
            (lambda: E.typed_projection(x, w, ids, bias=torch.zeros(2, 4)), "bias"),
            (lambda: E.typed_projection(x, w, ids[:3]), "3 rows"),
            (lambda: E.typed_projection(x, w, ids.float()), "int32 or int64"),
            (lambda: E.typed_projection(x, w, ids), "no CPU execution path"),
            (lambda: E.adapted_projection(x, w[0], torch.zeros(2, 3, 65), torch.zeros(2, 65, 5),
                                          ids), "at most 64"),
            (lambda: E.adapted_projection(x, w[0], torch.zeros(2, 3, 4), torch.zeros(2, 3, 5),
                                          ids), "up"),
            (lambda: E.adapted_projection(x, w[0], torch.zeros(2, 4, 4), torch.zeros(2, 4, 5),
                                          ids), "down"),
            (lambda: E.adapted_projection(x, w[0], torch.zeros(2, 3, 4), torch.zeros(2, 4, 5), ids,
                                          bias=torch.zeros(2, 5)), "dimensions"),
            (lambda: E.adapted_projection(x, w[0], torch.zeros(2, 3, 4), torch.zeros(2, 4, 5),
                                          ids), "no CPU execution path"),
            (lambda: E.TypePlan(ids, 0), "between 1"),
            (lambda: E.TypePlan(ids, 32769), "between 1"),
            (lambda: E.TypePlan(ids.float(), 2), "int32 or int64"),
            (lambda: E.TypePlan(ids, 2), "no CPU execution path"),
            (lambda: E.TypePlan.from_graph(E.karate_club(), "walks"), "'nodes' or 'edges'"),
            (lambda: E.TypePlan.from_graph(E.karate_club()), "do not have types")):
        with pytest.raises(ValueError, match=text):
            bad()


def test_refusals_at_the_c_boundary():
    L = _lib.lib()
    a, b = C.c_uint64(), C.c_uint64()
    assert L.gn2v_type_plan_words(10, 3, C.byref(a), C.byref(b)) == 0 and b.value == 0
    assert a.value == 2 * 10 + 2 * (3 + 2)
    for rows, types in ((1 << 31, 3), (10, 0), (10, 32769)):
        assert L.gn2v_type_plan_words(rows, types, C.byref(a), C.byref(b)) == 1
    assert L.gn2v_type_plan_words(10, 3, None, C.byref(b)) == 1
    assert L.gn2v_type_plan(None, 4, 10, 3, None, None, None) == 1
    assert L.gn2v_typed_product(None, None) == 1
    io = _lib.ProductIO()
    for name, value, text in (("dtype", 7, b"dtype"), ("n_types", 0, b"n_types"),
                              ("inputs", 0, b"inputs"), ("rank", 65, b"rank"), ("ldx", 1, b"stride"),
                              ("rows", 5, b"NULL")):
        io = _lib.ProductIO(dtype=0, n_types=2, inputs=4, outputs=4, ldx=4, ldy=4)
        io.weight.outer = 1
        setattr(io, name, value)
        for entry in (L.gn2v_typed_product, L.gn2v_adapted_product, L.gn2v_few_rows_product):
            assert entry(C.byref(io), None) == 1 and text in L.gn2v_last_error(), name
    io = _lib.ProductIO(dtype=0, n_types=2, inputs=4, outputs=4, ldx=4, ldy=4)
    io.weight.inner = io.weight.outer = 2
    assert L.gn2v_typed_product(C.byref(io), None) == 1 and b"must be 1" in L.gn2v_last_error()
    g = _lib.GradientIO(dtype=0, n_types=2, rows=100, inputs=4, outputs=4, ldx=4, ldy=4)
    assert L.gn2v_typed_gradient_temp(C.byref(g), C.byref(a)) == 0 and a.value > 0
    assert L.gn2v_typed_gradient(C.byref(g), None) == 1
    g.x_low = g.y_low = 1
    assert L.gn2v_typed_gradient_temp(C.byref(g), C.byref(a)) == 1
    g.y_low, g.inputs = 0, 65
    assert L.gn2v_typed_gradient_temp(C.byref(g), C.byref(a)) == 1


def test_the_packed_structure_has_its_fields():
    x, y = torch.zeros(3, 5), torch.zeros(3, 7)
    w, b = torch.zeros(2, 5, 7), torch.zeros(2, 7)
    down, up, low, ids = torch.zeros(2, 5, 4), torch.zeros(2, 4, 7), torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    views = [module._weights(t)[1] for t in (w, down, up)]
    io, _ = module._product_io(x, 5, views[0], y, 7, 2, b, None, ids, 4, 0.5, 1, views[1], views[2], low)
    for packed, structure in ((module._PRODUCT, _lib.ProductIO), (module._GRADIENT, _lib.GradientIO),
                              (module._ADAPTED_GRADIENT, _lib.AdaptedGradientIO)):
        assert packed.size == C.sizeof(structure)
        image = bytes(range(packed.size))
        filled = structure.from_buffer_copy(image)
        fields = []
        for name, _ in structure._fields_:
            value = getattr(filled, name)
            fields += [getattr(value, f) for f, _ in value._fields_] if isinstance(value, _lib.Weights) else [value]
        assert packed.unpack(image) == tuple(fields)
    assert (io.dtype, io.n_types, io.rows, io.inputs, io.outputs, io.ldx, io.ldy) == (0, 2, 3, 5, 7, 5, 7)
    assert (io.d_x, io.d_y, io.d_bias, io.d_types, io.d_low, io.d_plan) == (
        x.data_ptr(), y.data_ptr(), b.data_ptr(), ids.data_ptr(), low.data_ptr(), None)
    assert (io.bias_stride, io.type_bytes, io.rank, io.scale, io.low_rank_rows) == (7, 8, 4, 0.5, 1)
    for view, field in zip(views, (io.weight, io.down, io.up)):
        assert tuple(view) == (field.d_data, field.type_stride, field.inner, field.outer)


def test_weight_views_need_no_copies():
    w = torch.zeros(3, 4, 5)
    same, view = module._weights(w)
    assert same is w and (view.type_stride, view.inner, view.outer) == (20, 5, 1)
    t = w.transpose(1, 2)
    same, view = module._weights(t)
    assert same is t and (view.inner, view.outer) == (1, 5)
    copy, view = module._weights(t, rows_contiguous=True)
    assert copy is not t and (view.inner, view.outer) == (4, 1)
    strided = torch.zeros(3, 4, 10)[:, :, ::2]
    copy, view = module._weights(strided)
    assert copy is not strided and view.outer == 1
    wide = torch.zeros(6, 9)
    assert module._row_stride(wide[:, :4])[1] == 9 and module._row_stride(wide[::2])[1] == 18
    assert module._row_stride(wide[:1].expand(6, 9))[0].is_contiguous()
    assert module._row_stride(wide[:, ::2])[0].is_contiguous()
    assert module._row_stride(torch.zeros(1, 9)[:, :4])[1] >= 4


# ------------------------------------------------------------------------------------ the plan
@pytest.mark.gpu
@pytest.mark.parametrize("rows,types", [(0, 3), (1, 1), (1, 7), (63, 2), (64, 1), (65, 5), (511, 3), (512, 300),
                                        (513, 300), (1000, 3),
                                        (1024, 4000), (1025, 5), (5000, 1), (70_001, 37),
                                        (20_000, 20_000), (3000, 32_768),
                                        # counters that end at 64 KB of LDS, and just behind
                                        (5000, 4094), (5000, 4095), (5000, 4096), (2000, 16_383)])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_plan_is_the_stable_order(rows, types, id_type):
    gen = torch.Generator().manual_seed(rows + types)
    ids = torch.randint(0, types, (rows,), generator=gen)
    ids[torch.rand(rows, generator=gen) < 0.1] = -1
    ids[torch.rand(rows, generator=gen) < 0.02] = types  # one behind the last type
    ids[torch.rand(rows, generator=gen) < 0.02] = 2 ** 31 - 1
    plan = E.TypePlan(ids.to(id_type).cuda(), types)
    known = torch.where((ids < 0) | (ids >= types), torch.tensor(types), ids)
    order = torch.argsort(known, stable=True)
    assert torch.equal(plan.order.cpu().long(), order)
    offsets = torch.searchsorted(known[order], torch.arange(types + 2))
    offsets[types + 1] = rows
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    words = plan._words.cpu().long()
    assert torch.equal(words[rows:2 * rows], known[order])
    tiles = torch.cat([torch.zeros(1, dtype=torch.int64), ((offsets.diff() + 63) // 64).cumsum(0)])
    assert torch.equal(words[2 * rows + types + 2:], tiles)  # the types' first tiles of 64 rows


@pytest.mark.gpu
def test_plan_of_ids_beyond_32_bits_and_of_a_graph():
    ids = torch.tensor([0, 2 ** 32, 1, -2 ** 40, 2 ** 33 + 1, 0]).cuda()
    plan = E.TypePlan(ids, 2)
    assert plan.order.tolist() == [0, 5, 2, 1, 3, 4] and plan.offsets.tolist() == [0, 2, 3, 6]
    g = E.CSRGraph.from_edge_list([0, 1, 2], [1, 2, 3], node_types=["a", "b", None, "a"],
                                  edge_types=["u", "v", "u"])
    nodes = E.TypePlan.from_graph(g)
    assert nodes.number_of_types == 2 and nodes.order.tolist() == [0, 3, 1, 2]
    edges = E.TypePlan.from_graph(g, "edges")
    assert edges.number_of_rows == g.get_number_of_directed_edges()


# ----------------------------------------------------------------------------- typed projection
SHAPES = [  # rows, types, inputs, outputs
    (1, 1, 1, 1), (1, 3, 128, 128), (7, 2, 3, 5), (48, 7, 100, 100), (64, 1, 32, 32),
    (65, 3, 33, 31), (129, 5, 64, 65), (200, 300, 17, 129), (1025, 4, 100, 71),
    (3001, 9, 130, 96), (5000, 3, 256, 200), (2049, 1, 128, 128), (300, 4, 300, 1), (300, 4, 1, 300),
    (700, 3, 513, 140), (90, 2, 5000, 10), (1500, 3, 90, 100), (1400, 3, 65, 60), (1300, 4, 160, 150),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,types,inputs,outputs", SHAPES)
def test_typed_projection_and_its_gradients(rows, types, inputs, outputs, dtype):
    ids, (x, w, b, dy) = make(rows, types, (rows, inputs), (types, inputs, outputs),
                              (types, outputs), (rows, outputs), dtype=dtype, seed=rows + inputs)
    want, tolerance = typed_reference(x, w, ids, b, dy, dtype)
    plan = E.TypePlan(ids.cuda(), types)
    forward = run_typed(x, w, ids.cuda(), b)["y"]
    close(forward, want["y"], tolerance["y"], "forward")
    close(run_typed(x, w, plan, b)["y"], want["y"], tolerance["y"], "forward, plan")
    got = run_typed(x, w, plan, b, dy)
    for name in want:
        close(got[name], want[name], tolerance[name], name)
    again = run_typed(x, w, ids.int().cuda(), b, dy)
    assert all(torch.equal(got[name], again[name]) for name in got)  # the same bits in every run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_typed_projection_without_known_rows_without_rows_and_without_bias(dtype):
    _, (x, w, b) = make(90, 3, (90, 20), (3, 20, 24), (3, 24), dtype=dtype)
    for rows in (90, 5, 0):
        ids = torch.full((rows,), -1, dtype=torch.int32).cuda()
        out = run_typed(x[:rows], w, ids, b, torch.ones(rows, 24, dtype=dtype))
        assert out["y"].shape == (rows, 24) and all(bool((v == 0).all()) for v in out.values())
        y = E.typed_projection(x[:rows].cuda(), w.cuda(), ids)
        assert y.shape == (rows, 24) and bool((y == 0).all())
    ids = torch.arange(90) % 3
    want, tolerance = typed_reference(x, w, ids, torch.zeros_like(b), dtype=dtype)
    for m in (90, 10):
        y = E.typed_projection(x[:m].cuda(), w.cuda(), ids[:m].cuda())
        close(y, want["y"][:m], tolerance["y"][:m], "no bias")
        # a single gradient each
    for leaf, name in ((0, "dx"), (1, "dw"), (2, "db")):
        dy = torch.randn(90, 24, generator=torch.Generator().manual_seed(1)).to(dtype)
        want, tolerance = typed_reference(x, w, ids, b, dy, dtype)
        leaves = [v.cuda().requires_grad_(i == leaf) for i, v in enumerate((x, w, b))]
        y = E.typed_projection(leaves[0], leaves[1], ids.cuda(), bias=leaves[2])
        close(torch.autograd.grad(y, leaves[leaf], dy.cuda())[0], want[name], tolerance[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [20, 300])
def test_unknown_rows_may_hold_anything(rows, dtype):
    ids, (x, w, b, dy) = make(rows, 4, (rows, 40), (4, 40, 36), (4, 36), (rows, 36), dtype=dtype)
    ids[3] = -1
    want, tolerance = typed_reference(x, w, ids, b, dy, dtype)
    bad = ids < 0
    x[bad] = float("nan")
    dy[bad] = float("inf")
    got = run_typed(x, w, ids.cuda(), b, dy)
    for name in want:
        close(got[name], want[name], tolerance[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [30, 500])
def test_strided_rows_weights_and_gradients(rows, dtype):
    ids, (wide, w, b, dy) = make(rows, 5, (rows, 77), (5, 50, 33), (5, 33), (rows, 33), dtype=dtype)
    want, tolerance = typed_reference(wide[:, :50], w, ids, b, dy, dtype)
    device = wide.cuda()
    views = {
        "columns": (device[:, :50], w.cuda()),
        "every second row": (torch.stack([device, device], 1).view(2 * rows, 77)[::2, :50], w.cuda()),
        "columns in another order": (device[:, :50].t().contiguous().t(), w.cuda()),
        "offset by one element": (torch.cat([device[:, :1], device], 1)[:, 1:51], w.cuda()),
        "transposed weights": (device[:, :50], w.transpose(1, 2).contiguous().cuda().transpose(1, 2)),
        "sliced weights": (device[:, :50], torch.cat([w, w], 2).cuda()[:, :, :33]),
    }
    for what, (x, weight) in views.items():
        y = E.typed_projection(x, weight, ids.cuda(), bias=b.cuda())
        close(y, want["y"], tolerance["y"], what)
        x, weight = x.detach().requires_grad_(), weight.detach().requires_grad_()
        y = E.typed_projection(x, weight, ids.cuda(), bias=b.cuda())
        dx, dw = torch.autograd.grad(y, (x, weight), dy.cuda())
        close(dx, want["dx"], tolerance["dx"], what)
        close(dw, want["dw"], tolerance["dw"], what)
    # gradients that come in broadcast, and inputs that are
    ones = torch.ones(rows, 33, dtype=dtype)
    want, tolerance = typed_reference(wide[:1, :50].expand(rows, 50), w, ids, b, ones, dtype)
    row = device[:1, :50].clone().requires_grad_()
    weight = w.cuda().requires_grad_()
    y = E.typed_projection(row.expand(rows, 50), weight, ids.cuda(), bias=b.cuda())
    close(y, want["y"], tolerance["y"], "one row for all")
    (dw,) = torch.autograd.grad(y.sum(), (weight,))
    close(dw, want["dw"], tolerance["dw"], "one row for all")


@pytest.mark.gpu
def test_gradients_against_differences():
    """The projections are linear in every argument, so central differences of any width are exact but
    for rounding: |loss(+v) - loss(-v)| / 2 against the gradient along v."""
    rows, types, k, n, r = 300, 4, 24, 20, 3
    ids, (x, w, down, up, b, dy) = make(rows, types, (rows, k), (k, n), (types, k, r), (types, r, n),
                                        (n,), (rows, n), dtype=torch.float32, seed=5)
    types_ = ids.cuda()
    dy_ = dy.cuda()

    def loss(*leaves):
        y = E.adapted_projection(*leaves[:4], types_, bias=leaves[4], scale=0.7)
        return y, (y.double() * dy_.double()).sum()

    leaves = [v.cuda().requires_grad_() for v in (x, w, down, up, b)]
    grads = torch.autograd.grad(loss(*leaves)[0], leaves, dy_)
    # every y is off by at most (k + r + 8) U of its terms; generous: each |y| term below 200
    bound = 2 * (k + r + 8) * U * 200 * float(dy.abs().sum())
    for i, grad in enumerate(grads):
        v = torch.randn(grad.shape, generator=torch.Generator().manual_seed(i)).cuda()
        with torch.no_grad():
            plus, minus = ([p + s * v if j == i else p for j, p in enumerate(leaves)] for s in (1, -1))
            difference = float(loss(*plus)[1] - loss(*minus)[1]) / 2
        along = float((grad.double() * v.double()).sum())
        assert abs(difference - along) <= bound, (i, difference, along, bound)


# --------------------------------------------------------------------------- adapted projection
ADAPTED = [  # rows, types, inputs, outputs, rank, skew
    (1, 1, 1, 1, 1, False), (1, 4, 64, 64, 8, False), (33, 64, 128, 96, 16, False),
    (50, 3, 100, 100, 5, False), (64, 2, 33, 40, 33, False), (130, 200, 40, 70, 16, False),
    (700, 3, 100, 130, 64, True), (1500, 1, 65, 33, 7, False), (4000, 37, 128, 128, 16, True),
    (2100, 900, 50, 64, 4, False), (3000, 6, 200, 32, 32, True), (300, 4, 40, 1, 20, False),
    (300, 4, 1, 40, 20, False), (150, 3, 1, 1, 1, False), (400, 3, 300, 1, 1, False),
    (400, 3, 1, 300, 1, False), (500, 4, 300, 260, 16, False), (260, 5, 140, 130, 9, True),
    (1600, 7, 90, 90, 8, True), (1200, 3, 170, 80, 16, False),
    # rows of 300 elements: some runs of one type a tile, and nearly as many types as rows
    (800, 100, 300, 40, 8, False), (600, 500, 300, 70, 20, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,types,inputs,outputs,rank,skew", ADAPTED)
def test_adapted_projection_and_its_gradients(rows, types, inputs, outputs, rank, skew, dtype):
    ids, (x, w, down, up, b, dy) = make(
        rows, types, (rows, inputs), (inputs, outputs), (types, inputs, rank), (types, rank, outputs),
        (outputs,), (rows, outputs), dtype=dtype, seed=rows, skew=skew)
    scale = 0.5
    want, tolerance = adapted_reference(x, w, down, up, ids, b, scale, dy, dtype)
    plan = E.TypePlan(ids.cuda(), types)
    with torch.no_grad():
        for t in (ids.cuda(), plan):
            y = E.adapted_projection(x.cuda(), w.cuda(), down.cuda(), up.cuda(), t, bias=b.cuda(),
                                     scale=scale)
            close(y, want["y"], tolerance["y"], "forward")
    leaves = [v.cuda().requires_grad_() for v in (x, w, down, up, b)]
    names = ("dx", "dw", "d_down", "d_up", "db")
    both = []
    for _ in range(2):
        y = E.adapted_projection(*leaves[:4], plan, bias=leaves[4], scale=scale)
        both.append((y, *torch.autograd.grad(y, leaves, dy.cuda())))
    assert all(torch.equal(a, b) for a, b in zip(*both))
    for name, got in zip(("y",) + names, both[0]):
        close(got, want[name], tolerance[name], name)
    # frozen projection, and the bias alone
    y = E.adapted_projection(leaves[0], w.cuda(), leaves[2], leaves[3], plan, scale=scale)
    for name, got in zip(("dx", "d_down", "d_up"),
                         torch.autograd.grad(y, (leaves[0], leaves[2], leaves[3]), dy.cuda())):
        close(got, want[name], tolerance[name], name)
    y = E.adapted_projection(x.cuda(), w.cuda(), down.cuda(), up.cuda(), plan, bias=leaves[4])
    close(torch.autograd.grad(y, leaves[4], dy.cuda())[0], want["db"], tolerance["db"], "db")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [9, 400])
def test_rows_without_an_adapter_get_the_shared_part(rows, dtype):
    ids, (x, w, down, up, b) = make(rows, 3, (rows, 30), (30, 28), (3, 30, 4), (3, 4, 28), (28,),
                                    dtype=dtype)
    ids[:] = -1
    down[:], up[:] = float("nan"), float("nan")  # nobody reads them
    zero = torch.zeros(3, 30, 4)
    want, tolerance = adapted_reference(x, w, zero, zero.transpose(1, 2)[:, :, :28], ids, b, 1.0,
                                        dtype=dtype)
    y = E.adapted_projection(x.cuda(), w.cuda(), down.cuda(), up.cuda(), ids.cuda(), bias=b.cuda())
    close(y, want["y"], tolerance["y"], "shared part")
    leaves = [v.cuda().requires_grad_() for v in (x, down, up)]
    y = E.adapted_projection(leaves[0], w.cuda(), leaves[1], leaves[2], ids.cuda())
    dx, d_down, d_up = torch.autograd.grad(y.sum(), leaves)
    assert bool((d_down == 0).all()) and bool((d_up == 0).all()) and not torch.isnan(dx).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("inputs,rank", [(40, 5), (40, 20), (300, 5)])
def test_a_types_infinities_reach_no_other_type(rows, inputs, rank, dtype):
    """Adapters that hold infinities or NaN, forward and backward: rows, and gradients, of the other
    types are what they are without them."""
    ids, (x, w, down, up, b, dy) = make(rows, 3, (rows, inputs), (inputs, 70), (3, inputs, rank),
                                        (3, rank, 70), (70,), (rows, 70), dtype=dtype)
    want, tolerance = adapted_reference(x, w, down, up, ids, b, 1.0, dy, dtype)
    for value, place in ((float("inf"), up), (float("nan"), down)):
        kept = place[1].clone()
        place[1] = value
        leaves = [v.cuda().requires_grad_() for v in (x, down, up)]
        y = E.adapted_projection(leaves[0], w.cuda(), leaves[1], leaves[2], ids.cuda(), bias=b.cuda())
        dx, d_down, d_up = torch.autograd.grad(y, leaves, dy.cuda())
        others = ids != 1
        with torch.no_grad():
            few = E.adapted_projection(leaves[0], w.cuda(), leaves[1], leaves[2], ids.cuda(), bias=b.cuda())
        for name, got in (("y", y), ("y", few), ("dx", dx)):
            close(got[others.cuda()], want[name][others], tolerance[name][others], name)
            assert not torch.isfinite(got[~others.cuda()]).any()
        for name, got in (("d_down", d_down), ("d_up", d_up)):
            close(got[[0, 2]], want[name][[0, 2]], tolerance[name][[0, 2]], name)
        place[1] = kept


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("inputs,rank", [(40, 5), (40, 20), (300, 5)])
def test_an_infinite_element_gives_infinities(rows, inputs, rank, dtype):
    """All weights are positive, so an infinite element of a row makes infinities of its products, and
    no NaN: not by the padding of the rank and not by the two parts of a low-rank row."""
    ids, (x, w, down, up, dy) = make(rows, 3, (rows, inputs), (inputs, 70), (3, inputs, rank),
                                     (3, rank, 70), (rows, 70), dtype=dtype, unknown=0.0)
    w, down, up, dy = (v.abs() + 0.5 for v in (w, down, up, dy))
    x[7, 3] = float("inf")
    t = int(ids[7])
    leaves = [v.cuda().requires_grad_() for v in (x, w, down, up)]
    y = E.adapted_projection(*leaves, ids.cuda())
    with torch.no_grad():
        few = E.adapted_projection(*leaves, ids.cuda())
    for got in (y, few):
        assert bool((got[7] == float("inf")).all()) and bool(torch.isfinite(got[:7]).all())
        assert bool(torch.isfinite(got[8:]).all())
    dx, dw, d_down, d_up = torch.autograd.grad(y, leaves, dy.cuda())
    assert bool(torch.isfinite(dx).all())
    for got, infinite in ((dw, dw[3]), (d_down, d_down[t, 3]), (d_up, d_up[t])):
        assert bool((infinite == float("inf")).all())
        assert int((~torch.isfinite(got)).sum()) == infinite.numel()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_adapted_projection_of_transposed_weights(dtype):
    for rows in (20, 300):
        ids, (x, w, down, up, b, dy) = make(rows, 5, (rows, 36), (36, 44), (5, 36, 6), (5, 6, 44),
                                            (44,), (rows, 44), dtype=dtype)
        want, tolerance = adapted_reference(x, w, down, up, ids, b, 1.0, dy, dtype)
        turn = lambda v: v.transpose(-1, -2).contiguous().cuda().transpose(-1, -2)  # noqa: E731
        leaves = [v.requires_grad_() for v in (x.cuda(), turn(w), turn(down), turn(up), b.cuda())]
        y = E.adapted_projection(*leaves[:4], ids.cuda(), bias=leaves[4])
        close(y, want["y"], tolerance["y"], "transposed")
        with torch.no_grad():
            close(E.adapted_projection(*leaves[:4], ids.cuda(), bias=leaves[4]), want["y"],
                  tolerance["y"], "transposed, no gradient")
        for name, got in zip(("dx", "dw", "d_down", "d_up", "db"),
                             torch.autograd.grad(y, leaves, dy.cuda())):
            close(got, want[name], tolerance[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inputs", [40, 300])
def test_scaled_product_at_the_c_boundary(inputs, dtype):
    """The C structure has a scale for the typed product too: of the product, not of the bias."""
    ids, (x, w, b) = make(50, 4, (50, inputs), (4, inputs, 36), (4, 36), dtype=dtype)
    scaled = w.float() * 0.25  # exact
    want, tolerance = typed_reference(x, scaled.to(dtype), ids, b, dtype=dtype)
    x, w, b, ids = x.cuda(), w.cuda(), b.cuda(), ids.cuda()
    plan, y = E.TypePlan(ids, 4), torch.empty((50, 36), dtype=dtype, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for few in (False, True):
        y.fill_(float("nan"))
        io, _ = module._product_io(x, inputs, module._weights(w)[1], y, 36, 4, b, None if few else plan,
                                   ids if few else None, scale=0.25)
        call = _lib.lib().gn2v_few_rows_product if few else _lib.lib().gn2v_typed_product
        _lib.check(call(io, stream))
        close(y, want["y"], tolerance["y"], few)


# ---------------------------------------------------------------------- streams, graphs, devices
@pytest.mark.gpu
def test_side_stream_and_plan_of_other_sizes():
    ids, (x, w, b) = make(400, 6, (400, 48), (6, 48, 40), (6, 40), dtype=torch.float32)
    want, tolerance = typed_reference(x, w, ids, b)
    side = torch.cuda.Stream()
    x, w, b, t = x.cuda(), w.cuda(), b.cuda(), ids.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = E.typed_projection(x, w, t, bias=b)
    side.synchronize()
    close(y, want["y"], tolerance["y"], "side stream")
    plan = E.TypePlan(t, 6)
    with pytest.raises(ValueError, match="plan is for 6 types"):
        E.typed_projection(x, w[:5], plan)
    with pytest.raises(ValueError, match="400 rows"):
        E.typed_projection(x[:10], w, plan)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [12, 2000])
def test_captured_steps_follow_their_inputs(rows):
    """Forward and backward in a graph, replayed on other rows, types and weights, with eager work and
    waits between the replays."""
    types, k, n, r = 9, 40, 36, 5
    draw = lambda seed: make(rows, types, (rows, k), (types, k, n), (types, n), (rows, n), (k, n),  # noqa: E731
                             (types, k, r), (types, r, n), dtype=torch.float32, seed=seed)

    def step(ids, x, w, b, dy, shared, down, up):
        leaves = [v.detach().requires_grad_() for v in (x, w, b, shared, down, up)]
        y = E.typed_projection(leaves[0], leaves[1], ids, bias=leaves[2])
        z = E.adapted_projection(leaves[0], leaves[3], leaves[4], leaves[5], ids)
        out = [y.detach(), z.detach(), *torch.autograd.grad((y, z), leaves, (dy, dy))]
        with torch.no_grad():
            out.append(E.typed_projection(x, w, ids, bias=b))
            out.append(E.adapted_projection(x, shared, down, up, ids))
        return out

    ids, rest = draw(0)
    state = [ids.cuda(), *(v.cuda() for v in rest)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*state)
    for seed in (1, 2, 3, 1):
        ids, rest = draw(seed)
        for old, new in zip(state, [ids, *rest]):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(*state)
        assert all(torch.equal(a, b) for a, b in zip(captured, eager)), seed


@pytest.mark.gpu
def test_a_run_from_the_table_to_the_loss():
    """A typed graph's table through the layers as they are used together: 8-bit table, typed
    projection of its nodes, edge features of the projected rows, adapters per edge type, a step."""
    rng = np.random.RandomState(0)
    src, dst = rng.randint(0, 200, 900), rng.randint(0, 200, 900)
    g = E.CSRGraph.from_edge_list(src, dst, number_of_nodes=200, node_types=[f"t{i % 3}" for i in range(200)],
                                  edge_types=[f"r{i % 5}" for i in range(900)])
    model = E.Node2VecSkipGramEnsmallen(embedding_size=32, epochs=1, iterations=1, walk_length=16,
                                        verbose=False)
    central = model._model.fit_transform_device(g)[0]
    table = E.QuantizedTable.from_table(central, group_size=32)
    nodes, edges = E.TypePlan.from_graph(g), E.TypePlan.from_graph(g, "edges")
    gen = torch.Generator().manual_seed(1)
    w = (torch.randn(3, 32, 24, generator=gen) * 0.2).cuda().requires_grad_()
    shared = (torch.randn(24, 8, generator=gen) * 0.2).cuda()
    down = (torch.randn(5, 24, 4, generator=gen) * 0.2).cuda().requires_grad_()
    up = (torch.randn(5, 4, 8, generator=gen) * 0.2).cuda().requires_grad_()
    s = torch.from_numpy(g.get_directed_source_node_ids().astype(np.int64)).cuda()
    d = torch.from_numpy(g.get_destination_node_ids().astype(np.int64)).cuda()
    x = table.read()
    assert float((x - central).abs().max()) <= float(central.abs().max()) / 254 * 1.001
    h = E.typed_projection(x, w, nodes)
    z = E.adapted_projection(h[s] * h[d], shared, down, up, edges)
    loss = (z * z).mean()
    loss.backward()
    # the same in 64 bits
    node_ids = torch.from_numpy(g.node_type_ids.astype(np.int64))
    edge_ids = torch.from_numpy(g.edge_type_ids.astype(np.int64))
    ref = [v.detach().cpu().double().requires_grad_() for v in (w, down, up)]
    hr = torch.bmm(x.cpu().double()[:, None], ref[0][node_ids])[:, 0]
    e = hr[s.cpu()] * hr[d.cpu()]
    zr = e @ shared.cpu().double() + torch.bmm(torch.bmm(e[:, None], ref[1][edge_ids]),
                                               ref[2][edge_ids])[:, 0]
    (zr * zr).mean().backward()
    for got, want in zip((w, down, up), ref):
        # sums of up to 900 x 24 products behind one another, relative to the largest element
        off = float((got.grad.cpu().double() - want.grad).abs().max() / want.grad.abs().max())
        assert off <= 900 * 24 * U, off
    features = E.edge_embedding(table, s, d, "Hadamard")
    assert torch.equal(features, x[s] * x[d])

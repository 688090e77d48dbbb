"""What the projections refuse, and how they behave at the ends of what they allow: forward-mode
derivatives, many tiles a workgroup, sizes that pass 32 bits, other streams."""
import copy
import ctypes as C
import pickle

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import embiggen_amd as E
from embiggen_amd import _lib
from embiggen_amd.embedding_transformers import projections as module


class NoLaunches:
    """In place of the library: every entry point succeeds and computes nothing."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def on_the_cpu(monkeypatch):
    """Calls on CPU tensors run up to the launches, which do nothing."""
    monkeypatch.setattr(module, "_check_device", lambda x: None)
    monkeypatch.setattr(module, "_stream", lambda x: 0)
    monkeypatch.setattr(module._lib, "lib", lambda: NoLaunches())
    monkeypatch.setattr(module, "_plan_words", lambda rows, types: (2 * rows + 2 * (types + 2), 0))
    monkeypatch.setattr(module, "_gradient_bytes", lambda *sizes: 16)


# ------------------------------------------------------------------------------ refusals (CPU)
@pytest.mark.parametrize("rows", [4, module.FEW_ROWS + 1])  # the form of few rows, and the other one
def test_forward_mode_derivatives_are_refused(on_the_cpu, rows):
    ids = torch.arange(rows) % 3 - 1
    typed = [torch.zeros(rows, 3), torch.zeros(2, 3, 5), torch.zeros(2, 5)]
    adapted = [torch.zeros(rows, 3), torch.zeros(3, 5), torch.zeros(2, 3, 2), torch.zeros(2, 2, 5), torch.zeros(5)]

    def run(tensors):
        if len(tensors) == 3:
            return E.typed_projection(tensors[0], tensors[1], ids, bias=tensors[2])
        return E.adapted_projection(*tensors[:4], ids, bias=tensors[4])

    for tensors in (typed, adapted):
        with forward_ad.dual_level():
            assert run(tensors).shape == (rows, 5)  # nobody has a tangent
            for i, tensor in enumerate(tensors):
                dual = forward_ad.make_dual(tensor, torch.ones_like(tensor))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    run([dual if i == j else t for j, t in enumerate(tensors)])
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                    run([dual if i == j else t for j, t in enumerate(tensors)])
            # a gradient that comes in with a tangent would leave without one
            leaves = [t.clone().requires_grad_() for t in tensors]
            dy = forward_ad.make_dual(torch.ones(rows, 5), torch.ones(rows, 5))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(run(leaves), leaves, dy)
        leaves = [t.clone().requires_grad_() for t in tensors]
        grads = torch.autograd.grad(run(leaves), leaves, torch.ones(rows, 5))
        assert [g.shape for g in grads] == [t.shape for t in tensors]
        twice = torch.autograd.grad(run(leaves), leaves, torch.ones(rows, 5).requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            twice[0].sum().backward()


def test_a_plan_is_where_its_words_are(on_the_cpu):
    """A stored plan may be loaded onto another device than it was made on."""
    plan = E.TypePlan(torch.tensor([0, 1, -1]), 2)
    x, w = torch.zeros(3, 4), torch.zeros(2, 4, 5)
    assert E.typed_projection(x, w, plan).shape == (3, 5)
    plan._words = plan._words.to("meta")
    with pytest.raises(ValueError, match="types are on meta"):
        E.typed_projection(x, w, plan)
    with pytest.raises(ValueError, match="types are on meta"):
        E.adapted_projection(x, w[0], torch.zeros(2, 4, 1), torch.zeros(2, 1, 5), plan)


def test_scales_that_are_no_numbers_are_refused(on_the_cpu):
    tensors = [torch.zeros(3, 4), torch.zeros(4, 5), torch.zeros(2, 4, 1), torch.zeros(2, 1, 5), torch.tensor([0, 1, -1])]
    for scale in (None, "half", torch.ones(2), torch.tensor(0.5, requires_grad=True)):
        with pytest.raises(ValueError, match="scale"):
            E.adapted_projection(*tensors, scale=scale)
    for scale in (2, 0.5, torch.tensor(0.5), np.float64(0.25)):
        assert E.adapted_projection(*tensors, scale=scale).shape == (3, 5)


def test_launches_of_too_many_threads_are_refused():
    """A launch holds fewer than 2^32 threads: 2^24 workgroups of 256, one per 64 rows of the low-rank rows."""
    rows = (1 << 30) + (1 << 20)
    io = _lib.ProductIO(dtype=1, n_types=2, rows=rows, inputs=8, outputs=4, ldx=8, ldy=4, low_rank_rows=1,
                        d_x=4096, d_y=4096, d_plan=4096)
    io.weight = _lib.Weights(4096, 32, 4, 1)
    L = _lib.lib()
    assert L.gn2v_typed_product(C.byref(io), None) == 1 and b"too many rows" in L.gn2v_last_error()
    io.low_rank_rows, io.inputs, io.ldx, io.weight.inner = 0, 600, 600, 4
    assert L.gn2v_typed_product(C.byref(io), None) == 1 and b"too many rows" in L.gn2v_last_error()


# ------------------------------------------------------------------------------------ large sizes
@pytest.mark.gpu
def test_gradients_whose_join_fills_more_than_one_launch():
    """16 types of 8 192 x 8 192: the sums of 2^30 weights are joined by more threads than a launch holds,
    and types without rows get their zeros there."""
    types, size = 16, 8192
    gen = torch.Generator().manual_seed(0)
    ids = torch.tensor([0, 3, 3, 15, -1, 9, 0, 3, 15, 15, 1, 16])
    x, dy = (torch.randn(len(ids), size, generator=gen).bfloat16().cuda() for _ in range(2))
    w = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(types, size, size).contiguous().requires_grad_()
    y = E.typed_projection(x, w, ids.cuda())
    assert bool((y == 0).all())
    (dw,) = torch.autograd.grad(y, w, dy)
    for t in range(types):
        at = (ids == t).nonzero().squeeze(1).cuda()
        if not len(at):
            assert bool((dw[t] == 0).all()), t
            continue
        a, b = x[at].double(), dy[at].double()
        want, terms = a.T @ b, a.abs().T @ b.abs()
        # a float32 sum of len(at) products, rounded to bfloat16
        tolerance = (len(at) + 2) * 2.0 ** -24 * terms + 2.0 ** -8 * want.abs()
        assert bool(((dw[t].double() - want).abs() <= tolerance).all()), t


# ------------------------------------------------------------------- many tiles a workgroup, exactly
# Rows, weights and gradients are small whole numbers and the scale is a power of two, so that every sum is
# exact in float32, in any order (its terms' magnitudes add up to less than 2^24), and so are the two
# bfloat16 parts of a low-rank row (whole numbers below 2^16, halved).  Results equal the definition in 64
# bits, rounded once.
def whole(gen, most, *shape):
    return torch.randint(-most, most + 1, shape, generator=gen, dtype=torch.int8).double()


def skewed_types(gen, rows, types):
    """A few common types, a tail of rare ones and rows without a type."""
    ids = (torch.rand(rows, generator=gen) ** 3 * types).long().clamp_(max=types - 1)
    ids[torch.rand(rows, generator=gen) < 0.03] = -1
    return ids


def rounded(value, dtype):
    assert float(value.abs().max()) < 2 ** 24
    return value.float().to(dtype)


def same(got, want, what):
    got = got.cpu()
    assert got.shape == want.shape and got.dtype == want.dtype, what
    other = (got != want).nonzero()  # NaN is another value
    if len(other):
        at = tuple(other[0].tolist())
        raise AssertionError(f"{what}: {len(other)} of {got.numel()} differ, first {at}: {got[at]!r}, not {want[at]!r}")


def exact_steps(x, ids, dy, weight=None, bias=None, shared=None, down=None, up=None, scale=0.5):
    """Results and gradients in 64 bits: of the typed form (weight, bias by type) or of the adapted one
    (shared, bias, down, up)."""
    out = {}
    if weight is not None:
        out["y"], out["dx"] = x.new_zeros(len(x), weight.shape[2]), torch.zeros_like(x)
        out["dw"], out["db"] = torch.zeros_like(weight), torch.zeros_like(bias)
    else:
        out["y"], out["dx"] = x @ shared + bias, dy @ shared.T
        out["dw"], out["d_down"], out["d_up"] = x.T @ dy, torch.zeros_like(down), torch.zeros_like(up)
        out["db"] = dy.sum(0)
    for t in range(len(weight if weight is not None else down)):
        at = (ids == t).nonzero().squeeze(1)
        xt, dyt = x[at], dy[at]
        if weight is not None:
            out["y"][at], out["dx"][at] = xt @ weight[t] + bias[t], dyt @ weight[t].T
            out["dw"][t], out["db"][t] = xt.T @ dyt, dyt.sum(0)
        else:
            low, back = scale * xt @ down[t], scale * dyt @ up[t].T
            out["y"][at] += low @ up[t]
            out["dx"][at] += back @ down[t].T
            out["d_down"][t], out["d_up"][t] = xt.T @ back, low.T @ dyt
    return out


def run_steps(x, ids, dy, weight=None, bias=None, shared=None, down=None, up=None, scale=0.5):
    if weight is not None:
        leaves = [v.clone().requires_grad_() for v in (x, weight, bias)]
        y = E.typed_projection(leaves[0], leaves[1], ids, bias=leaves[2])
        names = ("dx", "dw", "db")
    else:
        leaves = [v.clone().requires_grad_() for v in (x, shared, down, up, bias)]
        y = E.adapted_projection(*leaves[:4], ids, bias=leaves[4], scale=scale)
        names = ("dx", "dw", "d_down", "d_up", "db")
    return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, leaves, dy)))}


def check_steps(dtype, ids, **tensors):
    want = exact_steps(ids=ids, **tensors)
    plan = E.TypePlan(ids.cuda(), len(tensors["weight" if "weight" in tensors else "down"]))
    device = {name: v.to(dtype).cuda() for name, v in tensors.items()}
    got, again = run_steps(ids=plan, **device), run_steps(ids=ids.int().cuda(), **device)
    for name, value in want.items():
        same(got[name], rounded(value, dtype), name)
        same(again[name], got[name].cpu(), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,types,inputs,outputs", [
    # 3 438 tiles: seven a workgroup of the product, three of the gradients' 1 024
    (220_001, 5, 16, 16), (150_003, 301, 90, 40), (130_001, 6, 100, 71), (140_000, 4, 128, 128), (100_001, 9, 192, 70),
    # nine blocks of columns, 64 workgroups each
    (15_001, 3, 40, 1100),
    # longer rows: 141 tiles of gradients for 32 workgroups a block; outputs above the widest block of columns
    (9_001, 4, 512, 512), (700, 3, 300, 257), (1_400, 5, 520, 390), (2_000, 1, 260, 150)])
def test_typed_steps_of_many_tiles(rows, types, inputs, outputs, dtype):
    gen = torch.Generator().manual_seed(rows + outputs)
    ids = skewed_types(gen, rows, types)
    check_steps(dtype, ids, x=whole(gen, 2, rows, inputs), dy=whole(gen, 2, rows, outputs),
                weight=whole(gen, 3, types, inputs, outputs), bias=whole(gen, 5, types, outputs))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,types,inputs,outputs,rank", [
    # 2 500 tiles: five a workgroup of the products, three to five of the gradients
    (160_001, 5, 16, 16, 3), (150_003, 237, 64, 40, 8), (110_001, 5, 128, 128, 16), (110_001, 7, 100, 33, 5),
    (100_001, 4, 256, 30, 16), (12_001, 3, 64, 1100, 4),
    # longer rows or ranks
    (20_001, 6, 300, 40, 20), (1_400, 4, 520, 390, 16), (1_200, 100, 260, 150, 40), (60_001, 5, 40, 48, 33)])
def test_adapted_steps_of_many_tiles(rows, types, inputs, outputs, rank, dtype):
    gen = torch.Generator().manual_seed(rows + outputs)
    ids = skewed_types(gen, rows, types)
    check_steps(dtype, ids, x=whole(gen, 1, rows, inputs), dy=whole(gen, 1, rows, outputs),
                shared=whole(gen, 3, inputs, outputs), bias=whole(gen, 5, outputs),
                down=whole(gen, 1, types, inputs, rank), up=whole(gen, 1, types, rank, outputs))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_frozen_and_single_gradients_of_many_tiles(dtype):
    """The corrections alone (one pass over the rows without the shared weight's sums), and each gradient by itself."""
    gen = torch.Generator().manual_seed(3)
    rows, types, inputs, outputs, rank = 120_001, 40, 100, 96, 5
    ids = skewed_types(gen, rows, types)
    tensors = dict(x=whole(gen, 1, rows, inputs), dy=whole(gen, 1, rows, outputs), shared=whole(gen, 3, inputs, outputs),
                   bias=whole(gen, 5, outputs), down=whole(gen, 1, types, inputs, rank),
                   up=whole(gen, 1, types, rank, outputs))
    want = {name: rounded(v, dtype) for name, v in exact_steps(ids=ids, **tensors).items()}
    device = {name: v.to(dtype).cuda() for name, v in tensors.items()}
    plan = E.TypePlan(ids.cuda(), types)
    order = ["x", "shared", "down", "up", "bias"]
    gradients = dict(zip(order, ("dx", "dw", "d_down", "d_up", "db")))
    for wanted in (["x", "down", "up"], ["down", "up"], ["x"], ["down"], ["up"], ["shared"], ["bias"], ["down", "up", "bias"]):
        leaves = {name: device[name].clone().requires_grad_(name in wanted) for name in order}
        y = E.adapted_projection(*(leaves[name] for name in order[:4]), plan, bias=leaves["bias"], scale=0.5)
        same(y.detach(), want["y"], "y")
        for name, got in zip(wanted, torch.autograd.grad(y, [leaves[name] for name in wanted], device["dy"])):
            same(got, want[gradients[name]], (wanted, name))


# ------------------------------------------------------------- the two parts of a low-rank row (bfloat16)
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("inputs,rank", [(40, 5), (40, 20), (300, 5)])
def test_small_low_rank_rows_keep_their_value(rows, inputs, rank):
    """Low-rank rows of 2^-120 times weights, rows and gradients of 2^120: one, and no part of theirs added."""
    ids = torch.arange(rows) % 3
    outputs, small, large, dtype = 70, 2.0 ** -60, 2.0 ** 120, torch.bfloat16
    counts = torch.bincount(ids).to(dtype)  # at most 100: exact
    x, w, dy = torch.zeros(rows, inputs), torch.zeros(inputs, outputs), torch.zeros(rows, outputs)
    down, up = torch.zeros(3, inputs, rank), torch.zeros(3, rank, outputs)
    x[:, 0], down[:, 0, 0], up[:, 0], dy[:] = small, small, large, large
    x, w, down, up, dy = (v.to(dtype).cuda() for v in (x, w, down, up, dy))
    one = torch.ones(rows, outputs, dtype=dtype)
    with torch.no_grad():
        same(E.adapted_projection(x, w, down, up, ids.cuda()), one, "forward")
    leaf = up.clone().requires_grad_()
    y = E.adapted_projection(x, w, down, leaf, ids.cuda())
    same(y.detach(), one, "y")
    (d_up,) = torch.autograd.grad(y, leaf, dy)
    same(d_up[:, 0], counts[:, None].expand(3, outputs), "d_up")
    assert bool((d_up[:, 1:] == 0).all())
    # the way back: dy up^T is 2^-120
    x, down, up, dy = (torch.zeros_like(v) for v in (x, down, up, dy))
    x[:], down[:, :, 0], up[:, 0, 0], dy[:, 0] = large, large, small, small
    leaves = [v.requires_grad_() for v in (x, down)]
    dx, d_down = torch.autograd.grad(E.adapted_projection(x, w, down, up, ids.cuda()), leaves, dy)
    same(dx, torch.ones(rows, inputs, dtype=dtype), "dx")
    same(d_down[:, :, 0], counts[:, None].expand(3, inputs), "d_down")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 300])
@pytest.mark.parametrize("inputs,rank", [(40, 5), (40, 20), (300, 5)])
def test_small_low_rank_rows_times_infinity(rows, inputs, rank):
    """Low-rank rows that take two parts, the second of them too small for a normal number."""
    ids = torch.arange(rows) % 3
    x, down = torch.zeros(rows, inputs), torch.zeros(3, inputs, rank)
    x[:, 0], down[:, 0] = 2.0 ** -62 * (1 + 2.0 ** -7), 2.0 ** -60 * (1 + 2.0 ** -7)
    up = torch.full((3, rank, 70), float("inf"))
    x, w, down, up = (v.bfloat16().cuda() for v in (x, torch.zeros(inputs, 70), down, up))
    with torch.no_grad():
        assert bool((E.adapted_projection(x, w, down, up, ids.cuda()) == float("inf")).all())
    y = E.adapted_projection(x, w, down.requires_grad_(), up, ids.cuda())
    assert bool((y == float("inf")).all())


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows whose elements, read and written, lie more than 2^31 elements and 2^32 bytes behind the first; the sums of
    a type's millions of rows stay below 2^24."""
    rows, types, inputs, outputs, dtype = 17_000_000, 5, 24, 136, torch.bfloat16
    gen = torch.Generator(device="cuda").manual_seed(0)

    def draw(most, *shape):
        return torch.randint(-most, most + 1, shape, generator=gen, dtype=torch.int8, device="cuda").to(dtype)

    x = torch.zeros(rows, 128, dtype=dtype, device="cuda")[:, :inputs]  # rows of a padded table
    x.copy_(draw(1, rows, inputs))
    dy = draw(1, rows, outputs)
    w, b = draw(2, types, inputs, outputs), draw(3, types, outputs)
    ids = torch.randint(-1, types, (rows,), generator=gen, dtype=torch.int32, device="cuda")
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    y = E.typed_projection(leaves[0], leaves[1], ids, bias=leaves[2])
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    y = y.detach()
    for t in range(-1, types):
        at = (ids == t).nonzero().squeeze(1)
        if t < 0:
            assert bool((y[at] == 0).all()) and bool((dx[at] == 0).all())
            continue
        sums = torch.zeros(inputs, outputs, dtype=torch.float64, device="cuda")
        for part in at.split(1 << 20):
            xt, dyt = x[part].double(), dy[part].double()
            assert torch.equal(y[part], rounded(xt @ w[t].double() + b[t].double(), dtype)), t
            assert torch.equal(dx[part], rounded(dyt @ w[t].double().T, dtype)), t
            sums += xt.T @ dyt
        assert torch.equal(dw[t], rounded(sums, dtype)), t
        assert torch.equal(db[t], rounded(dy[at].double().sum(0), dtype)), t


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [700, 40_000])
def test_forward_and_backward_on_a_side_stream(rows):
    gen = torch.Generator().manual_seed(1)
    ids = skewed_types(gen, rows, 6)
    tensors = dict(x=whole(gen, 1, rows, 64), dy=whole(gen, 1, rows, 48), shared=whole(gen, 3, 64, 48),
                   bias=whole(gen, 5, 48), down=whole(gen, 1, 6, 64, 4), up=whole(gen, 1, 6, 4, 48))
    want = exact_steps(ids=ids, **tensors)
    device = {name: v.float().cuda() for name, v in tensors.items()}
    types = ids.cuda()
    here = run_steps(ids=types, **device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = run_steps(ids=types, **device)
    # forward on the side stream, backward called from this one: it runs where the forward did
    with torch.cuda.stream(side):
        x = device["x"].clone().requires_grad_()
        y = E.adapted_projection(x, device["shared"], device["down"], device["up"], types, bias=device["bias"], scale=0.5)
    torch.cuda.current_stream().wait_stream(side)
    (dx,) = torch.autograd.grad(y, x, device["dy"])
    torch.cuda.synchronize()
    for name, value in want.items():
        same(here[name], rounded(value, torch.float32), name)
        same(there[name], here[name].cpu(), name)
    same(dx, here["dx"].cpu(), "dx")
    same(y.detach(), here["y"].cpu(), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [700, 40_000])
def test_the_memory_of_a_plan_waits_for_the_streams_that_read_it(rows):
    """A plan that goes out of scope while another stream has yet to use it: its words are row ids, and whoever gets
    their memory would send the kernels anywhere."""
    gen = torch.Generator().manual_seed(2)
    ids = skewed_types(gen, rows, 6)
    x, w = whole(gen, 1, rows, 64).float().cuda(), whole(gen, 2, 6, 64, 48).float().cuda()
    want = E.typed_projection(x, w, ids.cuda())
    a = torch.zeros(4096, 4096, device="cuda")
    side = torch.cuda.Stream()
    plan = E.TypePlan(ids.cuda(), 6)
    words, at = plan._words.numel(), plan._words.data_ptr()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(40):  # some 40 ms of work before the projection
            a = a @ a
        y = E.typed_projection(x, w, plan)
    del plan
    others = [torch.empty(words, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not side.query(), "the side stream is still at work"
    assert at not in [other.data_ptr() for other in others]
    side.synchronize()
    same(y, want.cpu(), "y")
    # a copy's words lie elsewhere, whatever stream is the current one
    plan = E.TypePlan(ids.cuda(), 6)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = [copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))]
        side.synchronize()
    for other in again:
        assert torch.equal(other.order, plan.order) and torch.equal(other.offsets, plan.offsets)
        same(E.typed_projection(x, w, other), want.cpu(), "copy")


@pytest.mark.gpu
def test_steps_captured_around_a_plan_made_before():
    gen = torch.Generator().manual_seed(4)
    rows, types = 3_000, 6
    ids = skewed_types(gen, rows, types)
    plan = E.TypePlan(ids.cuda(), types)
    draw = lambda: dict(x=whole(gen, 1, rows, 64), dy=whole(gen, 1, rows, 48), shared=whole(gen, 3, 64, 48),  # noqa: E731
                        bias=whole(gen, 5, 48), down=whole(gen, 1, types, 64, 4), up=whole(gen, 1, types, 4, 48))
    state = {name: v.float().cuda() for name, v in draw().items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_steps(ids=plan, **state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run_steps(ids=plan, **state)
    for _ in range(3):
        tensors = draw()
        for name, v in tensors.items():
            state[name].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for name, value in exact_steps(ids=ids, **tensors).items():
            same(captured[name], rounded(value, torch.float32), name)
    del plan, graph
    torch.cuda.synchronize()
    same(E.TypePlan(ids.cuda(), types).order, torch.argsort(torch.where(ids < 0, types, ids), stable=True).int(), "order")

"""What the projections refuse, and how they behave at the ends of what they allow: forward-mode
derivatives, many tiles a workgroup, sizes that pass 32 bits, other streams."""
import ctypes as C

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


# ------------------------------------------------------------- the two parts of a low-rank row (bfloat16)
def same(got, want, what):
    got = got.cpu()
    assert got.shape == want.shape and got.dtype == want.dtype, what
    other = (got != want).nonzero()  # NaN is another value
    if len(other):
        at = tuple(other[0].tolist())
        raise AssertionError(f"{what}: {len(other)} of {got.numel()} differ, first {at}: {got[at]!r}, not {want[at]!r}")


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

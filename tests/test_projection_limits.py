"""What the projections refuse, and how they behave at the ends of what they allow: forward-mode
derivatives, many tiles a workgroup, sizes that pass 32 bits, other streams."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import embiggen_amd as E
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

"""Projections of embedding rows by their type.

The rows of a typed graph's embedding table (or of its edges' embeddings) go through the weights of
their node or edge type, or through one shared projection plus a low-rank correction of their type --
an adapter.  The reference's classifiers treat types as one-hot columns beside the embedding
(embiggen/embedding_transformers/graph_transformer.py:196-243); here every type has weights of its own.
Both run in hand-written kernels that read the rows where they are: a *plan* (``TypePlan``) holds the
order of the rows by type, and no sorted copy of them is made.  Both can be differentiated; gradients
are summed in a fixed order, so a run gives the same bits every time.
"""
import ctypes as C
from typing import Optional, Union

from .. import _lib


def _torch():
    import torch

    return torch


def _check_rows(name: str, x, dims: int):
    torch = _torch()
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"The provided {name} should be a tensor, but we got {type(x)} instead.")
    if x.dim() != dims:
        raise ValueError(f"The provided {name} should have {dims} dimensions, but we got shape "
                         f"{tuple(x.shape)} instead.")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"The provided {name} should be float32 or bfloat16, but we got "
                         f"{x.dtype} instead.")


def _check_like(name: str, tensor, shape, x):
    _check_rows(name, tensor, len(shape))
    if tuple(tensor.shape) != tuple(shape):
        raise ValueError(f"The provided {name} should have shape {tuple(shape)}, but we got "
                         f"{tuple(tensor.shape)} instead.")
    if tensor.dtype != x.dtype or tensor.device != x.device:
        raise ValueError(f"The provided {name} should have the type and device of the rows "
                         f"({x.dtype}, {x.device}), but we got {tensor.dtype}, {tensor.device}.")


def _check_device(x):
    if x.device.type != "cuda":
        raise ValueError("The rows should be on a ROCm device (there is no CPU execution path), "
                         f"but they are on {x.device}.")


def _stream(x):
    return _torch().cuda.current_stream(x.device).cuda_stream


class TypePlan:
    """The order of rows by type: made once, used by every projection of the same rows.

    Parameters
    ------------------
    types
        int32 / int64 tensor on the device: the type id of every row.  -1 -- or any other id outside
        ``[0, number_of_types)`` -- is an unknown type.
    number_of_types: int
        How many types there are, 32 768 at most.
    """

    def __init__(self, types, number_of_types: int):
        torch = _torch()
        if not isinstance(types, torch.Tensor) or types.dim() != 1 or types.dtype not in (
                torch.int32, torch.int64):
            raise ValueError("The provided types should be a one-dimensional int32 or int64 tensor.")
        if not 1 <= number_of_types <= _lib.MAX_TYPES:
            raise ValueError(f"The number of types should be between 1 and {_lib.MAX_TYPES}, but "
                             f"we got {number_of_types} instead.")
        _check_device(types)
        self.number_of_types = int(number_of_types)
        self.number_of_rows = types.numel()
        self.device = types.device
        words, temp_words = C.c_uint64(), C.c_uint64()
        L = _lib.lib()
        _lib.check(L.gn2v_type_plan_words(self.number_of_rows, self.number_of_types,
                                          C.byref(words), C.byref(temp_words)))
        types = types.contiguous()
        self._words = torch.empty(words.value, dtype=torch.int32, device=types.device)
        temp = torch.empty(temp_words.value, dtype=torch.int32, device=types.device)
        _lib.check(L.gn2v_type_plan(types.data_ptr(), types.element_size(), self.number_of_rows,
                                    self.number_of_types, self._words.data_ptr(), temp.data_ptr(),
                                    _stream(types)))

    @classmethod
    def from_graph(cls, graph, of: str = "nodes", device: int = 0) -> "TypePlan":
        """The plan of a typed graph's nodes (``of="nodes"``) or of its directed edges in CSR order
        (``of="edges"``); nodes with several labels count by their label set."""
        import numpy as np

        if of not in ("nodes", "edges"):
            raise ValueError(f"`of` should be 'nodes' or 'edges', but we got {of!r} instead.")
        ids = graph.node_type_ids if of == "nodes" else graph.edge_type_ids
        if ids is None:
            raise ValueError(f"The {of} of the graph do not have types.")
        ids = np.ascontiguousarray(ids, dtype=np.uint32).view(np.int32)
        count = max(1, int(ids.max(initial=-1)) + 1)
        return cls(_torch().from_numpy(ids).to(_torch().device("cuda", device)), count)

    @property
    def order(self):
        """int32 row ids in the order of their types, rows of one type in ascending order; rows of
        unknown types come last."""
        return self._words[:self.number_of_rows]

    @property
    def offsets(self):
        """int32 [number_of_types + 2]: where the rows of every type begin in ``order``, where those
        of unknown types do, and the number of rows."""
        first = 2 * self.number_of_rows
        return self._words[first:first + self.number_of_types + 2]


def _row_stride(x):
    """(tensor, elements between rows): the tensor itself where its rows lie apart."""
    if x.shape[1] > 1 and x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        if x.shape[0] == 1 and (x.shape[1] == 1 or x.stride(1) == 1):
            return x, x.shape[1]
        x = x.contiguous()
    return x, max(x.stride(0), x.shape[1])


def _weights(w, rows_contiguous: bool = False):
    """(tensor, gn2v_weights) of [inputs, outputs] or [types, inputs, outputs] weights: as they are
    where one of the two last strides is 1 (``rows_contiguous``: the last one), else a copy."""
    inner, outer = w.stride(-2), w.stride(-1)
    if w.shape[-1] == 1:
        outer = 1
    elif w.shape[-2] == 1 and outer != 1 and not rows_contiguous:
        inner = 1
    if outer != 1 and (rows_contiguous or inner != 1):
        w = w.contiguous()
        inner, outer = w.stride(-2), 1
    return w, _lib.Weights(w.data_ptr(), w.stride(0) if w.dim() == 3 else 0, inner, outer)


def _transposed(view):
    return _lib.Weights(view.d_data, view.type_stride, view.outer, view.inner)


def _dtype(x) -> int:
    return 0 if x.dtype == _torch().float32 else 1


def _product_io(x, ldx, weight, y, inputs, outputs, n_types):
    io = _lib.ProductIO()
    io.dtype, io.n_types, io.rows = _dtype(x), n_types, x.shape[0]
    io.inputs, io.outputs, io.scale = inputs, outputs, 1.0
    io.d_x, io.ldx, io.weight = x.data_ptr(), ldx, weight
    io.d_y, io.ldy = y.data_ptr(), y.shape[1]
    return io


def _set_bias(io, bias):
    if bias is not None:
        if bias.shape[-1] > 1 and bias.stride(-1) != 1:
            bias = bias.contiguous()
        io.d_bias = bias.data_ptr()
        io.bias_stride = bias.stride(0) if bias.dim() == 2 else 0
    return bias


def _typed_product(x, ldx, weight, plan, outputs, bias=None):
    y = _torch().empty((x.shape[0], outputs), dtype=x.dtype, device=x.device)
    io = _product_io(x, ldx, weight, y, x.shape[1], outputs, plan.number_of_types)
    io.d_plan = plan._words.data_ptr()
    bias = _set_bias(io, bias)
    _lib.check(_lib.lib().gn2v_typed_product(C.byref(io), _stream(x)))
    return y


def _adapted_product(x, ldx, weight, down, up, rank, scale, plan, outputs, bias=None, low=None):
    """``low``: float32 [rows, rank], filled with the low-rank rows at their positions in the plan's
    order; None where nobody needs them."""
    torch = _torch()
    if low is None and (rank > _lib.FUSED_RANK
                        or x.shape[1] * x.element_size() > _lib.FUSED_ROW_BYTES):
        low = torch.empty((x.shape[0], rank), dtype=torch.float32, device=x.device)
    y = torch.empty((x.shape[0], outputs), dtype=x.dtype, device=x.device)
    io = _product_io(x, ldx, weight, y, x.shape[1], outputs, plan.number_of_types)
    io.d_plan, io.down, io.up, io.rank, io.scale = plan._words.data_ptr(), down, up, rank, scale
    if low is not None:
        io.d_low = low.data_ptr()
    bias = _set_bias(io, bias)
    _lib.check(_lib.lib().gn2v_adapted_product(C.byref(io), _stream(x)))
    return y


def _low_rows(x, ldx, weight, plan, rank, scale):
    """scale * x[r] W[type of r] as float32 rows at their positions in the plan's order."""
    low = _torch().empty((x.shape[0], rank), dtype=_torch().float32, device=x.device)
    io = _product_io(x, ldx, weight, low, x.shape[1], rank, plan.number_of_types)
    io.d_plan, io.scale, io.low_rank_rows = plan._words.data_ptr(), scale, 1
    _lib.check(_lib.lib().gn2v_typed_product(C.byref(io), _stream(x)))
    return low


def _gradient(x, dy, plan, dw, db):
    """Fills dw [types, inputs, outputs] and db [types, outputs], those that are not None."""
    torch = _torch()
    x, ldx = _row_stride(x)
    io = _lib.GradientIO()
    io.dtype, io.n_types, io.rows = _dtype(x), plan.number_of_types, x.shape[0]
    io.d_x, io.ldx = x.data_ptr(), ldx
    if dw is not None:
        io.inputs, io.d_dw = x.shape[1], dw.data_ptr()
    dy, io.ldy = _row_stride(dy)
    io.outputs, io.d_dy, io.d_plan = dy.shape[1], dy.data_ptr(), plan._words.data_ptr()
    if db is not None:
        io.d_db = db.data_ptr()
    need = C.c_uint64()
    L = _lib.lib()
    _lib.check(L.gn2v_typed_gradient_temp(C.byref(io), C.byref(need)))
    temp = torch.empty(need.value, dtype=torch.uint8, device=dy.device)
    io.d_temp, io.temp_bytes = temp.data_ptr(), need.value
    _lib.check(L.gn2v_typed_gradient(C.byref(io), _stream(dy)))


def _adapted_gradient(x, dy, low, back, rank, plan, d_down, d_up, dw, db):
    """Fills the gradients that are not None."""
    torch = _torch()
    x, ldx = _row_stride(x)
    dy, ldy = _row_stride(dy)
    io = _lib.AdaptedGradientIO()
    io.dtype, io.n_types, io.rows = _dtype(x), plan.number_of_types, x.shape[0]
    io.inputs, io.outputs, io.rank = x.shape[1], dy.shape[1], rank
    io.d_x, io.ldx, io.d_dy, io.ldy = x.data_ptr(), ldx, dy.data_ptr(), ldy
    io.d_plan = plan._words.data_ptr()
    for name, tensor in (("d_low", low), ("d_back", back), ("d_down", d_down), ("d_up", d_up),
                         ("d_dw", dw), ("d_db", db)):
        if tensor is not None:
            setattr(io, name, tensor.data_ptr())
    need = C.c_uint64()
    L = _lib.lib()
    _lib.check(L.gn2v_adapted_gradient_temp(C.byref(io), C.byref(need)))
    temp = torch.empty(need.value, dtype=torch.uint8, device=dy.device)
    io.d_temp, io.temp_bytes = temp.data_ptr(), need.value
    _lib.check(L.gn2v_adapted_gradient(C.byref(io), _stream(dy)))


# A few rows are worth one launch in which every row reads its type's weights by itself.
FEW_ROWS = 64


def _few_rows(x, plan, types, weight, number_of_types, bias=None, down=None, up=None, scale=1.0):
    """The one-launch form, or None where it does not apply."""
    rows, inputs = x.shape
    outputs = weight.shape[-1]
    if not 0 < rows <= FEW_ROWS or inputs > _lib.FEW_ROWS_DEPTH:
        return None
    if any(w is not None and w.shape[-1] > 1 and w.stride(-1) != 1 for w in (weight, down, up)):
        return None  # transposed weights would be copied whole
    x, ldx = _row_stride(x)
    weight, view = _weights(weight, rows_contiguous=True)
    y = _torch().empty((rows, outputs), dtype=x.dtype, device=x.device)
    io = _product_io(x, ldx, view, y, inputs, outputs, number_of_types)
    if plan is not None:
        io.d_plan = plan._words.data_ptr()
    else:
        types = types.contiguous()
        io.d_types, io.type_bytes = types.data_ptr(), types.element_size()
    bias = _set_bias(io, bias)
    if down is not None:
        (down, io.down), (up, io.up) = _weights(down, True), _weights(up, True)
        io.rank, io.scale = down.shape[2], scale
    _lib.check(_lib.lib().gn2v_few_rows_product(C.byref(io), _stream(x)))
    return y


def _functions():
    """The autograd functions, made on first use (torch is imported lazily in this package)."""
    global _FUNCTIONS
    if _FUNCTIONS is not None:
        return _FUNCTIONS
    torch = _torch()
    from torch.autograd.function import once_differentiable

    class Typed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, plan):
            ctx.save_for_backward(x, weight)
            ctx.plan, ctx.bias_shape = plan, None if bias is None else bias.shape
            x, ldx = _row_stride(x)
            weight, view = _weights(weight)
            return _typed_product(x, ldx, view, plan, weight.shape[2], bias)

        @staticmethod
        @once_differentiable
        def backward(ctx, dy):
            x, weight = ctx.saved_tensors
            plan = ctx.plan
            dx = dw = db = None
            dy, ldy = _row_stride(dy)
            if ctx.needs_input_grad[0]:
                weight_, view = _weights(weight)
                dx = _typed_product(dy, ldy, _transposed(view), plan, weight.shape[1])
            if ctx.needs_input_grad[2]:
                db = torch.empty(ctx.bias_shape, dtype=x.dtype, device=x.device)
            if ctx.needs_input_grad[1]:
                dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
            if dw is not None or db is not None:
                _gradient(x, dy, plan, dw, db)
            return dx, dw, db, None

    class Adapted(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, down, up, bias, plan, scale):
            ctx.plan, ctx.scale = plan, scale
            rows, ldx = _row_stride(x)
            weight_, view = _weights(weight, rows_contiguous=True)
            down_, down_view = _weights(down)
            up_, up_view = _weights(up, rows_contiguous=True)
            rank, low = down.shape[2], None
            if ctx.needs_input_grad[3]:  # up's gradient is made of the low-rank rows
                low = torch.empty((x.shape[0], rank), dtype=torch.float32, device=x.device)
            ctx.save_for_backward(x, weight, down, up, low)
            return _adapted_product(rows, ldx, view, down_view, up_view, rank, scale, plan,
                                    weight.shape[1], bias, low)

        @staticmethod
        @once_differentiable
        def backward(ctx, dy):
            x, weight, down, up, low = ctx.saved_tensors
            plan, wanted = ctx.plan, ctx.needs_input_grad
            dx = dw = d_down = d_up = db = None
            dy, ldy = _row_stride(dy)
            rank, back = down.shape[2], None
            up_, up_view = _weights(up)
            if wanted[0]:
                # scale * dy up^T, which down's gradient is made of, comes on the way
                if wanted[2]:
                    back = torch.empty((x.shape[0], rank), dtype=torch.float32, device=x.device)
                weight_, view = _weights(weight, rows_contiguous=True)
                down_, down_view = _weights(down, rows_contiguous=True)
                dx = _adapted_product(dy, ldy, _transposed(view), _transposed(up_view),
                                      _transposed(down_view), rank, ctx.scale, plan,
                                      weight.shape[0], low=back)
            if wanted[2]:
                if back is None:
                    back = _low_rows(dy, ldy, _transposed(up_view), plan, rank, ctx.scale)
                d_down = torch.empty(down.shape, dtype=x.dtype, device=x.device)
            if wanted[3]:
                d_up = torch.empty(up.shape, dtype=x.dtype, device=x.device)
            if wanted[4]:
                db = torch.empty(weight.shape[1], dtype=x.dtype, device=x.device)
            if wanted[1]:
                dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
            if any(wanted[1:5]):
                _adapted_gradient(x, dy, low, back, rank, plan, d_down, d_up, dw, db)
            return dx, dw, d_down, d_up, db, None, None

    _FUNCTIONS = Typed, Adapted
    return _FUNCTIONS


_FUNCTIONS = None


def _check_types(types, x, number_of_types: int):
    if isinstance(types, TypePlan):
        if types.number_of_types != number_of_types:
            raise ValueError(f"The provided plan is for {types.number_of_types} types, but there are "
                             f"weights for {number_of_types}.")
        rows, device = types.number_of_rows, types.device
    else:
        torch = _torch()
        if not isinstance(types, torch.Tensor) or types.dim() != 1 or types.dtype not in (
                torch.int32, torch.int64):
            raise ValueError("The provided types should be a TypePlan or a one-dimensional int32 or "
                             "int64 tensor.")
        if number_of_types > _lib.MAX_TYPES:
            raise ValueError(f"There can be at most {_lib.MAX_TYPES} types, but we got weights for "
                             f"{number_of_types}.")
        rows, device = types.numel(), types.device
    if rows != x.shape[0]:
        raise ValueError(f"There are types for {rows} rows, but {x.shape[0]} rows.")
    if device != x.device:
        raise ValueError(f"The types are on {device}, but the rows on {x.device}.")


def _wants_gradient(*tensors) -> bool:
    return _torch().is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def typed_projection(x, weight, types: Union["TypePlan", "object"], bias=None):
    """``x[r] @ weight[types[r]] + bias[types[r]]`` for every row, zeros for rows of unknown type.

    Parameters
    ------------------
    x
        float32 or bfloat16 tensor [rows, inputs] on the device; rows may be strided (the first columns
        of a padded table).
    weight
        [types, inputs, outputs] of the same type; a transposed view is read as it is.
    types
        The type id of every row (int32 / int64; an id outside [0, types) is an unknown type), or the
        ``TypePlan`` of such ids: make the plan once where the types stay, as those of a graph do.
    bias
        [types, outputs] or None.

    Returns
    ------------------
    [rows, outputs] of the rows' type; products are summed in float32 and rounded once.  Differentiable
    in ``x``, ``weight`` and ``bias``.
    """
    _check_rows("rows", x, 2)
    _check_rows("weight", weight, 3)
    if 0 in weight.shape:
        raise ValueError(f"The provided weight should not be empty, but we got {tuple(weight.shape)}.")
    n_types, inputs, outputs = weight.shape
    _check_like("weight", weight, (n_types, x.shape[1], outputs), x)
    if bias is not None:
        _check_like("bias", bias, (n_types, outputs), x)
    _check_types(types, x, n_types)
    _check_device(x)
    plan = types if isinstance(types, TypePlan) else None
    if not _wants_gradient(x, weight, bias):
        y = _few_rows(x, plan, types, weight, n_types, bias)
        if y is not None:
            return y
    return _functions()[0].apply(x, weight, bias, plan or TypePlan(types, n_types))


def adapted_projection(x, weight, down, up, types: Union["TypePlan", "object"], bias=None,
                       scale: Optional[float] = 1.0):
    """``x[r] @ weight + bias + scale * (x[r] @ down[types[r]]) @ up[types[r]]`` for every row: one
    projection that all rows share and a low-rank correction of their type.  Rows of unknown type get
    the shared part alone.

    Parameters
    ------------------
    x
        float32 or bfloat16 tensor [rows, inputs] on the device; rows may be strided.
    weight
        [inputs, outputs], shared by all types.
    down, up
        [types, inputs, rank] and [types, rank, outputs]; rank at most 64.
    types
        As for ``typed_projection``.
    bias
        [outputs] or None.
    scale: float
        Of the correction.

    Returns
    ------------------
    [rows, outputs] of the rows' type.  Differentiable in every tensor but the types; leave the
    gradient of ``weight`` and ``bias`` off to train the corrections alone.
    """
    _check_rows("rows", x, 2)
    _check_rows("weight", weight, 2)
    _check_rows("down", down, 3)
    _check_rows("up", up, 3)
    for name, tensor in (("weight", weight), ("down", down), ("up", up)):
        if 0 in tensor.shape:
            raise ValueError(f"The provided {name} should not be empty, but we got "
                             f"{tuple(tensor.shape)}.")
    inputs, outputs = weight.shape
    n_types, _, rank = down.shape
    if rank > _lib.MAX_RANK:
        raise ValueError(f"The rank should be at most {_lib.MAX_RANK}, but we got {rank} instead.")
    _check_like("weight", weight, (x.shape[1], outputs), x)
    _check_like("down", down, (n_types, inputs, rank), x)
    _check_like("up", up, (n_types, rank, outputs), x)
    if bias is not None:
        _check_like("bias", bias, (outputs,), x)
    _check_types(types, x, n_types)
    _check_device(x)
    plan = types if isinstance(types, TypePlan) else None
    scale = float(scale)
    if not _wants_gradient(x, weight, down, up, bias):
        y = _few_rows(x, plan, types, weight, n_types, bias, down, up, scale)
        if y is not None:
            return y
    return _functions()[1].apply(x, weight, down, up, bias, plan or TypePlan(types, n_types), scale)

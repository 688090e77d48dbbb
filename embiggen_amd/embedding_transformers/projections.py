"""Projections of embedding rows by their type.

The rows of a typed graph's embedding table (or of its edges' embeddings) go through the weights of
their node or edge type, or through one shared projection plus a low-rank correction of their type --
an adapter.  The reference's classifiers treat types as one-hot columns beside the embedding
(embiggen/embedding_transformers/graph_transformer.py:196-243); here every type has weights of its own.
Both run in hand-written kernels that read the rows where they are: a *plan* (``TypePlan``) holds the
order of the rows by type, and no sorted copy of them is made.  Both can be differentiated backwards, once
(forward-mode derivatives are refused); gradients are summed in a fixed order, so a run gives the same bits
every time.  Calls are made on the current stream and can be captured into a graph, the plan's among them; a
backward pass that is captured takes leaves that no eager graph holds at the time.
"""
import collections
import ctypes as C
import functools
import struct
from typing import Union

from .. import _lib


_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:  # imported on first use, as everywhere in this package
        import torch

        _TORCH = torch
    return _TORCH


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
    if (isinstance(tensor, _torch().Tensor) and tensor.shape == shape and tensor.dtype == x.dtype
            and tensor.device == x.device):
        return
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
    # the raw handle of torch.cuda.current_stream(x.device), a fifth of its time
    return _torch()._C._cuda_getCurrentRawStream(x.get_device())


@functools.lru_cache(maxsize=1024)
def _plan_words(rows: int, n_types: int):
    """(words of a plan, words of scratch): a function of the sizes alone."""
    words, temp_words = C.c_uint64(), C.c_uint64()
    _lib.check(_lib.lib().gn2v_type_plan_words(rows, n_types, C.byref(words), C.byref(temp_words)))
    return words.value, temp_words.value


class TypePlan:
    """The order of rows by type: made once, used by every projection of the same rows.

    Parameters
    ------------------
    types
        int32 / int64 tensor on the device: the type id of every row.  -1 -- or any other id outside
        ``[0, number_of_types)`` -- is an unknown type.
    number_of_types: int
        How many types there are, 32 768 at most.

    A plan may be used on other streams than the one that it was made on, once they wait for it.
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
        words, temp_words = _plan_words(self.number_of_rows, self.number_of_types)
        types = types.contiguous()
        self._made_on = _stream(types)
        self._words = torch.empty(words, dtype=torch.int32, device=types.device)
        temp = None
        if temp_words:
            temp = torch.empty(temp_words, dtype=torch.int32, device=types.device)
        _lib.check(_lib.lib().gn2v_type_plan(
            types.data_ptr(), types.element_size(), self.number_of_rows, self.number_of_types,
            self._words.data_ptr(), None if temp is None else temp.data_ptr(), self._made_on))

    def _used_by(self, x):
        """Called before a projection of ``x``: the words are row ids that kernels follow, so their memory is not given
        to others while another stream than the plan's still reads them."""
        if _stream(x) != self._made_on:
            self._words.record_stream(_torch().cuda.current_stream(x.device))

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._made_on = None  # a copy's words are of another stream, or of another process

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
    def device(self):
        return self._words.device

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
    (rows, width), (apart, inner) = x.shape, x.stride()
    if width > 1 and inner != 1 or apart < width:
        if rows != 1 or width > 1 and inner != 1:
            x = x.contiguous()
        return x, width
    return x, apart


# gn2v_weights (include/gn2v_internal.h) by its fields
_View = collections.namedtuple("_View", "d_data type_stride inner outer")


def _weights(w, rows_contiguous: bool = False):
    """(tensor, _View) of [inputs, outputs] or [types, inputs, outputs] weights: as they are
    where one of the two last strides is 1 (``rows_contiguous``: the last one), else a copy."""
    strides = w.stride()
    inner, outer = strides[-2:]
    if outer == 1:
        return w, _View(w.data_ptr(), strides[0] if len(strides) == 3 else 0, inner, 1)
    if w.shape[-1] == 1:
        outer = 1
    elif w.shape[-2] == 1 and outer != 1 and not rows_contiguous:
        inner = 1
    if outer != 1 and (rows_contiguous or inner != 1):
        w = w.contiguous()
        inner, outer = w.stride(-2), 1
    return w, _View(w.data_ptr(), w.stride(0) if w.dim() == 3 else 0, inner, outer)


def _transposed(view):
    return _View(view.d_data, view.type_stride, view.outer, view.inner)


def _dtype(x) -> int:
    return 0 if x.dtype == _torch().float32 else 1


_NO_WEIGHTS = _View(0, 0, 0, 0)
# gn2v_product_io as it lies in memory: packed at once, in a quarter of the time its fields take one by one
_PRODUCT = struct.Struct("IIQIIPqPqqqPqPqPPIIfIPqqqPqqqP")
_GRADIENT = struct.Struct("IIQIIPPqqIIIIPPPPQ")
_ADAPTED_GRADIENT = struct.Struct("IIQIIIIPPqqPPPPPPPPQ")


def _product_io(x, ldx, weight, y, outputs, n_types, bias=None, plan=None, types=None, rank=0,
                scale=1.0, low_rank_rows=0, down=_NO_WEIGHTS, up=_NO_WEIGHTS, low=None):
    """(gn2v_product_io, what has to outlive the call)."""
    bias_stride = 0
    if bias is not None:
        strides = bias.stride()
        if strides[-1] != 1 and bias.shape[-1] > 1:
            bias = bias.contiguous()
            strides = bias.stride()
        bias_stride = strides[0] if len(strides) == 2 else 0
    if types is not None:
        types = types.contiguous()
    return _lib.ProductIO.from_buffer_copy(_PRODUCT.pack(
        _dtype(x), n_types, *x.shape, outputs, x.data_ptr(), ldx, *weight,
        0 if bias is None else bias.data_ptr(), bias_stride, y.data_ptr(), y.shape[1],
        0 if plan is None else plan._words.data_ptr(),
        0 if types is None else types.data_ptr(), 0 if types is None else types.element_size(),
        rank, scale, low_rank_rows, *down, *up, 0 if low is None else low.data_ptr())), (bias, types)


def _typed_product(x, ldx, weight, plan, outputs, bias=None):
    y = _torch().empty((x.shape[0], outputs), dtype=x.dtype, device=x.device)
    io, keep = _product_io(x, ldx, weight, y, outputs, plan.number_of_types, bias, plan)
    _lib.check(_lib.lib().gn2v_typed_product(io, _stream(x)))
    return y


def _adapted_product(x, ldx, weight, down, up, rank, scale, plan, outputs, bias=None, low=None):
    """``low``: float32 [rows, rank], filled with the low-rank rows at their positions in the plan's
    order; None where nobody needs them."""
    torch = _torch()
    if low is None and (rank > _lib.FUSED_RANK
                        or x.shape[1] * x.element_size() > _lib.FUSED_ROW_BYTES):
        low = torch.empty((x.shape[0], rank), dtype=torch.float32, device=x.device)
    y = torch.empty((x.shape[0], outputs), dtype=x.dtype, device=x.device)
    io, keep = _product_io(x, ldx, weight, y, outputs, plan.number_of_types, bias, plan, None, rank,
                           scale, 0, down, up, low)
    _lib.check(_lib.lib().gn2v_adapted_product(io, _stream(x)))
    return y


def _low_rows(x, ldx, weight, plan, rank, scale):
    """scale * x[r] W[type of r] as float32 rows at their positions in the plan's order."""
    low = _torch().empty((x.shape[0], rank), dtype=_torch().float32, device=x.device)
    io, keep = _product_io(x, ldx, weight, low, rank, plan.number_of_types, None, plan, None, 0, scale,
                           1)
    _lib.check(_lib.lib().gn2v_typed_product(io, _stream(x)))
    return low


@functools.lru_cache(maxsize=1024)
def _gradient_bytes(adapted: bool, *sizes) -> int:
    """Scratch of a gradient, a function of its sizes and of which parts are wanted: ``sizes`` as the
    fields of the structure, pointers as truth values."""
    need = C.c_uint64()
    L = _lib.lib()
    if adapted:
        dtype, n_types, rows, inputs, outputs, rank, down, up, dw, db = sizes
        io = _lib.AdaptedGradientIO(dtype, n_types, rows, inputs, outputs, rank)
        io.d_down, io.d_up, io.d_dw, io.d_db = down, up, dw, db
        _lib.check(L.gn2v_adapted_gradient_temp(io, C.byref(need)))
    else:
        io = _lib.GradientIO(*sizes)
        _lib.check(L.gn2v_typed_gradient_temp(io, C.byref(need)))
    return need.value


def _ptr(tensor):
    return 0 if tensor is None else tensor.data_ptr()


def _gradient(x, dy, plan, dw, db):
    """Fills dw [types, inputs, outputs] and db [types, outputs], those that are not None."""
    torch = _torch()
    x, ldx = _row_stride(x)
    dy, ldy = _row_stride(dy)
    sizes = (_dtype(x), plan.number_of_types, x.shape[0], 0 if dw is None else x.shape[1],
             dy.shape[1])
    need = _gradient_bytes(False, *sizes)
    temp = torch.empty(need, dtype=torch.uint8, device=dy.device)
    io = _lib.GradientIO.from_buffer_copy(_GRADIENT.pack(
        *sizes, x.data_ptr(), dy.data_ptr(), ldx, ldy, 0, 0, 0, 0, plan._words.data_ptr(), _ptr(dw),
        _ptr(db), temp.data_ptr(), need))
    _lib.check(_lib.lib().gn2v_typed_gradient(io, _stream(dy)))


def _adapted_gradient(x, dy, low, back, rank, plan, d_down, d_up, dw, db):
    """Fills the gradients that are not None."""
    torch = _torch()
    x, ldx = _row_stride(x)
    dy, ldy = _row_stride(dy)
    sizes = (_dtype(x), plan.number_of_types, x.shape[0], x.shape[1], dy.shape[1], rank)
    need = _gradient_bytes(True, *sizes, d_down is not None, d_up is not None, dw is not None,
                           db is not None)
    temp = torch.empty(need, dtype=torch.uint8, device=dy.device)
    io = _lib.AdaptedGradientIO.from_buffer_copy(_ADAPTED_GRADIENT.pack(
        *sizes, 0, x.data_ptr(), dy.data_ptr(), ldx, ldy, _ptr(low), _ptr(back),
        plan._words.data_ptr(), _ptr(d_down), _ptr(d_up), _ptr(dw), _ptr(db), temp.data_ptr(), need))
    _lib.check(_lib.lib().gn2v_adapted_gradient(io, _stream(dy)))


# A few rows are worth one launch in which every row reads its type's weights by itself: while there are
# at most so many, and what they read together is at most so many bytes.  One launch / plan and product
# (the plan given), microseconds: 128 -> 128 float32, 1 024 rows 6.4 / 20.5 (10.2), 4 096 rows 16.6 / 22.4
# (11.7); 512 -> 256, 512 rows (268 MB) float32 15.7 / 44.4 (34.9), 1 024 rows bfloat16 (268 MB) 18.3 /
# 23.6 (13.6), 2 048 rows (537 MB) 32.4 / 23.2 (13.7); 1 024 -> 1 024, 64 rows (268 MB) float32 18.1 / 68.4.
# One rule, plan or none: with a plan at hand the largest bfloat16 calls inside it lose up to 5 us.
FEW_ROWS = 1024
FEW_BYTES = 1 << 28


def _few_rows(x, plan, types, weight, number_of_types, bias=None, down=None, up=None, scale=1.0):
    """The one-launch form, or None where it does not apply."""
    rows, inputs = x.shape
    outputs = weight.shape[-1]
    if (not 0 < rows <= FEW_ROWS or inputs > _lib.FEW_ROWS_DEPTH
            or rows * inputs * outputs * x.element_size() > FEW_BYTES):
        return None
    for w in (weight,) if down is None else (weight, down, up):
        if w.stride(-1) != 1 and w.shape[-1] > 1:
            return None  # transposed weights would be copied whole
    x, ldx = _row_stride(x)
    weight, view = _weights(weight, True)
    y = _torch().empty((rows, outputs), dtype=x.dtype, device=x.device)
    if plan is not None:
        types = None
    if down is None:
        io, keep = _product_io(x, ldx, view, y, outputs, number_of_types, bias, plan, types)
    else:
        (down, down_view), (up, up_view) = _weights(down, True), _weights(up, True)
        io, keep = _product_io(x, ldx, view, y, outputs, number_of_types, bias, plan, types,
                               down.shape[2], scale, 0, down_view, up_view)
    _lib.check(_lib.lib().gn2v_few_rows_product(io, _stream(x)))
    return y


def _functions():
    """The autograd functions, made on first use (torch is imported lazily in this package)."""
    global _FUNCTIONS
    if _FUNCTIONS is not None:
        return _FUNCTIONS
    torch = _torch()
    from torch.autograd.function import once_differentiable

    def once(backward):
        # the check for a second differentiation costs more than a launch: made where gradients of
        # gradients are recorded at all
        checked = once_differentiable(backward)
        return staticmethod(lambda ctx, dy: (checked if torch.is_grad_enabled() else backward)(ctx, dy))

    class Typed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, plan):
            ctx.save_for_backward(x, weight)
            ctx.plan, ctx.bias_shape = plan, None if bias is None else bias.shape
            x, ldx = _row_stride(x)
            weight, view = _weights(weight)
            return _typed_product(x, ldx, view, plan, weight.shape[2], bias)

        @once
        def backward(ctx, dy):
            _refuse_tangents(dy)
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

        @once
        def backward(ctx, dy):
            _refuse_tangents(dy)
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


def _check_scale(scale) -> float:
    if getattr(scale, "requires_grad", False):
        raise ValueError("The provided scale takes no gradient: multiply `up` by it instead.")
    try:
        return float(scale)
    except (TypeError, ValueError, RuntimeError):
        raise ValueError(f"The provided scale should be a number, but we got {scale!r} instead.") from None


def _refuse_tangents(*tensors):
    """The kernels see a tensor's values alone: a forward-mode tangent would be lost without a word."""
    forward_ad = _torch().autograd.forward_ad
    if forward_ad._current_level < 0:  # nobody differentiates forwards; unpacking costs 0.3 us a tensor
        return
    for tensor in tensors:
        if tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None:
            raise NotImplementedError("The projections have no forward-mode derivatives, but one of the "
                                      "provided tensors has a tangent.")


def _wants_gradient(*tensors) -> bool:
    for tensor in tensors:
        if tensor is not None and tensor.requires_grad:
            return _torch().is_grad_enabled()
    return False


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
    in ``x``, ``weight`` and ``bias`` (backwards, once; a tensor with a forward-mode tangent is refused).
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
    _refuse_tangents(x, weight, bias)
    plan = types if isinstance(types, TypePlan) else None
    if plan is not None:
        plan._used_by(x)
    if not _wants_gradient(x, weight, bias):
        y = _few_rows(x, plan, types, weight, n_types, bias)
        if y is not None:
            return y
    return _functions()[0].apply(x, weight, bias, plan or TypePlan(types, n_types))


def adapted_projection(x, weight, down, up, types: Union["TypePlan", "object"], bias=None,
                       scale: float = 1.0):
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
        Of the correction; a number, which takes no gradient.

    Returns
    ------------------
    [rows, outputs] of the rows' type.  Differentiable in every tensor but the types, as
    ``typed_projection`` is; leave the gradient of ``weight`` and ``bias`` off to train the corrections alone.
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
    _refuse_tangents(x, weight, down, up, bias)
    plan = types if isinstance(types, TypePlan) else None
    if plan is not None:
        plan._used_by(x)
    scale = _check_scale(scale)
    if not _wants_gradient(x, weight, down, up, bias):
        y = _few_rows(x, plan, types, weight, n_types, bias, down, up, scale)
        if y is not None:
            return y
    return _functions()[1].apply(x, weight, down, up, bias, plan or TypePlan(types, n_types), scale)

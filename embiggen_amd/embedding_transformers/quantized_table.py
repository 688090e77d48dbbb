"""Embedding tables held in 8 bits.

A trained table of float32 rows is the largest thing a user of the embeddings keeps around: the edge
operators (embiggen/embedding_transformers/edge_transformer.py:12-343) and every model behind them read
its rows again and again.  ``QuantizedTable`` holds them as int8 or e4m3 codes with one float32 scale
per row and group of columns -- 0.26 to 0.31 of the bytes at 128 columns --, quantises rows as they are
written and gives them back as float32 or bfloat16; ``edge_embedding`` and ``EdgeTransformer`` read the
8-bit rows directly.
"""
from typing import Optional

from .. import _lib
from .projections import _stream, _torch

GROUP_SIZES = (16, 32, 64, 128)
_CODES = {}


def _codes():
    if not _CODES:
        torch = _torch()
        _CODES.update({torch.int8: 0, torch.float8_e4m3fn: 1})
    return _CODES


def _ids(rows, device, what: str):
    """A contiguous id tensor as it is (int32 / int64)."""
    torch = _torch()
    if not isinstance(rows, torch.Tensor) or rows.dim() != 1 or rows.dtype not in (
            torch.int32, torch.int64):
        raise ValueError(f"The provided {what} should be a one-dimensional int32 or int64 tensor.")
    if rows.device != device:
        raise ValueError(f"The provided {what} are on {rows.device}, but the table is on {device}.")
    return rows.contiguous()


def _value_type(dtype) -> int:
    torch = _torch()
    if dtype == torch.float32:
        return 0
    if dtype == torch.bfloat16:
        return 1
    raise ValueError(f"Rows are float32 or bfloat16, but we got {dtype} instead.")


def _taken_up(cls, codes, dtype, *rest):
    return cls(codes.view(dtype), *rest)


class QuantizedTable:
    """A table of ``embedding_size`` columns in 8 bits.

    The scale of a group is its largest magnitude times the float32 1 / 127 (int8) or 1 / 448 (e4m3), in
    float32 (within 2**-23 of the quotient), and at least 2**-90; a code is the value divided by it, rounded to
    the nearest code, ties to even; a value read back is code * scale.  A group that holds an infinity or a NaN
    reads back as NaN.

    Parameters
    ------------------
    codes
        int8 or float8_e4m3fn tensor [rows, stride] on the device, contiguous, ``stride`` a multiple of
        16 and at least ``embedding_size``.
    scales
        Contiguous float32 tensor [rows, ceil(embedding_size / group_size)].
    embedding_size: Optional[int] = None
        The number of columns; by default the stride of the codes.
    group_size: int = 64
        Consecutive columns that share a scale: 16, 32, 64 or 128.

    The tensors are used as they are, not copied: a stored table can be taken up by its parts, and
    ``codes`` and ``scales`` are what to store.  ``empty`` and ``from_table`` make new ones.
    """

    def __init__(self, codes, scales, embedding_size: Optional[int] = None, group_size: int = 64):
        torch = _torch()
        if not isinstance(codes, torch.Tensor) or codes.dtype not in _codes() or codes.dim() != 2:
            raise ValueError("The codes should be a two-dimensional int8 or float8_e4m3fn tensor.")
        if group_size not in GROUP_SIZES:
            raise ValueError(f"The group size should be one of {GROUP_SIZES}, but we got "
                             f"{group_size} instead.")
        size = codes.shape[1] if embedding_size is None else int(embedding_size)
        if not 0 < size <= codes.shape[1] or codes.shape[1] % 16 or not codes.is_contiguous():
            raise ValueError("The codes should be contiguous rows of a multiple of 16 columns, at "
                             f"least the embedding size, but we got shape {tuple(codes.shape)} for "
                             f"an embedding size of {size}.")
        groups = -(-size // group_size)
        if (not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32
                or tuple(scales.shape) != (codes.shape[0], groups) or not scales.is_contiguous()):
            raise ValueError(f"The scales should be a contiguous float32 tensor of shape "
                             f"{(codes.shape[0], groups)}.")
        if codes.device != scales.device:
            raise ValueError(f"The codes are on {codes.device}, but the scales on {scales.device}.")
        if codes.device.type != "cuda":
            raise ValueError("The table should be on a ROCm device (there is no CPU execution path), "
                             f"but it is on {codes.device}.")
        if codes.data_ptr() % 16:
            raise ValueError("The codes should be aligned to 16 bytes.")
        self._codes, self._scales = codes, scales
        self.embedding_size, self.group_size = size, group_size
        self._io = _lib.Table8(codes.data_ptr(), scales.data_ptr(), codes.shape[0], size,
                               codes.shape[1], group_size, _codes()[codes.dtype])
        self._taken = self._where()

    def _where(self):
        codes, scales = self._codes, self._scales
        return codes.data_ptr(), scales.data_ptr(), codes.shape, scales.shape

    def _table(self):
        """The table for a call.  The tensors are the caller's too: one that has other memory now (its ``data`` set,
        resized) is taken up anew, behind the same checks."""
        if self._where() != self._taken:
            self.__init__(self._codes, self._scales, self.embedding_size, self.group_size)
        return self._io

    # Copies and pickles hold the tensors; the addresses are taken anew, behind the same checks.  Codes go as bytes:
    # a tensor of float8 elements cannot be pickled by itself.
    def __copy__(self):
        return type(self)(self._codes, self._scales, self.embedding_size, self.group_size)

    def __reduce__(self):
        return _taken_up, (type(self), self._codes.view(_torch().uint8), self._codes.dtype, self._scales,
                           self.embedding_size, self.group_size)

    @classmethod
    def empty(cls, number_of_rows: int, embedding_size: int, dtype=None, group_size: int = 64,
              device: int = 0) -> "QuantizedTable":
        """A table of zero rows.  ``dtype``: torch.int8 (the default) or torch.float8_e4m3fn."""
        torch = _torch()
        dtype = torch.int8 if dtype is None else dtype
        if dtype not in _codes():
            raise ValueError(f"The codes are int8 or float8_e4m3fn, but we got {dtype} instead.")
        if number_of_rows < 0 or embedding_size < 1:
            raise ValueError("A table needs at least one column and no negative number of rows.")
        if group_size not in GROUP_SIZES:
            raise ValueError(f"The group size should be one of {GROUP_SIZES}, but we got "
                             f"{group_size} instead.")
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        stride = -(-embedding_size // 16) * 16
        codes = torch.zeros((number_of_rows, stride), dtype=torch.uint8, device=dev).view(dtype)
        scales = torch.zeros((number_of_rows, -(-embedding_size // group_size)),
                             dtype=torch.float32, device=dev)
        return cls(codes, scales, embedding_size, group_size)

    @classmethod
    def from_table(cls, table, dtype=None, group_size: int = 64,
                   embedding_size: Optional[int] = None) -> "QuantizedTable":
        """The float32 or bfloat16 rows of ``table`` in 8 bits (``embedding_size``: its first columns
        alone)."""
        torch = _torch()
        if not isinstance(table, torch.Tensor) or table.dim() != 2:
            raise ValueError("The table should be a two-dimensional tensor.")
        _value_type(table.dtype)
        if table.device.type != "cuda":
            raise ValueError("The table should be on a ROCm device (there is no CPU execution path), "
                             f"but it is on {table.device}.")
        if embedding_size is not None:
            if not 0 < embedding_size <= table.shape[1]:
                raise ValueError(f"The embedding size should be between 1 and {table.shape[1]}, but "
                                 f"we got {embedding_size} instead.")
            table = table[:, :embedding_size]
        new = cls.empty(table.shape[0], table.shape[1], dtype, group_size, table.device)
        new.write(table)
        return new

    @property
    def codes(self):
        """int8 or float8_e4m3fn [rows, stride]: the tensor itself, not a copy."""
        return self._codes

    @property
    def scales(self):
        """float32 [rows, groups]: the tensor itself, not a copy."""
        return self._scales

    @property
    def shape(self):
        return (self.codes.shape[0], self.embedding_size)

    @property
    def device(self):
        return self.codes.device

    def __len__(self) -> int:
        return self.codes.shape[0]

    def write(self, values, rows=None):
        """Quantises ``values`` [entries, embedding_size] (float32 or bfloat16; rows may be strided)
        into the table.  ``rows``: the row of every entry, int32 / int64; by default the first rows in
        order.  An entry whose row lies outside the table (-1 in a padded batch) is left out; of
        several entries of one row the last is kept."""
        torch = _torch()
        if not isinstance(values, torch.Tensor) or values.dim() != 2:
            raise ValueError("The values should be a two-dimensional tensor.")
        kind = _value_type(values.dtype)
        n, width = values.shape
        if width != self.embedding_size or values.device != self._codes.device:
            raise ValueError(f"The values should be rows of {self.embedding_size} columns on "
                             f"{self.device}, but we got shape {tuple(values.shape)} on "
                             f"{values.device}.")
        if rows is None:
            if n > len(self):
                raise ValueError(f"{n} rows do not fit a table of {len(self)}.")
        else:
            rows = _ids(rows, values.device, "rows")
            if rows.shape[0] != n:
                raise ValueError(f"There are {n} values, but rows for {rows.numel()}.")
        io = self._table()
        apart, inner = values.stride()
        if inner != 1 or apart < self.embedding_size:
            values = values.detach().contiguous()
            apart = values.stride(0)
        owner = None
        if rows is not None and n > _lib.TABLE_FEW_ENTRIES:
            owner = torch.empty(len(self), dtype=torch.int32, device=self.device)
        _lib.check(_lib.lib().gn2v_table_write(
            io, values.data_ptr(), kind, max(apart, self.embedding_size),
            None if rows is None else rows.data_ptr(), 0 if rows is None else rows.element_size(), n,
            None if owner is None else owner.data_ptr(), _stream(self._codes)))

    def read(self, rows=None, dtype=None):
        """The rows ``rows`` (int32 / int64; by default all) as a float32 (or bfloat16: ``dtype``)
        tensor [entries, embedding_size]; an id outside the table reads as zeros."""
        torch = _torch()
        dtype = torch.float32 if dtype is None else dtype
        kind = _value_type(dtype)
        if rows is not None:
            rows = _ids(rows, self._codes.device, "rows")
        n = len(self) if rows is None else rows.shape[0]
        out = torch.empty((n, self.embedding_size), dtype=dtype, device=self._codes.device)
        _lib.check(_lib.lib().gn2v_table_read(
            self._table(), None if rows is None else rows.data_ptr(),
            0 if rows is None else rows.element_size(), n, out.data_ptr(), kind,
            self.embedding_size, _stream(self._codes)))
        return out


def quantized_edge_embedding(table, sources, destinations, method: int, width: int,
                             destination_table=None):
    """``edge_embedding`` on tables in 8 bits (method id and output width already known)."""
    torch = _torch()
    other = table if destination_table is None else destination_table
    if not isinstance(other, QuantizedTable):
        raise ValueError("Source and destination tables should both be in 8 bits, or neither.")
    if (table.embedding_size != other.embedding_size or table.codes.dtype != other.codes.dtype
            or table.device != other.device):
        raise ValueError("Source and destination tables should have the same embedding size, type of "
                         "codes and device.")
    src = _ids(sources, table.device, "sources")
    dst = _ids(destinations, table.device, "destinations")
    if src.shape != dst.shape:
        raise ValueError("sources and destinations must have the same shape.")
    if src.dtype != dst.dtype:
        src, dst = src.long(), dst.long()
    out = torch.empty((src.numel(), width), dtype=torch.float32, device=table.device)
    _lib.check(_lib.lib().gn2v_table_edge_embedding(
        table._table(), other._table(), src.data_ptr(), dst.data_ptr(), src.element_size(),
        src.numel(), method, out.data_ptr(), width, _stream(table.codes)))
    return out

"""QuantizedRows: feature rows held in 8 or 4 bits, quantised as they are written and expanded as they are read
(psl_rows_write / psl_rows_read; no reference counterpart -- the reference keeps every feature row in fp32).

A row is `heads` x `dim` values -- the geometry and the colour feature of a neural point are two heads of 32 -- and every
`group` of values shares one fp32 scale:

    scale = max|x| / Q     Q = 127 ("int8"), 7 ("int4"), 448 ("e4m3")        code = nearest(x / scale), ties to even; 0 for scale 0
    value = code * scale   in fp32, then converted to the type that is read

so a value is off by at most half a code step (scale / 2 for the integer formats, 2^-4 of the value for e4m3's normal
range).  A group with an infinite or NaN value reads back as NaN throughout.  dist.FrameParallelSync(wire=...) sends new
points and trained rows in this form, checkpoint.checkpoint_dict(feature_format=...) saves them in it.
There is no torch fallback, and no gradient passes through a store.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

FORMATS = {"int8": _lib.ROWS_INT8, "e4m3": _lib.ROWS_E4M3, "int4": _lib.ROWS_INT4}
BITS = {"int8": 8, "e4m3": 8, "int4": 4}
_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _check_layout(heads, dim, fmt, group):
    if fmt not in FORMATS:
        raise ValueError(f"row format {fmt!r}: one of {sorted(FORMATS)}")
    if not (1 <= heads <= 4096 and 1 <= dim <= 4096 and 1 <= group <= 1024) or dim % group:
        raise ValueError(f"heads {heads}, dim {dim}, group {group}: heads and dim up to 4096, group up to 1024 and a divisor of dim")
    if BITS[fmt] == 4 and group % 2:
        raise ValueError(f"two int4 codes share a byte: group {group} must be even")


def _call(entry, values, rows, first, n, fmt, group, capacity, codes, codes_row_stride, scales, scales_row_stride, owner=None):
    """One psl_rows_* call.  values [n, heads, dim], rows ids or None; codes / scales: tensors whose data_ptr is row 0."""
    dev = values.device
    if dev.type != "cuda":
        raise _lib.PslError(f"{entry}: tensors on {dev}; the kernels run on the GPU and have no host fallback")
    _, heads, dim = values.shape
    row, head, _ = values.stride()
    _lib.call_on(dev, entry, _lib.psl_rows_args(         # in the order of the struct's fields
        FORMATS[fmt], _DTYPES[values.dtype], heads, dim, group, 0 if rows is None else rows.element_size() * 8, n, capacity, first,
        None if rows is None else rows.data_ptr(), values.data_ptr(), row, head, codes.data_ptr(), codes_row_stride,
        scales.data_ptr(), scales_row_stride, None if owner is None else owner.data_ptr()))


def record_floats(heads: int, dim: int, fmt: str, group: Optional[int] = None) -> tuple:
    """(floats that the codes of a row fill, floats that its scales fill) inside a record of 32-bit words."""
    group = dim if group is None else group
    _check_layout(heads, dim, fmt, group)
    bits = heads * dim * BITS[fmt]
    if bits % 32:
        raise ValueError(f"{heads} x {dim} codes of {BITS[fmt]} bits do not fill whole 32-bit words")
    return bits // 32, heads * (dim // group)


def write_records(rec: torch.Tensor, values: torch.Tensor, fmt: str, code_col: int, scale_col: int, group: Optional[int] = None):
    """Quantise values [n, heads, dim] into columns of fp32 records [n, W]: codes from column code_col (as raw 32-bit words),
    scales from column scale_col.  What the multi-GPU exchange sends; the other columns stay as they are."""
    _record_call("psl_rows_write", rec, values.detach().contiguous(), fmt, code_col, scale_col, group)
    return rec


def read_records(rec: torch.Tensor, heads: int, dim: int, fmt: str, code_col: int, scale_col: int, group: Optional[int] = None) -> torch.Tensor:
    """The values [n, heads, dim] fp32 that write_records put into `rec`."""
    out = torch.empty(rec.shape[0], heads, dim, dtype=torch.float32, device=rec.device)
    _record_call("psl_rows_read", rec, out, fmt, code_col, scale_col, group)
    return out


def _record_call(entry, rec, values, fmt, code_col, scale_col, group):
    n, heads, dim = values.shape
    group = dim if group is None else group
    cw, sw = record_floats(heads, dim, fmt, group)
    if rec.dtype != torch.float32 or rec.dim() != 2 or rec.shape[0] != n or not rec.is_contiguous() or values.dtype not in _DTYPES:
        raise ValueError(f"records: contiguous float32 [{n}, width], got {tuple(rec.shape)} {rec.dtype}")
    spans = sorted([(code_col, code_col + cw), (scale_col, scale_col + sw)])
    if spans[0][0] < 0 or spans[0][1] > spans[1][0] or spans[1][1] > rec.shape[1] or rec.device != values.device:
        raise ValueError(f"codes at {code_col} (+{cw}) and scales at {scale_col} (+{sw}) in records of {rec.shape[1]}")
    if n:
        _call(entry, values, None, 0, n, fmt, group, n, rec[:, code_col:], 4 * rec.shape[1], rec[:, scale_col:], rec.shape[1])


class QuantizedRows:
    """A store of `capacity` rows.  codes: uint8 [capacity, heads, dim * bits / 8], scales: fp32 [capacity, heads, dim / group];
    rows that were never written read as zeros."""

    def __init__(self, capacity: int, heads: int = 2, dim: int = 32, fmt: str = "int8", group: Optional[int] = None,
                 device="cuda:0"):
        group = dim if group is None else group
        _check_layout(heads, dim, fmt, group)
        if capacity < 0:
            raise ValueError(f"capacity {capacity}")
        self.capacity, self.heads, self.dim, self.fmt, self.group = int(capacity), heads, dim, fmt, group
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.codes = torch.zeros(self.capacity, heads, dim * BITS[fmt] // 8, dtype=torch.uint8, device=self.device)
        self.scales = torch.zeros(self.capacity, heads, dim // group, dtype=torch.float32, device=self.device)

    def bytes_per_row(self) -> int:
        return self.heads * (self.dim * BITS[self.fmt] // 8 + 4 * (self.dim // self.group))

    def _rows(self, rows):
        if not torch.is_tensor(rows) or rows.dtype not in (torch.int32, torch.int64) or rows.dim() != 1:
            raise ValueError("rows: a one-dimensional int32 or int64 tensor")
        if rows.device != self.device:
            raise ValueError(f"rows on {rows.device}, the store on {self.device}")
        return rows.contiguous()

    def _range(self, first, n):
        if first < 0 or n < 0 or first + n > self.capacity:
            raise ValueError(f"rows [{first}, {first + n}) of a store of {self.capacity}")

    def _args(self):
        return (self.fmt, self.group, self.capacity, self.codes, self.codes.stride(0), self.scales, self.scales.stride(0))

    def write(self, values: torch.Tensor, rows: Optional[torch.Tensor] = None, first: int = 0, distinct: bool = False):
        """values [n, heads, dim] (fp32, bf16 or fp16) into rows `rows` [n], or into [first, first + n) when rows is None.
        Ids outside the store (padding: -1) are skipped.  When an id comes more than once the last one wins;
        `distinct=True` vouches that none does and saves that bookkeeping (two launches)."""
        if values.dtype not in _DTYPES or values.dim() != 3 or values.shape[1] != self.heads or values.shape[2] != self.dim:
            raise ValueError(f"values: [n, {self.heads}, {self.dim}] in float32, bfloat16 or float16, got {tuple(values.shape)} {values.dtype}")
        if values.device != self.device:
            raise ValueError(f"values on {values.device}, the store on {self.device}")
        n = values.shape[0]
        if values.stride(2) != 1:
            values = values.contiguous()
        owner = None
        if rows is None:
            self._range(first, n)
        else:
            rows = self._rows(rows)
            if rows.shape[0] != n:
                raise ValueError(f"{n} rows of values for {rows.shape[0]} ids")
            if not distinct and n > 1:
                owner = torch.empty(self.capacity, dtype=torch.int32, device=self.device)
        if n and self.capacity:
            _call("psl_rows_write", values, rows, first, n, *self._args(), owner)
        return self

    def read(self, rows: Optional[torch.Tensor] = None, first: int = 0, count: Optional[int] = None,
             dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values [n, heads, dim] of rows `rows`, or of [first, first + count) (to the end by default).  Ids outside the
        store give zeros; the same id may come any number of times.  `out` may be strided (rows inside wider records, or
        [heads, n, dim] memory seen as [n, heads, dim]) as long as no two of its values share memory."""
        if rows is None:
            n = self.capacity - first if count is None else int(count)
            self._range(first, n)
        else:
            rows = self._rows(rows)
            n = rows.shape[0]
        if out is None:
            if dtype not in _DTYPES:
                raise ValueError(f"dtype {dtype}: float32, bfloat16 or float16")
            out = torch.empty(n, self.heads, self.dim, dtype=dtype, device=self.device)
        elif (tuple(out.shape) != (n, self.heads, self.dim) or out.dtype not in _DTYPES or out.device != self.device
              or out.stride(2) != 1 or out.requires_grad):
            raise ValueError(f"out: [{n}, {self.heads}, {self.dim}] on {self.device}, contiguous rows, no gradient")
        if n and self.capacity:
            _call("psl_rows_read", out, rows, first, n, *self._args())
        elif n:
            out.zero_()
        return out

    def state_dict(self) -> dict:
        """Codes and scales with their layout: what a checkpoint keeps."""
        return {"capacity": self.capacity, "heads": self.heads, "dim": self.dim, "format": self.fmt, "group": self.group,
                "codes": self.codes, "scales": self.scales}

    @classmethod
    def from_state(cls, state: dict, device="cuda:0") -> "QuantizedRows":
        st = cls(state["capacity"], state["heads"], state["dim"], state["format"], state["group"], device)
        if tuple(state["codes"].shape) != tuple(st.codes.shape) or tuple(state["scales"].shape) != tuple(st.scales.shape):
            raise ValueError("codes and scales do not have the layout the state names")
        st.codes.copy_(state["codes"])
        st.scales.copy_(state["scales"])
        return st

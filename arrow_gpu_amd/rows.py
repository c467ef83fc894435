"""Rows: the array model of whole rows (include/arrow_gpu.h "rows"; no counterpart in the reference, whose arrays are columns of 1 / 2 / 4-byte
values).  RowsGPU is a strided view of a tensor in HBM, QuantisedRowsGPU a cache of rows in 8 or 4 bits, PageMap says where the rows of ragged
sequences lie in a paged cache, BeamSelection holds what select_beams found.  The operators are in kernels/rows.py."""
from __future__ import annotations

import struct
from typing import Optional

import numpy as np

from . import _capi as capi
from .array import Float32ArrayGPU, UInt32ArrayGPU
from .gpu_utils import DeviceBuffer, GpuDevice, borrow_tensor, settle, tensor_type

ITEM_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "u8": 1, "i16": 2, "u16": 2, "i32": 4, "u32": 4, "i64": 8, "f64": 8}
_FLOATING = ("f32", "f16", "bf16", "f64")
ROW_TYPE = {"f32": capi.ROW_F32, "f16": capi.ROW_F16, "bf16": capi.ROW_BF16}
CODE_TYPE = {"i8": capi.CODE_I8, "i4": capi.CODE_I4, "e4m3": capi.CODE_E4M3}
_NUMPY = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i8": np.int8, "u8": np.uint8, "i16": np.int16, "u16": np.uint16, "i32": np.int32,
          "u32": np.uint32, "i64": np.int64, "f64": np.float64}


# The ABI's structs (include/arrow_gpu.h) as bytes: a serving loop makes them anew in every call, and packing costs a fifth of filling ctypes fields
_PACK_ROWS = struct.Struct("=QQQi4x").pack          # agpu_rows
_PACK_STORE = struct.Struct("=QQQIIIi").pack        # agpu_quantised_rows
_PACK_PAGES = struct.Struct("=QQQQIII4x").pack      # agpu_page_map


def shape_error(message: str) -> capi.ArrowErrorGPU:
    return capi.ArrowErrorGPU("ShapeError", message, capi.ERR_SHAPE)


def _dense(shape):
    strides, at = [], 1
    for n in reversed(shape):
        strides.append(at)
        at *= n
    return tuple(reversed(strides)), at


class RowsGPU:
    """Rows of values in HBM: shape (n, …) of 2 to 4 axes, strides in elements, the values of the last axis next to each other."""

    PARTS = ("data",)
    __slots__ = ("data", "gpu_device", "shape", "strides", "type", "ptr", "item_size", "_rows", "_pieces")

    def __init__(self, data: DeviceBuffer, gpu_device: GpuDevice, shape, type_: str, strides=None, ptr: Optional[int] = None):
        if type_ not in ITEM_SIZE:
            raise capi.OperationNotSupported(f"rows of {type_}")
        shape = tuple(shape)
        strides = _dense(shape)[0] if strides is None else tuple(strides)
        if not 2 <= len(shape) <= 4 or len(strides) != len(shape) or min(shape) < 0:
            raise shape_error(f"rows have 2 to 4 axes: got {shape}")
        if min(strides) < 0 or (strides[-1] != 1 and shape[-1] > 1):
            raise shape_error(f"the values of a row's last axis lie next to each other: got strides {strides}")
        self.data, self.gpu_device, self.type, self.shape, self.strides = data, gpu_device, type_, shape, strides
        self.item_size = ITEM_SIZE[type_]
        self.ptr = data.ptr if ptr is None else ptr
        end = (self.ptr - data.ptr) + (1 + sum((n - 1) * s for n, s in zip(shape, strides))) * self.item_size if 0 not in shape else 0
        if data._owned and (self.ptr < data.ptr or end > data.nbytes):  # (of memory that is not the library's, the caller knows the extent)
            raise shape_error(f"rows {shape} with strides {strides} in a buffer of {data.nbytes} bytes")
        self._rows = self._pieces = None

    # -- construction
    @classmethod
    def of_tensor(cls, tensor, gpu_device: GpuDevice) -> "RowsGPU":
        """The rows over a tensor's memory, without a copy (a slice of a bigger tensor keeps its strides)."""
        t = tensor_type(tensor)
        shape, strides, item = tuple(tensor.shape), tensor.stride(), ITEM_SIZE[t]
        if not 2 <= len(shape) <= 4 or (strides[-1] != 1 and shape[-1] > 1):
            return cls(None, gpu_device, shape, t, strides, 0)  # raises
        self = cls.__new__(cls)
        self.data = data = borrow_tensor(tensor, gpu_device, tensor.numel() * item, t in _FLOATING)
        self.ptr, self.gpu_device, self.type, self.shape, self.strides, self.item_size = data.ptr, gpu_device, t, shape, strides, item
        self._rows = self._pieces = None
        return self

    # -- what the ABI's calls take
    def as_rows(self) -> bytes:
        """agpu_rows of (n, heads, dim)"""
        if self._rows is None:
            if self.type not in ROW_TYPE:
                raise capi.OperationNotSupported(f"rows of {self.type} in a quantised cache")
            self._rows = _PACK_ROWS(self.ptr, self.strides[0], self.strides[1], ROW_TYPE[self.type])
        return self._rows

    def as_pieces(self):
        """(row stride, piece stride, pieces, piece bytes, position bytes) for agpu_state: the trailing axes that lie densely are one piece, the axis
        that is left, if any, are the pieces; position bytes 0: the positions (the axis before the last) are not inside one."""
        if self._pieces is None:
            item, shape, strides = self.item_size, self.shape, self.strides
            inner, axis = shape[-1], len(shape) - 1
            while axis > 1 and (shape[axis - 1] == 1 or strides[axis - 1] == inner) and not (axis == 2 and len(shape) == 4):
                axis -= 1
                inner *= shape[axis]
            if axis > 2:
                raise shape_error(f"the positions and values of a state lie next to each other: got strides {strides}")
            counted = shape[-1] * item if len(shape) > 2 and axis <= len(shape) - 2 else 0
            self._pieces = (strides[0] * item, strides[1] * item if axis == 2 else 0, shape[1] if axis == 2 else 1, inner * item, counted)
        return self._pieces

    def as_split_pieces(self):
        """as_pieces() of (n, positions, values) with each position a piece of its own: beside a state whose positions do not lie densely."""
        item, (_, positions, values) = self.item_size, self.shape
        return self.strides[0] * item, self.strides[1] * item, positions, values * item, 0

    @classmethod
    def empty(cls, shape, type_: str, gpu_device: GpuDevice) -> "RowsGPU":
        if type_ not in ITEM_SIZE:
            raise capi.OperationNotSupported(f"rows of {type_}")
        return cls(gpu_device.create_empty_buffer(max(_dense(shape)[1] * ITEM_SIZE[type_], 1)), gpu_device, shape, type_)

    @classmethod
    def from_numpy(cls, values: np.ndarray, gpu_device: GpuDevice, type_: Optional[str] = None) -> "RowsGPU":
        """type_ "bf16": from float32 values, rounded to nearest even."""
        if type_ == "bf16":
            bits = np.ascontiguousarray(values, dtype=np.float32).view(np.uint32)
            nan = (bits & 0x7FFFFFFF) > 0x7F800000
            values = np.where(nan, 0x7FC0, (bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
        else:
            type_ = tensor_type(values) if type_ is None else type_
            if type_ not in ITEM_SIZE:
                raise capi.OperationNotSupported(f"rows of {type_}")
            values = np.ascontiguousarray(values, dtype=_NUMPY[type_])
        return cls(gpu_device.create_gpu_buffer_with_data(values), gpu_device, values.shape, type_)

    @classmethod
    def of_array(cls, array, shape) -> "RowsGPU":
        """The rows of a primitive array's values (a flat column read as rows), without a copy."""
        t = np.dtype(array.NP_DTYPE)
        if int(np.prod(shape)) != array.len:
            raise shape_error(f"{array.len} values are no rows of {tuple(shape)}")
        return cls(array.data, array.gpu_device, shape, t.kind + str(8 * t.itemsize))

    # -- read back
    def values(self) -> np.ndarray:
        """The values on the host (bf16: as float32).  Blocking."""
        span = 1 + sum((n - 1) * s for n, s in zip(self.shape, self.strides)) if 0 not in self.shape else 0
        settle(self.gpu_device, self)
        view = DeviceBuffer(self.gpu_device, self.ptr, span * self.item_size, owned=False)
        flat = self.gpu_device.retrive_data(view).view(_NUMPY[self.type])
        got = np.lib.stride_tricks.as_strided(flat, self.shape, [s * self.item_size for s in self.strides]).copy() if span else np.zeros(self.shape, _NUMPY[self.type])
        return (got.astype(np.uint32) << 16).view(np.float32) if self.type == "bf16" else got

    def __len__(self) -> int:
        return self.shape[0]

    def __repr__(self):
        return f"RowsGPU(shape={self.shape}, type={self.type})"


class QuantisedRowsGPU:
    """A cache of `n_slots` rows of heads x dim values in 8 or 4 bits, one factor for each group of `group` values.

    code "i8": whole numbers -127..127, "e4m3": 8-bit floating, "i4": whole numbers 0..15 above the group's lowest value.  An empty cache's rows
    read back as zeros."""

    PARTS = ("codes", "scales")
    __slots__ = ("codes", "scales", "gpu_device", "n_slots", "heads", "dim", "group", "code", "shape", "packed")

    def __init__(self, codes: DeviceBuffer, scales: DeviceBuffer, gpu_device: GpuDevice, n_slots: int, heads: int, dim: int, group: int, code: str):
        self._check(n_slots, heads, dim, group, code)
        need = self.bytes_of(n_slots, heads, dim, group, code)
        if (codes._owned and codes.nbytes < need[0]) or (scales._owned and scales.nbytes < need[1]):
            raise shape_error(f"{n_slots} rows of {heads} x {dim} need {need} bytes, not {codes.nbytes, scales.nbytes}")
        self.codes, self.scales, self.gpu_device = codes, scales, gpu_device
        self.n_slots, self.heads, self.dim, self.group, self.code = n_slots, heads, dim, group, code
        self.shape = (heads, dim)  # of a row
        self.packed = _PACK_STORE(codes.ptr, scales.ptr, n_slots, heads, dim, group, CODE_TYPE[code])

    @staticmethod
    def _check(n_slots, heads, dim, group, code):
        if code not in CODE_TYPE:
            raise capi.OperationNotSupported(f"codes of {code}")
        if heads < 1 or dim < 1 or heads * dim > 1 << 30 or not 1 <= group <= 65536 or dim % group or (code == "i4" and group % 2):
            raise shape_error(f"group {group} of {code} codes in rows of {heads} x {dim}")
        if not 0 <= n_slots <= 1 << 32:
            raise shape_error(f"a cache of {n_slots} rows")

    @staticmethod
    def bytes_of(n_slots: int, heads: int, dim: int, group: int, code: str):
        """(bytes of the codes, bytes of the scales)"""
        values = n_slots * heads * dim
        return (values // 2, values // group * 8) if code == "i4" else (values, values // group * 4)

    @classmethod
    def empty(cls, n_slots: int, heads: int, dim: int, gpu_device: GpuDevice, code: str = "i8", group: Optional[int] = None) -> "QuantisedRowsGPU":
        group = dim if group is None else group
        cls._check(n_slots, heads, dim, group, code)
        codes, scales = (gpu_device.create_empty_buffer(max(n, 1), zero_fill=True) for n in cls.bytes_of(n_slots, heads, dim, group, code))
        return cls(codes, scales, gpu_device, n_slots, heads, dim, group, code)

    @classmethod
    def of_tensors(cls, codes, scales, gpu_device: GpuDevice, code: str, heads: int, dim: int, group: int) -> "QuantisedRowsGPU":
        """The cache over two contiguous tensors' memory: codes (8-bit), scales (f32)."""
        cls._check(0, heads, dim, group, code)
        per = heads * dim // 2 if code == "i4" else heads * dim
        if codes.element_size() != 1 or tensor_type(scales) != "f32" or not codes.is_contiguous() or not scales.is_contiguous():
            raise shape_error("codes: a contiguous 8-bit tensor, scales: a contiguous f32 one")
        n_slots = codes.numel() // per
        want = cls.bytes_of(n_slots, heads, dim, group, code)
        if (codes.numel(), 4 * scales.numel()) != want:
            raise shape_error(f"{codes.numel()} codes and {scales.numel()} scales are no cache of rows of {heads} x {dim} in groups of {group}")
        return cls(borrow_tensor(codes, gpu_device, want[0]), borrow_tensor(scales, gpu_device, want[1]), gpu_device, n_slots, heads, dim, group, code)

    def __len__(self) -> int:
        return self.n_slots

    def __repr__(self):
        return f"QuantisedRowsGPU(n_slots={self.n_slots}, heads={self.heads}, dim={self.dim}, group={self.group}, code={self.code})"


class PageMap:
    """Where the rows of ragged sequences lie in a paged cache: row i of sequence s (offsets[s] <= i < offsets[s + 1]) is its position
    t = first[s] + i - offsets[s], in slot tables[s][t // page_rows] * page_rows + t % page_rows.

    tables: RowsGPU of u32 / i32, (sequences, pages); offsets: UInt32ArrayGPU of sequences + 1; first: UInt32ArrayGPU of sequences, or none."""

    PARTS = ("tables", "offsets", "first")
    __slots__ = ("tables", "page_rows", "offsets", "first", "packed")

    def __init__(self, tables: RowsGPU, page_rows: int, offsets: UInt32ArrayGPU, first: Optional[UInt32ArrayGPU] = None):
        if tables.type not in ("u32", "i32") or len(tables.shape) != 2:
            raise shape_error("page tables are rows of 32-bit page numbers")
        n = tables.shape[0]
        if (not isinstance(offsets, UInt32ArrayGPU) or offsets.null_buffer is not None
                or (first is not None and (not isinstance(first, UInt32ArrayGPU) or first.null_buffer is not None))):
            raise capi.OperationNotSupported("offsets and first positions: UInt32ArrayGPUs without nulls")
        if offsets.len != n + 1 or (first is not None and first.len != n):
            raise shape_error(f"{n} page tables need {n + 1} offsets and {n} first positions")
        if not 1 <= page_rows < 1 << 32:
            raise shape_error(f"pages of {page_rows} rows")
        self.tables, self.page_rows, self.offsets, self.first = tables, page_rows, offsets, first
        self.packed = _PACK_PAGES(tables.ptr, tables.strides[0], offsets.data.ptr, first.data.ptr if first is not None else 0, n, tables.shape[1],
                                  page_rows)


class BeamSelection:
    """What select_beams found, [batch, k] flat: scores (Float32ArrayGPU), parents (UInt32ArrayGPU: rows of the logits, indices for take_rows) and
    tokens (UInt32ArrayGPU), best first.  It holds the selection's workspace too: a selection that is passed as `out` again is not in use by two
    calls at one time, and lives as long as a captured graph that writes it."""

    PARTS = ("scores", "parents", "tokens")
    __slots__ = ("scores", "parents", "tokens", "gpu_device", "batch", "k", "workspace", "_workspace_of", "_outgrown")

    def __init__(self, scores: Float32ArrayGPU, parents: UInt32ArrayGPU, tokens: UInt32ArrayGPU, gpu_device: GpuDevice, batch: int, k: int):
        if not (scores.len == parents.len == tokens.len == batch * k):
            raise shape_error(f"a selection of {batch} x {k} has that many scores, parents and tokens")
        self.scores, self.parents, self.tokens, self.gpu_device = scores, parents, tokens, gpu_device
        self.batch, self.k = batch, k
        self.workspace = self._workspace_of = None
        self._outgrown = []

    @classmethod
    def empty(cls, batch: int, k: int, gpu_device: GpuDevice) -> "BeamSelection":
        made = [c(gpu_device.create_empty_buffer(max(4 * batch * k, 1)), gpu_device, batch * k, None) for c in (Float32ArrayGPU, UInt32ArrayGPU, UInt32ArrayGPU)]
        return cls(*made, gpu_device, batch, k)

    @classmethod
    def of_tensors(cls, scores, parents, tokens, gpu_device: GpuDevice) -> "BeamSelection":
        """Over three contiguous [batch, k] tensors' memory: f32 scores, 32-bit parents and tokens."""
        if len(scores.shape) != 2 or tuple(parents.shape) != tuple(scores.shape) or tuple(tokens.shape) != tuple(scores.shape):
            raise shape_error("a selection's tensors are all [batch, k]")
        return cls(Float32ArrayGPU.of_tensor(scores, gpu_device), UInt32ArrayGPU.of_tensor(parents, gpu_device),
                   UInt32ArrayGPU.of_tensor(tokens, gpu_device), gpu_device, scores.shape[0], scores.shape[1])

    def ensure_workspace(self, beams: int, vocab: int) -> DeviceBuffer:
        """The workspace for rows of `vocab` logits, `beams` a request."""
        if self._workspace_of != (beams, vocab):
            nbytes = capi.select_beams_workspace(self.batch, beams, vocab, self.k)
            if self.workspace is None or self.workspace.nbytes < nbytes:
                if self.workspace is not None:
                    self._outgrown.append(self.workspace)  # a captured graph may hold it
                self.workspace = self.gpu_device.create_empty_buffer(max(nbytes, 16))
            self._workspace_of = (beams, vocab)
        return self.workspace

    def values(self):
        """(scores, parents, tokens) as [batch, k] arrays on the host.  Blocking."""
        return tuple(a.raw_values().reshape(self.batch, self.k) for a in (self.scores, self.parents, self.tokens))


__all__ = ["RowsGPU", "QuantisedRowsGPU", "PageMap", "BeamSelection"]

"""Operators on whole rows (include/arrow_gpu.h "rows"): put_quantised / take_quantised — take and put with a cast to 8 or 4 bits between them —
select_beams, whose parents are an index column, and take_rows, which reorders the states by it.  No counterpart in the reference.

As everywhere here the `*_op` forms enqueue on a pipeline and return without waiting; the plain forms run on a pipeline of their own — over tensors'
memory on torch's current stream — and wait, so that an index out of range is raised by the call.  `out` writes into memory the caller has (a torch
tensor's, last step's)."""
from __future__ import annotations

import struct

from .. import _capi as capi
from ..array import BooleanArrayGPU, Float32ArrayGPU, UInt32ArrayGPU
from ..gpu_utils import ArrowComputePipeline, pipeline_for
from ..rows import ROW_TYPE, BeamSelection, PageMap, QuantisedRowsGPU, RowsGPU, shape_error

_MAX_COLUMNS = 64
_PACK_STATE = struct.Struct("=QQQQQQQQQ")            # agpu_state
_PACK_BEAMS = struct.Struct("=QQiIIIIIQQQQQQQQQ")  # agpu_beams


def _keep(pipeline, *buffers) -> None:
    """The buffers of a call, until the pipeline's sync(); tensors' memory only where torch's stream does not keep its order."""
    if pipeline.own_stream:
        pipeline.keep(*buffers)
        return
    for b in buffers:
        if b._owned:
            pipeline.keep(b)


def _on(pipeline, *things) -> None:
    dev = pipeline.device
    for t in things:
        if t.gpu_device is not dev and t.gpu_device.ordinal != dev.ordinal:
            raise capi.ArrowErrorGPU("ArgumentError", f"memory of GPU {t.gpu_device.ordinal} in a pipeline of GPU {dev.ordinal}", capi.ERR_ARG)


def _u32(array, what: str):
    if not isinstance(array, UInt32ArrayGPU) or array.null_buffer is not None:
        raise capi.OperationNotSupported(f"{what}: a UInt32ArrayGPU without nulls")
    return array


def _quantised(name: str, stores, rows, where, n: int, pipeline) -> None:
    if len(stores) > _MAX_COLUMNS:
        raise shape_error(f"{len(stores)} caches in one call: at most {_MAX_COLUMNS}")
    dev, s, r = pipeline.device, b"", b""
    for store, x in zip(stores, rows):
        shape = x.shape
        if shape[0] != n or (shape[1:] != store.shape and (store.heads != 1 or shape[1:] != store.shape[1:])):
            raise shape_error(f"rows {shape} for {n} rows of {store.heads} x {store.dim}")
        if x.gpu_device is not dev or store.gpu_device is not dev:
            _on(pipeline, store, x)
        s += store.packed
        r += x._rows or x.as_rows()
    if isinstance(where, PageMap):
        held = (where.tables, where.offsets) if where.first is None else (where.tables, where.offsets, where.first)
        _on(pipeline, *held)
        capi.call(name + "_pages", pipeline._handle, len(stores), s, r, where.packed, n)
        _keep(pipeline, *[x.data for x in held])
    else:
        if where.gpu_device is not dev:
            _on(pipeline, where)
        capi.call(name, pipeline._handle, len(stores), s, r, where.data.ptr, n)
        if where.data._owned or pipeline.own_stream:
            pipeline.keep(where.data)
    own = pipeline.own_stream
    for store, x in zip(stores, rows):
        if own or store.codes._owned or store.scales._owned or x.data._owned:
            _keep(pipeline, store.codes, store.scales, x.data)


def put_quantised_op(stores, rows, where, pipeline: ArrowComputePipeline) -> None:
    """stores[c] row where[i] = rows[c] row i, quantised: the columns of one table (keys and values, of one layer or of all) by one slot column.

    where: a UInt32ArrayGPU of slots (0xFFFFFFFF: not stored) or a PageMap.  A slot out of range is dropped, and ShapeError at the next sync."""
    stores = [stores] if isinstance(stores, QuantisedRowsGPU) else stores
    rows = [rows] if isinstance(rows, RowsGPU) else rows
    if len(stores) != len(rows):
        raise shape_error(f"{len(rows)} rows for {len(stores)} caches")
    if not stores:
        return
    n = len(rows[0])
    if not isinstance(where, PageMap) and _u32(where, "slots").len != n:
        raise shape_error(f"{where.len} slots for {n} rows")
    _quantised("agpu_put_quantised", stores, rows, where, n, pipeline)


def take_quantised_op(stores, where, pipeline: ArrowComputePipeline, type_: str = "f32", n_rows: int | None = None, out=None) -> list:
    """[rows of every store], row i = the values of row where[i], in `type_` ("f32", "f16", "bf16").

    where: a UInt32ArrayGPU of slots or a PageMap; with a PageMap `n_rows` (or `out`) says how many rows there are.  A row that `where` names none
    for (0xFFFFFFFF, behind the last sequence) is left as it was — in `out`; in memory allocated here it is unspecified.  A slot out of range gives
    zeros, and ShapeError at the next sync."""
    stores = [stores] if isinstance(stores, QuantisedRowsGPU) else stores
    out = [out] if isinstance(out, RowsGPU) else out
    if not stores:
        return []
    if out is not None:
        if len(out) != len(stores):
            raise shape_error(f"{len(out)} outputs for {len(stores)} caches")
        n = len(out[0])
    elif isinstance(where, PageMap):
        if n_rows is None:
            raise shape_error("take_quantised through a page map: how many rows? (n_rows or out)")
        n = int(n_rows)
        if n < 0:
            raise shape_error(f"{n} rows")
    else:
        n = _u32(where, "slots").len
    if not isinstance(where, PageMap) and _u32(where, "slots").len != n:
        raise shape_error(f"{where.len} slots for {n} rows")
    if out is None:
        out = [RowsGPU.empty((n, s.heads, s.dim), type_, s.gpu_device) for s in stores]
    _quantised("agpu_take_quantised", stores, out, where, n, pipeline)
    return out


def take_rows_op(states, indexes: UInt32ArrayGPU, pipeline: ArrowComputePipeline, lengths: UInt32ArrayGPU | None = None, out=None) -> list:
    """[row indexes[i] of every state]: the states reordered by a selection's parents (any element type, 2 to 4 axes: rows, (pieces,) (positions,)
    values; the positions of four axes lie next to each other, of three they may lie apart).  lengths: per row how many positions (the axis before the last,
    next to each other) hold anything; what lies behind them is left as it was in `out` (in memory allocated here: unspecified).  An index out of range gives a row of zeros, and ShapeError at the next sync; 0xFFFFFFFF leaves it."""
    states = [states] if isinstance(states, RowsGPU) else states
    out = [out] if isinstance(out, RowsGPU) else out
    n = _u32(indexes, "indexes").len
    if lengths is not None and _u32(lengths, "lengths").len != n:
        raise shape_error(f"{lengths.len} lengths for {n} rows")
    if not states:
        return []
    if len(states) > _MAX_COLUMNS:
        raise shape_error(f"{len(states)} states in one call: at most {_MAX_COLUMNS}")
    if out is None:
        out = [RowsGPU.empty((n,) + tuple(s.shape[1:]), s.type, s.gpu_device) for s in states]
    if len(out) != len(states):
        raise shape_error(f"{len(out)} outputs for {len(states)} states")
    n_src, dev, packed = states[0].shape[0], pipeline.device, b""
    for s, o in zip(states, out):
        here, there = s.shape, o.shape
        if here[0] != n_src or there[0] != n or o.item_size != s.item_size or (here != there and here[1:] != there[1:]):
            raise shape_error(f"rows {there} from a state {here} by {n} indexes, in a call over {n_src} rows")
        row, step, pieces, size, position = s._pieces or s.as_pieces()
        out_row, out_step, out_pieces, out_size, _ = o._pieces or o.as_pieces()
        if (pieces, size) != (out_pieces, out_size):  # of three axes, one of the two dense and the other not
            row, step, pieces, size, position = s.as_split_pieces()
            out_row, out_step, *_ = o.as_split_pieces()
        if lengths is not None and not position:
            raise shape_error("lengths count positions, the axis before the last: they lie next to each other")
        packed += _PACK_STATE.pack(s.ptr, o.ptr, row, step, out_row, out_step, pieces, size, position)
        if s.gpu_device is not dev or o.gpu_device is not dev:
            _on(pipeline, s, o)
    given = (indexes,) if lengths is None else (indexes, lengths)
    for x in given:
        if x.gpu_device is not dev:
            _on(pipeline, x)
    capi.call("agpu_take_rows", pipeline._handle, len(states), packed, n_src, indexes.data.ptr, lengths.data.ptr if lengths is not None else None, n)
    own = pipeline.own_stream
    for x in given:
        if own or x.data._owned:
            pipeline.keep(x.data)
    for s, o in zip(states, out):
        if own or s.data._owned or o.data._owned:
            _keep(pipeline, s.data, o.data)
    return out


def select_beams_op(logits: RowsGPU, beams: int, k: int, pipeline: ArrowComputePipeline, scores: Float32ArrayGPU | None = None,
                    allowed: BooleanArrayGPU | None = None, finished: BooleanArrayGPU | None = None, end_token: int = 0,
                    out: BeamSelection | None = None) -> BeamSelection:
    """Per request the k best of its beams x tokens by scores[row] + log_softmax(logits[row])[token], best first.

    logits: rows of (batch * beams, vocab).  scores: the rows' running scores (none: 0).  allowed: a bitmap of one row's, or of every row's,
    vocab bits, each row's on a multiple of 64 bits.  finished: a bitmap of the rows; a finished row's one candidate is (end_token, its score)."""
    if logits.type not in ROW_TYPE:
        raise capi.OperationNotSupported(f"logits of {logits.type}")
    if len(logits.shape) != 2 or beams < 1 or logits.shape[0] % beams:
        raise shape_error(f"logits {logits.shape} of {beams} beams a request")
    rows, vocab = logits.shape
    if vocab >= 1 << 31 or rows >= 1 << 24:
        raise shape_error(f"logits {logits.shape}: less than 2^24 rows of less than 2^31")
    batch, pitch = rows // beams, (vocab + 63) // 64 * 64
    if scores is not None and (not isinstance(scores, Float32ArrayGPU) or scores.null_buffer is not None or scores.len != rows):
        raise shape_error(f"scores: a Float32ArrayGPU of {rows} values without nulls")
    stride = 0
    if allowed is not None:
        if not isinstance(allowed, BooleanArrayGPU) or allowed.null_buffer is not None or allowed.len not in (rows * pitch, pitch, vocab):
            raise shape_error(f"allowed: a BooleanArrayGPU of {rows} x {pitch} bits, or of one row's, without nulls")
        stride = pitch // 8 if allowed.len == rows * pitch else 0
    if finished is not None and (not isinstance(finished, BooleanArrayGPU) or finished.null_buffer is not None or finished.len != rows):
        raise shape_error(f"finished: a BooleanArrayGPU of {rows} bits without nulls")
    if not 0 <= end_token < vocab:
        raise shape_error(f"end_token {end_token} of {vocab} tokens")
    if not 1 <= k <= 64 or k > beams * vocab:
        raise shape_error(f"k {k}: 1 to 64, at most {beams} x {vocab}")
    if out is None:
        out = BeamSelection.empty(batch, k, pipeline.device)
    elif (out.batch, out.k) != (batch, k):
        raise shape_error(f"a selection of {out.batch} x {out.k} for {batch} x {k}")
    dev, given = pipeline.device, [x for x in (logits, scores, allowed, finished) if x is not None]
    if out.gpu_device is not dev:
        _on(pipeline, out)
    for x in given:
        if x.gpu_device is not dev:
            _on(pipeline, x)
    if batch == 0:
        return out
    work = out.workspace if out._workspace_of == (beams, vocab) else out.ensure_workspace(beams, vocab)
    args = _PACK_BEAMS.pack(logits.ptr, logits.strides[0], ROW_TYPE[logits.type], batch, beams, vocab, k, end_token,
                            scores.data.ptr if scores is not None else 0, allowed.data.ptr if allowed is not None else 0, stride,
                            finished.data.ptr if finished is not None else 0, out.scores.data.ptr, out.parents.data.ptr, out.tokens.data.ptr,
                            work.ptr, work.nbytes)
    capi.call("agpu_select_beams", pipeline._handle, args)
    own = pipeline.own_stream
    for x in given:
        if own or x.data._owned:
            pipeline.keep(x.data)
    _keep(pipeline, out.scores.data, out.parents.data, out.tokens.data, work)
    return out


def _waited(device, label: str, op, *things):
    p = pipeline_for(device, label, *things)
    got = op(p)
    p.finish()
    p.sync()  # surfaces an index out of range here
    return got


def _device_of(where):
    return where.tables.gpu_device if isinstance(where, PageMap) else _u32(where, "slots").gpu_device


def put_quantised(stores, rows, where) -> None:
    _waited(_device_of(where), "put_quantised", lambda p: put_quantised_op(stores, rows, where, p), stores, rows, where)


def take_quantised(stores, where, type_: str = "f32", n_rows: int | None = None, out=None) -> list:
    return _waited(_device_of(where), "take_quantised", lambda p: take_quantised_op(stores, where, p, type_, n_rows, out), stores, where, out)


def take_rows(states, indexes: UInt32ArrayGPU, lengths: UInt32ArrayGPU | None = None, out=None) -> list:
    return _waited(indexes.gpu_device, "take_rows", lambda p: take_rows_op(states, indexes, p, lengths, out), states, indexes, lengths, out)


def select_beams(logits: RowsGPU, beams: int, k: int, scores: Float32ArrayGPU | None = None, allowed: BooleanArrayGPU | None = None,
                 finished: BooleanArrayGPU | None = None, end_token: int = 0, out: BeamSelection | None = None) -> BeamSelection:
    return _waited(logits.gpu_device, "select_beams", lambda p: select_beams_op(logits, beams, k, p, scores, allowed, finished, end_token, out),
                   logits, scores, allowed, finished, out)


__all__ = ["put_quantised", "put_quantised_op", "take_quantised", "take_quantised_op", "take_rows", "take_rows_op", "select_beams", "select_beams_op"]

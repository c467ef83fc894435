"""CPU: the row operators' refusals (argument checks come before anything touches a device: with valid arguments the only complaint left is the
missing pipeline), the Python host's, and the slot arithmetic of the page tables — broken tables too — compiled for the host."""
import ctypes as C
import os
import subprocess
import types

import numpy as np
import pytest

import rows_ref as R
from arrow_gpu_amd import _capi as capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NO_PIPELINE = (capi.ERR_ARG, "null pipeline")


# the ABI's structs, field by field (the Python host packs them as bytes)
class RowsStruct(C.Structure):  # agpu_rows
    _fields_ = [("data", C.c_void_p), ("row_stride", C.c_uint64), ("head_stride", C.c_uint64), ("type", C.c_int32)]


class QuantisedRowsStruct(C.Structure):  # agpu_quantised_rows
    _fields_ = [("codes", C.c_void_p), ("scales", C.c_void_p), ("n_slots", C.c_uint64), ("heads", C.c_uint32), ("dim", C.c_uint32),
                ("group", C.c_uint32), ("code", C.c_int32)]


class PageMapStruct(C.Structure):  # agpu_page_map
    _fields_ = [("tables", C.c_void_p), ("table_stride", C.c_uint64), ("offsets", C.c_void_p), ("first", C.c_void_p), ("n_seqs", C.c_uint32),
                ("max_pages", C.c_uint32), ("page_rows", C.c_uint32)]


class StateStruct(C.Structure):  # agpu_state
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("src_row_stride", C.c_uint64), ("src_piece_stride", C.c_uint64),
                ("dst_row_stride", C.c_uint64), ("dst_piece_stride", C.c_uint64), ("n_pieces", C.c_uint64), ("piece_bytes", C.c_uint64),
                ("position_bytes", C.c_uint64)]


class BeamsStruct(C.Structure):  # agpu_beams
    _fields_ = [("logits", C.c_void_p), ("row_stride", C.c_uint64), ("type", C.c_int32), ("batch", C.c_uint32), ("beams", C.c_uint32),
                ("vocab", C.c_uint32), ("k", C.c_uint32), ("end_token", C.c_uint32), ("scores", C.c_void_p), ("allowed", C.c_void_p),
                ("allowed_stride", C.c_uint64), ("finished", C.c_void_p), ("out_scores", C.c_void_p), ("out_parents", C.c_void_p),
                ("out_tokens", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


def status(name, *args):
    st = getattr(capi.lib(), name)(*args)
    return st, capi.last_error()


def store(**kw):
    a = dict(codes=1 << 20, scales=1 << 21, n_slots=8, heads=2, dim=64, group=32, code=capi.CODE_I8)
    a.update(kw)
    return QuantisedRowsStruct(**a)


def rows(**kw):
    a = dict(data=1 << 22, row_stride=128, head_stride=64, type=capi.ROW_BF16)
    a.update(kw)
    return RowsStruct(**a)


@pytest.mark.parametrize("name", ["agpu_put_quantised", "agpu_take_quantised"])
@pytest.mark.parametrize("kw,rw,code,text", [
    ({}, {}, *NO_PIPELINE),
    (dict(code=3), {}, capi.ERR_ARG, "code type"), (dict(code=-1), {}, capi.ERR_ARG, "code type"),
    ({}, dict(type=3), capi.ERR_ARG, "row type"),
    (dict(heads=0), {}, capi.ERR_SHAPE, "heads"), (dict(dim=0), {}, capi.ERR_SHAPE, "heads"), (dict(heads=1 << 20, dim=1 << 12, group=1 << 12), {}, capi.ERR_SHAPE, "heads"),
    (dict(group=0), {}, capi.ERR_SHAPE, "group"), (dict(group=48), {}, capi.ERR_SHAPE, "group"), (dict(heads=1, dim=1 << 17, group=1 << 17), {}, capi.ERR_SHAPE, "group"),
    (dict(code=capi.CODE_I4, dim=9, group=9), {}, capi.ERR_SHAPE, "even"),
    (dict(n_slots=(1 << 32) + 1), {}, capi.ERR_SHAPE, "n_slots"),
    (dict(codes=0), {}, capi.ERR_ARG, "null"), (dict(scales=0), {}, capi.ERR_ARG, "null"), ({}, dict(data=0), capi.ERR_ARG, "null"),
    ({}, dict(data=(1 << 22) + 1), capi.ERR_SHAPE, "alignment"), ({}, dict(data=(1 << 22) + 2, type=capi.ROW_F32), capi.ERR_SHAPE, "alignment"),
    (dict(scales=(1 << 21) + 2), {}, capi.ERR_SHAPE, "alignment")])
def test_quantised_arguments(name, kw, rw, code, text):
    st, msg = status(name, None, 1, C.byref(store(**kw)), C.byref(rows(**rw)), 1 << 23, 4)
    assert st == code and text in msg, msg


def test_quantised_calls():
    s, r = store(), rows()
    for name in ("agpu_put_quantised", "agpu_take_quantised"):
        assert status(name, None, 65, C.byref(s), C.byref(r), 1 << 23, 4)[0] == capi.ERR_ARG
        assert status(name, None, -1, C.byref(s), C.byref(r), 1 << 23, 4)[0] == capi.ERR_ARG
        assert "null pointer" in status(name, None, 1, C.byref(s), C.byref(r), None, 4)[1]
        assert "null pointer" in status(name, None, 1, None, C.byref(r), 1 << 23, 4)[1]
        assert "alignment" in status(name, None, 1, C.byref(s), C.byref(r), (1 << 23) + 1, 4)[1]
        assert status(name, None, 1, C.byref(s), C.byref(r), 1 << 23, 1 << 31)[0] == capi.ERR_SHAPE
        assert NO_PIPELINE[1] in status(name, None, 0, None, None, None, 4)[1]  # nothing to do, but still a pipeline's call
        assert NO_PIPELINE[1] in status(name, None, 1, None, None, None, 0)[1]
    # rows that are written may not lie on each other; read ones may (a broadcast row)
    assert NO_PIPELINE[1] in status("agpu_take_quantised", None, 1, C.byref(s), C.byref(rows(row_stride=64, head_stride=256)), 1 << 23, 4)[1]  # heads, then rows
    assert NO_PIPELINE[1] in status("agpu_take_quantised", None, 1, C.byref(s), C.byref(rows(row_stride=0, head_stride=64)), 1 << 23, 1)[1]     # one row
    for kw in (dict(head_stride=63), dict(row_stride=63), dict(head_stride=0), dict(row_stride=64, head_stride=64), dict(row_stride=127), dict(row_stride=64, head_stride=255),
               dict(row_stride=(1 << 64) - 1, head_stride=1)):
        assert "overlap" in status("agpu_take_quantised", None, 1, C.byref(s), C.byref(rows(**kw)), 1 << 23, 4)[1]
        assert NO_PIPELINE[1] in status("agpu_put_quantised", None, 1, C.byref(s), C.byref(rows(**kw)), 1 << 23, 4)[1]


def test_page_arguments():
    def pages(**kw):
        a = dict(tables=1 << 24, table_stride=4, offsets=1 << 25, first=None, n_seqs=3, max_pages=4, page_rows=16)
        a.update(kw)
        return PageMapStruct(**a)

    s, r = store(), rows()
    for name in ("agpu_put_quantised_pages", "agpu_take_quantised_pages"):
        call = lambda m: status(name, None, 1, C.byref(s), C.byref(r), C.byref(m), 4)  # noqa: E731, B023
        assert NO_PIPELINE[1] in call(pages())[1]
        assert NO_PIPELINE[1] in call(pages(tables=None, max_pages=0))[1]
        assert call(pages(tables=None))[0] == capi.ERR_ARG
        assert call(pages(offsets=None))[0] == capi.ERR_ARG
        for kw in (dict(n_seqs=0), dict(n_seqs=1 << 31), dict(page_rows=0), dict(tables=(1 << 24) + 1), dict(offsets=(1 << 25) + 2), dict(first=3)):
            assert call(pages(**kw))[0] == capi.ERR_SHAPE, kw
        assert status(name, None, 1, C.byref(s), C.byref(r), None, 4)[0] == capi.ERR_ARG


def test_take_rows_arguments():
    def state(**kw):
        a = dict(src=1 << 30, dst=1 << 40, src_row_stride=4096, src_piece_stride=1024, dst_row_stride=4096, dst_piece_stride=1024, n_pieces=4, piece_bytes=1024, position_bytes=64)
        a.update(kw)
        return StateStruct(**a)

    def call(*states, n_src=8, idx=1 << 20, lengths=None, n=8):
        v = (StateStruct * max(len(states), 1))(*states)
        return status("agpu_take_rows", None, len(states), v, n_src, idx, lengths, n)

    assert NO_PIPELINE[1] in call(state())[1] and NO_PIPELINE[1] in call()[1] and NO_PIPELINE[1] in call(state(), n=0)[1]
    assert NO_PIPELINE[1] in call(state(), lengths=1 << 21)[1]
    assert call(*[state()] * 65)[0] == capi.ERR_ARG
    assert call(state(), idx=None)[0] == capi.ERR_ARG
    assert call(state(src=None))[0] == capi.ERR_ARG and call(state(dst=None))[0] == capi.ERR_ARG
    assert NO_PIPELINE[1] in call(state(src=None), n_src=0)[1]  # no rows to take from: every index is out of range
    assert call(state(), idx=(1 << 20) + 2)[0] == capi.ERR_SHAPE and call(state(), lengths=(1 << 20) + 2)[0] == capi.ERR_SHAPE
    assert "overlap" in call(state(dst_row_stride=1024))[1] and NO_PIPELINE[1] in call(state(dst_row_stride=1024, dst_piece_stride=8192))[1]
    assert "overlap" in call(state(dst_piece_stride=1023))[1] and "overlap" in call(state(dst_row_stride=100))[1]
    assert "position_bytes" in call(state(position_bytes=0), lengths=1 << 21)[1]
    assert NO_PIPELINE[1] in call(state(position_bytes=0))[1]
    assert "address space" in call(state(src_row_stride=1 << 62))[1] and "address space" in call(state(n_pieces=1 << 40, piece_bytes=1 << 30, dst_piece_stride=1 << 30))[1]
    assert "address space" in call(state(piece_bytes=(1 << 64) - 1, dst_piece_stride=(1 << 64) - 1, dst_row_stride=(1 << 64) - 1))[1]
    assert "2^31" in call(state(n_pieces=1, piece_bytes=1 << 31, src=1 << 43, dst=1 << 42, src_row_stride=1 << 31, dst_row_stride=1 << 31))[1]
    # in place, by one byte, and one state's dst on another's src
    assert call(state(dst=1 << 30))[0] == capi.ERR_ARG
    assert call(state(dst=(1 << 30) + 8 * 4096 - 1))[0] == capi.ERR_ARG and NO_PIPELINE[1] in call(state(dst=(1 << 30) + 8 * 4096))[1]
    assert call(state(dst=(1 << 30) - 8 * 4096 + 1))[0] == capi.ERR_ARG and NO_PIPELINE[1] in call(state(dst=(1 << 30) - 8 * 4096))[1]
    assert call(state(), state(src=1 << 40, dst=1 << 41))[0] == capi.ERR_ARG


def test_select_beams_arguments():
    def beams(**kw):
        a = dict(logits=1 << 20, row_stride=1000, type=capi.ROW_F16, batch=2, beams=4, vocab=1000, k=8, end_token=0, scores=1 << 21, allowed=1 << 22, allowed_stride=128,
                 finished=1 << 23, out_scores=1 << 24, out_parents=1 << 25, out_tokens=1 << 26, workspace=1 << 27, workspace_bytes=1 << 30)
        a.update(kw)
        return status("agpu_select_beams", None, C.byref(BeamsStruct(**a)))

    assert NO_PIPELINE[1] in beams()[1] and NO_PIPELINE[1] in beams(batch=0, logits=0)[1]
    assert NO_PIPELINE[1] in beams(row_stride=0)[1]
    assert NO_PIPELINE[1] in beams(scores=0, allowed=0, finished=0, allowed_stride=0)[1]
    assert status("agpu_select_beams", None, None)[0] == capi.ERR_ARG
    for kw in (dict(type=3), dict(logits=0), dict(out_scores=0), dict(out_parents=0), dict(out_tokens=0), dict(workspace=0)):
        assert beams(**kw)[0] == capi.ERR_ARG, kw
    for kw in (dict(k=0), dict(k=65), dict(beams=0), dict(beams=1025), dict(vocab=0), dict(vocab=1 << 31), dict(k=9, beams=1, vocab=8), dict(batch=1 << 22),
               dict(workspace_bytes=8), dict(end_token=1000), dict(allowed_stride=120), dict(allowed_stride=132), dict(logits=(1 << 20) + 1),
               dict(scores=(1 << 21) + 1), dict(allowed=(1 << 22) + 4), dict(finished=(1 << 23) + 4), dict(out_scores=(1 << 24) + 2), dict(out_tokens=(1 << 26) + 2),
               dict(workspace=(1 << 27) + 8)):
        assert beams(**kw)[0] == capi.ERR_SHAPE, kw
    # 2 x 8 results of 4 bytes, 8 scores: where the last step's scores are, on the workspace, and just beside both
    for out in ("out_scores", "out_parents", "out_tokens"):
        for at in ((1 << 21), (1 << 21) + 28, (1 << 21) - 60):
            assert "scores" in beams(**{out: at})[1]
        assert "workspace" in beams(**{out: (1 << 27) + 64})[1] and "workspace" in beams(**{out: (1 << 27) - 60})[1]
        for at in ((1 << 21) + 32, (1 << 21) - 64, (1 << 27) - 64):
            assert NO_PIPELINE[1] in beams(**{out: at})[1]
        assert NO_PIPELINE[1] in beams(**{out: 1 << 21, "scores": 0})[1]
    n = C.c_uint64(1)
    assert status("agpu_select_beams_workspace", 0, 0, 0, 0, C.byref(n))[0] == 0 and n.value == 0
    assert status("agpu_select_beams_workspace", 2, 4, 1000, 8, C.byref(n))[0] == 0 and n.value > 0
    assert status("agpu_select_beams_workspace", 2, 4, 1000, 8, None)[0] == capi.ERR_ARG


def test_what_a_selection_writes_lies_apart():
    """outputs on each other or on the bitmap of finished rows, the workspace on an input: blocks would write what others still read"""
    def beams(**kw):
        a = dict(logits=1 << 20, row_stride=1000, type=capi.ROW_F16, batch=2, beams=4, vocab=1000, k=8, end_token=0, scores=1 << 21, allowed=1 << 22, allowed_stride=128,
                 finished=1 << 23, out_scores=1 << 24, out_parents=1 << 25, out_tokens=1 << 26, workspace=1 << 27, workspace_bytes=1 << 30)
        a.update(kw)
        return status("agpu_select_beams", None, C.byref(BeamsStruct(**a)))

    assert "two outputs" in beams(out_parents=1 << 24)[1] and "two outputs" in beams(out_tokens=(1 << 25) + 60)[1] and "two outputs" in beams(out_tokens=(1 << 24) - 60)[1]
    for at in ((1 << 24) + 64, (1 << 24) - 64):
        assert NO_PIPELINE[1] in beams(out_parents=at)[1]
    for out in ("out_scores", "out_parents", "out_tokens"):
        assert "finished" in beams(**{out: 1 << 23})[1] and "finished" in beams(**{out: (1 << 23) + 4})[1] and "finished" in beams(**{out: (1 << 23) - 60})[1]
        assert NO_PIPELINE[1] in beams(**{out: (1 << 23) + 8})[1] and NO_PIPELINE[1] in beams(**{out: (1 << 23) - 64})[1]
        assert NO_PIPELINE[1] in beams(**{out: 1 << 23, "finished": 0})[1]
    n = C.c_uint64()
    assert status("agpu_select_beams_workspace", 2, 4, 1000, 8, C.byref(n))[0] == 0
    for at, size in ((1 << 20, 16000), (1 << 21, 32), (1 << 22, 1024), (1 << 23, 8)):  # logits, scores, masks, finished rows
        last = (at + size - 1) // 16 * 16
        assert "workspace" in beams(workspace=at)[1] and "workspace" in beams(workspace=last)[1] and "workspace" in beams(workspace=at - (n.value - 1) // 16 * 16)[1]
        assert NO_PIPELINE[1] in beams(workspace=last + 16)[1] and NO_PIPELINE[1] in beams(workspace=at - (n.value + 15) // 16 * 16)[1]
    assert NO_PIPELINE[1] in beams(workspace=(1 << 20) + 2000, row_stride=0)[1]  # one row for all
    assert "workspace" in beams(workspace=(1 << 22) + 112, allowed_stride=0)[1] and NO_PIPELINE[1] in beams(workspace=(1 << 22) + 128, allowed_stride=0)[1]
    assert "address space" in beams(row_stride=1 << 62)[1]


def test_the_largest_calls():
    """what a launch's threads and 31-bit counts bound is refused, what the documentation allows is not"""
    n = C.c_uint64(0)
    workspace = lambda batch, beams, vocab, k: status("agpu_select_beams_workspace", batch, beams, vocab, k, C.byref(n))[0]  # noqa: E731
    for batch, beams, vocab, k in ((1, 1, (1 << 31) - 1, 64), (127, 1, (1 << 31) - 1, 1), (1, 64, (1 << 31) - 1, 64), (1 << 14, 1023, 8191, 64), (1, 1024, 1 << 26, 64),
                                   (1 << 14, 1023, 1, 1), ((1 << 24) - 1, 1, 1 << 14, 64)):
        assert batch * beams * vocab < 1 << 38 and beams * k * vocab < 1 << 43
        assert workspace(batch, beams, vocab, k) == 0 and n.value > 0, (batch, beams, vocab, k)
    for batch, beams, vocab, k in ((1, 1024, (1 << 31) - 1, 64), (1 << 13, 1, (1 << 31) - 1, 1), (1 << 23, 1, 1 << 20, 1)):
        assert workspace(batch, beams, vocab, k) == capi.ERR_SHAPE, (batch, beams, vocab, k)
    s, r = store(heads=1 << 13, dim=1 << 6, group=64), rows(row_stride=1 << 19)
    assert NO_PIPELINE[1] in status("agpu_put_quantised", None, 1, C.byref(s), C.byref(r), 1 << 23, 1 << 28)[1]
    assert "2^48" in status("agpu_put_quantised", None, 1, C.byref(s), C.byref(r), 1 << 23, 1 << 29)[1]


def test_positions_larger_than_a_piece():
    """2^31 positions of 2^33 bytes are 2^64: the kernel's product would wrap, and of a row that is copied whole nothing would be"""
    for position, ok in ((1, True), (1024, True), (1025, False), (1 << 33, False), ((1 << 64) - 1, False)):
        s = StateStruct(1 << 30, 1 << 40, 4096, 1024, 4096, 1024, 4, 1024, position)
        st, msg = status("agpu_take_rows", None, 1, C.byref(s), 8, 1 << 20, 1 << 21, 8)
        assert (NO_PIPELINE[1] in msg) == ok and (ok or (st == capi.ERR_SHAPE and "position_bytes" in msg)), (position, msg)
        assert NO_PIPELINE[1] in status("agpu_take_rows", None, 1, C.byref(s), 8, 1 << 20, None, 8)[1]  # no lengths, no positions


def test_what_is_written_lies_apart():
    """two outputs on each other, an output on an index column or on a cache; and what lies interleaved in one allocation is none of these"""
    def state(**kw):
        a = dict(src=1 << 30, dst=1 << 40, src_row_stride=4096, src_piece_stride=1024, dst_row_stride=4096, dst_piece_stride=1024, n_pieces=4, piece_bytes=1024, position_bytes=64)
        a.update(kw)
        return StateStruct(**a)

    def call(*states, idx=1 << 20, lengths=None):
        return status("agpu_take_rows", None, len(states), (StateStruct * len(states))(*states), 8, idx, lengths, 8)

    other = dict(src=1 << 31)
    for dst in (1 << 40, (1 << 40) + 8 * 4096 - 1, (1 << 40) - 8 * 4096 + 1, (1 << 40) + 1024):
        assert call(state(), state(**other, dst=dst))[0] == capi.ERR_ARG and "dsts" in capi.last_error()
    assert NO_PIPELINE[1] in call(state(), state(**other, dst=(1 << 40) + 8 * 4096))[1]
    # the halves of rows of 8192 bytes, of pieces of 2048; source and destination of one state, and two states
    row, piece = dict(src_row_stride=8192, dst_row_stride=8192), dict(src_row_stride=8192, dst_row_stride=8192, src_piece_stride=2048, dst_piece_stride=2048)
    for kw, step in ((row, 4096), (piece, 1024)):
        for off, ok in ((step, True), (-step, True), (0, False), (step - 1, False), (step + 1, False), (8 * 8192 + step, True), (3 * 8192 - step, True), (3 * 8192, False)):
            for got in (call(state(**kw, dst=(1 << 30) + off)), call(state(**kw), state(**kw, src=1 << 31, dst=(1 << 40) + off))):
                assert (NO_PIPELINE[1] in got[1]) == ok and (ok or got[0] == capi.ERR_ARG and "overlap" in got[1]), (kw, off, got)
    for kw in (dict(idx=(1 << 40) + 64), dict(idx=(1 << 40) - 28), dict(lengths=(1 << 40) + 4096 * 8 - 4)):
        assert call(state(), **kw)[0] == capi.ERR_ARG and "lengths" in capi.last_error()
    assert NO_PIPELINE[1] in call(state(), idx=(1 << 40) - 32, lengths=(1 << 40) + 8 * 4096)[1]

    def columns(name, stores, rws, at=1 << 23):
        return status(name, None, len(stores), (QuantisedRowsStruct * len(stores))(*stores), (RowsStruct * len(rws))(*rws), at, 4)

    two = [store(), store(codes=1 << 26, scales=1 << 27)]
    take, put = "agpu_take_quantised", "agpu_put_quantised"
    assert NO_PIPELINE[1] in columns(take, two, [rows(), rows(data=(1 << 22) + 1024)])[1]                # 4 rows of 256 bytes, one behind the other
    assert NO_PIPELINE[1] in columns(take, two, [rows(row_stride=256), rows(row_stride=256, data=(1 << 22) + 256)])[1]  # beside each other in wider rows
    assert columns(take, two, [rows(), rows()])[0] == capi.ERR_ARG and "two columns" in capi.last_error()
    assert columns(take, two, [rows(), rows(data=(1 << 22) + 1022)])[0] == capi.ERR_ARG
    assert NO_PIPELINE[1] in columns(put, two, [rows(), rows()])[1]                                      # read twice
    for at in (1 << 20, (1 << 20) + 1022, (1 << 21) + 60, (1 << 23) + 8, (1 << 26)):
        assert columns(take, two, [rows(), rows(data=at)])[0] == capi.ERR_ARG and "cache or the slots" in capi.last_error(), at
    assert NO_PIPELINE[1] in columns(take, two, [rows(), rows(data=(1 << 20) + 1024)])[1]
    assert NO_PIPELINE[1] in columns(take, [store(), store()], [rows(), rows(data=1 << 25)])[1]          # one cache read twice
    for kw in ({}, dict(codes=(1 << 20) + 1023), dict(codes=(1 << 21) + 32), dict(scales=(1 << 20) + 4, codes=1 << 26)):
        assert columns(put, [store(), store(**kw)], [rows(), rows()])[0] == capi.ERR_ARG and "one cache" in capi.last_error()
    pages = PageMapStruct(1 << 24, 4, 1 << 25, 1 << 28, 3, 4, 16)
    for at, ok in ((1 << 24, False), ((1 << 24) + 44, False), ((1 << 24) + 48, True), ((1 << 25) + 12, False), ((1 << 25) + 16, True), ((1 << 28) + 8, False)):
        st, msg = status("agpu_take_quantised_pages", None, 1, C.byref(store()), C.byref(rows(data=at)), C.byref(pages), 4)
        assert (NO_PIPELINE[1] in msg) == ok and (ok or st == capi.ERR_ARG), (at, msg)
    assert "address space" in status("agpu_take_quantised", None, 1, C.byref(store()), C.byref(rows(row_stride=1 << 62)), 1 << 23, 4)[1]


# ---------------------------------------------------------------------------------------------------------- the Python host
class _Device:
    ordinal = 0
    _handle = None


def _host():
    import arrow_gpu_amd as ag

    dev = _Device()
    buf = lambda n: ag.DeviceBuffer(dev, 4096, n, owned=False)  # noqa: E731
    pipe = types.SimpleNamespace(device=dev, _handle=None, keep=lambda *a: None)
    return ag, dev, buf, pipe


def test_the_python_host_packs_the_structs_as_the_header_has_them():
    ag, dev, buf, _ = _host()
    import arrow_gpu_amd.kernels.rows as K

    r = ag.RowsGPU(buf(1), dev, (3, 2, 8), "bf16", (40, 16, 1), 4100)
    assert bytes(RowsStruct(4100, 40, 16, capi.ROW_BF16)) == r.as_rows()
    c = ag.QuantisedRowsGPU(buf(1), ag.DeviceBuffer(dev, 8192, 1, owned=False), dev, 5, 2, 8, 4, "i4")
    assert bytes(QuantisedRowsStruct(4096, 8192, 5, 2, 8, 4, capi.CODE_I4)) == c.packed
    idx = ag.UInt32ArrayGPU(buf(16), dev, 4, None)
    m = ag.PageMap(ag.RowsGPU(buf(1), dev, (3, 2), "u32", (7, 1)), 16, idx)
    assert bytes(PageMapStruct(4096, 7, 4096, None, 3, 2, 16)) == m.packed
    assert C.sizeof(StateStruct) == K._PACK_STATE.size and C.sizeof(BeamsStruct) == K._PACK_BEAMS.size
    v = tuple(range(1, 18))
    assert bytes(BeamsStruct(*v)) == K._PACK_BEAMS.pack(*v) and bytes(StateStruct(*v[:9])) == K._PACK_STATE.pack(*v[:9])
    state = ag.RowsGPU(buf(1), dev, (3, 2, 5, 4), "f16", (100, 30, 4, 1))
    assert state.as_pieces() == (200, 60, 2, 40, 8)                                       # pieces of 5 positions of 8 bytes
    assert ag.RowsGPU(buf(1), dev, (3, 5, 4), "f16").as_pieces() == (40, 0, 1, 40, 8)     # one piece
    assert ag.RowsGPU(buf(1), dev, (3, 5, 4), "f16", (50, 8, 1)).as_pieces() == (100, 16, 5, 8, 0)
    assert ag.RowsGPU(buf(1), dev, (3, 7), "u8").as_pieces() == (7, 0, 1, 7, 0)


def test_rows_past_their_buffer_are_refused():
    ag, dev, _, _ = _host()
    dev._handle = None
    own = lambda n: ag.DeviceBuffer(dev, 4096, n)  # noqa: E731
    for make in (lambda n: ag.RowsGPU(own(n), dev, (3, 2, 8), "bf16", (40, 16, 1), 4100), lambda n: ag.QuantisedRowsGPU(own(n - 132), own(80), dev, 5, 2, 8, 4, "i8"),
                 lambda n: ag.QuantisedRowsGPU(own(80), own(n - 132), dev, 5, 2, 8, 4, "i8")):
        make(4 + 2 * (2 * 40 + 16 + 8))
        with pytest.raises(ag.ArrowErrorGPU) as e:
            make(4 + 2 * (2 * 40 + 16 + 8) - 1)
        assert e.value.status == capi.ERR_SHAPE
    with pytest.raises(ag.ArrowErrorGPU):
        ag.RowsGPU(own(4096), dev, (3, 8), "f32", None, 4092)
    ag.RowsGPU(own(1), dev, (0, 8), "f32")


def test_python_refusals():
    ag, dev, buf, pipe = _host()
    idx = lambda n: ag.UInt32ArrayGPU(buf(4 * n), dev, n, None)  # noqa: E731
    view = lambda shape, t="f32", strides=None: ag.RowsGPU(buf(1), dev, shape, t, strides)  # noqa: E731
    cache = lambda **kw: ag.QuantisedRowsGPU(buf(1), buf(1), dev, **{**dict(n_slots=4, heads=2, dim=8, group=4, code="i8"), **kw})  # noqa: E731
    for bad in (lambda: view((3,)), lambda: view((1, 2, 3, 4, 5)), lambda: view((2, 2), strides=(1, 2)), lambda: view((2, 2), strides=(-2, 1)),
                lambda: cache(group=3), lambda: cache(dim=6, group=3, code="i4"), lambda: cache(heads=0),
                lambda: ag.put_quantised_op(cache(), view((3, 2, 8)), idx(4), pipe), lambda: ag.put_quantised_op(cache(), view((3, 16)), idx(3), pipe),
                lambda: ag.put_quantised_op([cache(), cache()], [view((3, 2, 8))], idx(3), pipe),
                lambda: ag.put_quantised_op([cache(), cache()], [view((3, 2, 8)), view((4, 2, 8))], idx(3), pipe),
                lambda: ag.take_quantised_op(cache(), idx(3), pipe, out=view((4, 2, 8))), lambda: ag.put_quantised_op([cache()] * 65, [view((3, 2, 8))] * 65, idx(3), pipe),
                lambda: ag.PageMap(view((3, 2), "u32"), 4, idx(3)), lambda: ag.PageMap(view((3, 2), "u32"), 0, idx(4)), lambda: ag.PageMap(view((3, 2)), 4, idx(4)),
                lambda: ag.PageMap(view((3, 2), "u32"), 4, idx(4), idx(4)),
                lambda: ag.take_quantised_op(cache(), ag.PageMap(view((3, 2), "u32"), 4, idx(4)), pipe),
                lambda: ag.take_rows_op(view((3, 4)), idx(3), pipe, lengths=idx(3), out=view((3, 4))), lambda: ag.take_rows_op(view((3, 2, 4)), idx(3), pipe, lengths=idx(2), out=view((3, 2, 4))),
                lambda: ag.take_rows_op(view((3, 4)), idx(3), pipe, out=view((2, 4))), lambda: ag.take_rows_op([view((3, 4)), view((2, 4))], idx(3), pipe, out=[view((3, 4))] * 2),
                lambda: ag.take_rows_op(view((3, 4)), idx(3), pipe, out=view((3, 4), "f16")),
                lambda: ag.take_rows_op(view((3, 2, 5, 4), strides=(100, 50, 8, 1)), idx(3), pipe, out=view((3, 2, 5, 4))),
                lambda: ag.take_rows_op(view((3, 5, 4), strides=(100, 8, 1)), idx(3), pipe, lengths=idx(3), out=view((3, 5, 4))),
                lambda: ag.select_beams_op(view((7, 10)), 2, 4, pipe), lambda: ag.select_beams_op(view((6, 10)), 2, 0, pipe), lambda: ag.select_beams_op(view((6, 10)), 2, 65, pipe),
                lambda: ag.select_beams_op(view((6, 10)), 2, 21, pipe), lambda: ag.select_beams_op(view((6, 10)), 2, 4, pipe, end_token=10),
                lambda: ag.select_beams_op(view((6, 10)), 2, 4, pipe, scores=ag.Float32ArrayGPU(buf(4), dev, 5, None)),
                lambda: ag.select_beams_op(view((6, 10)), 2, 4, pipe, allowed=ag.BooleanArrayGPU(buf(8), dev, 60, None)),
                lambda: ag.select_beams_op(view((6, 10)), 2, 4, pipe, finished=ag.BooleanArrayGPU(buf(8), dev, 64, None)),
                lambda: ag.select_beams_op(view((6, 10)), 2, 4, pipe, out=ag.BeamSelection(*[t(buf(4), dev, 9, None) for t in (ag.Float32ArrayGPU, ag.UInt32ArrayGPU, ag.UInt32ArrayGPU)], dev, 3, 3))):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            bad()
        assert e.value.status == capi.ERR_SHAPE, e.value
    for bad in (lambda: view((2, 2), "c64"), lambda: cache(code="i5"), lambda: ag.put_quantised_op(cache(), view((3, 2, 8), "i32"), idx(3), pipe),
                lambda: ag.take_rows_op(view((3, 4)), ag.Int32ArrayGPU(buf(12), dev, 3, None), pipe), lambda: ag.select_beams_op(view((6, 10), "i32"), 2, 4, pipe)):
        with pytest.raises(ag.OperationNotSupported):
            bad()
    other = _Device()
    other.ordinal = 1
    with pytest.raises(ag.ArrowErrorGPU) as e:  # memory of another GPU
        ag.take_rows_op(ag.RowsGPU(buf(1), other, (3, 4), "f32"), idx(3), pipe, out=view((3, 4)))
    assert e.value.status == capi.ERR_ARG


def test_python_refusals_of_sizes_and_types(monkeypatch):
    """what no field of a struct holds, and index columns of another type or with nulls: an error of this library's, before anything is packed"""
    ag, dev, buf, pipe = _host()
    u32 = lambda n: ag.UInt32ArrayGPU(buf(4 * n), dev, n, None)  # noqa: E731
    nulls = ag.UInt32ArrayGPU(buf(16), dev, 4, object())
    view = lambda shape, t="f32", strides=None: ag.RowsGPU(buf(1), dev, shape, t, strides)  # noqa: E731
    cache = lambda **kw: ag.QuantisedRowsGPU(buf(1), buf(1), dev, **{**dict(n_slots=4, heads=2, dim=8, group=4, code="i8"), **kw})  # noqa: E731
    tables = view((3, 2), "u32")
    for bad in (lambda: cache(n_slots=-1), lambda: cache(n_slots=(1 << 32) + 1), lambda: cache(heads=1 << 33, dim=4), lambda: cache(heads=1, dim=1 << 17, group=1 << 17),
                lambda: ag.QuantisedRowsGPU.empty(-1, 2, 8, dev), lambda: ag.QuantisedRowsGPU.empty(4, 0, 8, dev), lambda: ag.QuantisedRowsGPU.empty(4, 2, 8, dev, group=3),
                lambda: ag.QuantisedRowsGPU.empty(4, 2, 8, dev, group=0), lambda: view((-1, 4)), lambda: view((3, -4)), lambda: ag.RowsGPU.of_array(u32(4), (-1, -4)),
                lambda: ag.PageMap(tables, 1 << 32, u32(4)), lambda: ag.PageMap(tables, -1, u32(4)),
                lambda: ag.take_quantised_op(cache(), ag.PageMap(tables, 4, u32(4)), pipe, n_rows=-1),
                lambda: ag.select_beams_op(view((1, 1 << 33)), 1, 4, pipe), lambda: ag.select_beams_op(view((1 << 24, 4)), 1, 4, pipe)):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            bad()
        assert e.value.status == capi.ERR_SHAPE, e.value
    f32 = ag.Float32ArrayGPU(buf(16), dev, 4, None)
    for bad in (lambda: ag.PageMap(tables, 4, f32), lambda: ag.PageMap(tables, 4, nulls), lambda: ag.PageMap(tables, 4, u32(4), ag.Int32ArrayGPU(buf(12), dev, 3, None)),
                lambda: ag.put_quantised(cache(), view((4, 2, 8)), f32), lambda: ag.take_quantised(cache(), nulls)):
        with pytest.raises(ag.OperationNotSupported):
            bad()
    ag.PageMap(tables, (1 << 32) - 1, u32(4), u32(3))
    # no caches at all is a call that does nothing, on the index column's device
    import arrow_gpu_amd.kernels.rows as K

    asked = []
    done = types.SimpleNamespace(device=dev, _handle=None, keep=lambda *a: None, own_stream=True, finish=lambda: None, sync=lambda: None)
    monkeypatch.setattr(K, "pipeline_for", lambda device, *a: asked.append(device) or done)
    ag.put_quantised([], [], u32(3))
    assert ag.take_quantised([], u32(3)) == [] and ag.take_quantised([], ag.PageMap(tables, 4, u32(4)), n_rows=3) == [] and asked == [dev] * 3


def test_positions_that_lie_apart_go_into_dense_rows_and_back(monkeypatch):
    """(rows, positions, values): each position is a piece, in the state and in the output, whichever of the two is dense"""
    import arrow_gpu_amd.kernels.rows as K

    ag, dev, buf, _ = _host()
    pipe = types.SimpleNamespace(device=dev, _handle=None, keep=lambda *a: None, own_stream=True)
    called = []
    monkeypatch.setattr(K.capi, "call", lambda *a: called.append(a))
    idx = ag.UInt32ArrayGPU(buf(12), dev, 3, None)
    apart = ag.RowsGPU(buf(1), dev, (3, 5, 4), "f16", (100, 8, 1))
    dense = ag.RowsGPU(ag.DeviceBuffer(dev, 8192, 1, owned=False), dev, (3, 5, 4), "f16")
    for s, o, want in ((apart, dense, (4096, 8192, 200, 16, 40, 8, 5, 8, 0)), (dense, apart, (8192, 4096, 40, 8, 200, 16, 5, 8, 0)),
                       (apart, apart, (4096, 4096, 200, 16, 200, 16, 5, 8, 0)), (dense, dense, (8192, 8192, 40, 0, 40, 0, 1, 40, 8))):
        assert K.take_rows_op(s, idx, pipe, out=o) == [o]
        assert called.pop()[3] == bytes(StateStruct(*want))
        if s is not o or s is apart:
            with pytest.raises(ag.ArrowErrorGPU) as e:
                K.take_rows_op(s, idx, pipe, lengths=idx, out=o)
            assert e.value.status == capi.ERR_SHAPE and not called


# ------------------------------------------------------------------------------------------------- slots, broken tables too
SRC = r"""
#include "%s/arrow_gpu_amd/csrc/row_address.hpp"
extern "C" void slots(const uint32_t* slot_column, const uint32_t* tables, uint64_t stride, const uint32_t* offsets, const uint32_t* first, uint32_t n_seqs,
                      uint32_t max_pages, uint32_t page_rows, uint64_t n, uint64_t n_slots, int64_t* out) {
  const RowAddr a = {slot_column, tables, stride, offsets, first, n_seqs, max_pages, page_rows};
  for (uint64_t i = 0; i < n; i++) out[i] = (int64_t)row_slot(a, i, n_slots);
}
"""


DIVIDE = r"""
extern "C" uint32_t divide(uint32_t d) {  // the first x from 0, or around the multiples of d and 2^31, whose quotient is wrong; 0xFFFFFFFF: none
  const Divide by = divide_by(d);
  const auto wrong = [&](uint64_t x) { return x < (1ull << 31) && (uint32_t)x / by != (uint32_t)x / d; };
  for (uint32_t x = 0; x < 5000; x++)
    if (wrong(x)) return x;
  for (uint64_t k = 1; k < 4000; k++)
    for (int64_t o = -2; o <= 2; o++) {
      const uint64_t near = (uint64_t)((int64_t)(k * d) + o), far = (((1ull << 31) - 1) / d - k + 1) * d + o;
      if (wrong(near)) return (uint32_t)near;
      if (k <= ((1ull << 31) - 1) / d && wrong(far)) return (uint32_t)far;
    }
  return 0xFFFFFFFFu;
}
"""


APART = r"""
extern "C" int overlap(const uint64_t* a, const uint64_t* b) {  // at, n, row stride, m, part stride, size
  Places p[2] = {{a[0], a[1], a[2], a[3], a[4], a[5], true, 0}, {b[0], b[1], b[2], b[3], b[4], b[5], false, 1}};
  uint32_t x, y;
  return overlapping(p, 2, &x, &y);
}
"""


@pytest.fixture(scope="module")
def slots_lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("rows")
    (d / "s.cpp").write_text(SRC % ROOT + DIVIDE + APART)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", str(d / "s.so"), str(d / "s.cpp")], check=True, timeout=120)
    return C.CDLL(str(d / "s.so"))


def _slots(lib, n, n_slots, column=None, tables=None, offsets=None, first=None, page_rows=1):
    ptr = lambda a: a.ctypes.data_as(C.c_void_p) if a is not None else None  # noqa: E731
    got = np.zeros(n, np.int64)
    lib.slots(ptr(column), ptr(tables), C.c_uint64(tables.shape[1] if tables is not None else 0), ptr(offsets), ptr(first), C.c_uint32(len(offsets) - 1 if offsets is not None else 0),
              C.c_uint32(tables.shape[1] if tables is not None else 0), C.c_uint32(page_rows), C.c_uint64(n), C.c_uint64(n_slots), ptr(got))
    return got


def test_quotients_by_products(slots_lib):
    slots_lib.divide.restype = C.c_uint32
    rng = np.random.default_rng(0)
    for d in [*range(1, 300), *(1 << np.arange(31)).tolist(), *((1 << np.arange(2, 31)) - 1).tolist(), *((1 << np.arange(30)) + 1).tolist(), *rng.integers(1, 1 << 31, 200).tolist(), (1 << 31) - 1]:
        assert slots_lib.divide(C.c_uint32(int(d))) == 0xFFFFFFFF, d


def test_places_that_are_called_apart_share_no_byte(slots_lib):
    """against the sets of their bytes, for random strides; and rows, parts or both within a common stride are found apart"""
    rng = np.random.default_rng(0)

    def bytes_of(at, n, row, m, part, size):
        return {at + i * row + j * part + k for i in range(n) for j in range(m) for k in range(size)}

    def overlap(a, b):
        return slots_lib.overlap((C.c_uint64 * 6)(*a), (C.c_uint64 * 6)(*b)) != 0

    apart = meet = 0
    for _ in range(20000):
        strides = rng.integers(0, 40, 3).tolist()
        some = lambda: [int(rng.integers(0, 120)), int(rng.integers(1, 5)), int(rng.choice(strides)) * int(rng.integers(1, 4)), int(rng.integers(1, 4)),  # noqa: E731, B023
                        int(rng.choice(strides)), int(rng.integers(1, 12))]
        a, b = some(), some()
        if not overlap(a, b):
            assert not bytes_of(*a) & bytes_of(*b), (a, b)
            apart += 1
        else:
            meet += bool(bytes_of(*a) & bytes_of(*b))
    assert apart > 5000 and meet > 2000
    for _ in range(3000):  # [n, m, 2, size] or [n, 2, m, size] or [m, n, 2, size], gaps behind any
        size, n, m = (int(v) for v in rng.integers(1, 6, 3))
        first, gap = int(rng.integers(0, 50)), int(rng.integers(0, 3))
        part = 2 * size + gap
        row = m * part + int(rng.integers(0, 3)) * part
        assert not overlap((first, n, row, m, part, size), (first + size, n, row, m, part, size))
        row = 2 * m * size + gap
        assert not overlap((first + m * size, n, row, m, size, size), (first, n, row, m, size, size))
        assert not overlap((first + size, n, part, m, part * n, size), (first, n + 2, part, m, part * n, size))
        row = m * part + int(rng.integers(0, 9))  # no multiple of the parts' stride
        a, b = (first, n, row, m, part, size), (first + size, n, row, m, part, size)
        assert not overlap(a, b) and not overlap(b, a)


def test_slots_of_a_column(slots_lib):
    c = np.array([0, 7, 8, R.NO_ROW, 0xFFFFFFFE, 3], np.uint32)
    assert _slots(slots_lib, 6, 8, c).tolist() == [0, 7, -2, -1, -2, 3]
    assert _slots(slots_lib, 6, 1 << 32, c).tolist() == [0, 7, 8, -1, 0xFFFFFFFE, 3]
    assert _slots(slots_lib, 6, 0, c).tolist() == [-2, -2, -2, -1, -2, -2]


@pytest.mark.parametrize("seed", range(30))
def test_slots_of_pages(slots_lib, seed):
    rng = np.random.default_rng(seed)
    seqs, page = int(rng.integers(1, 20)), int(rng.choice([1, 2, 5, 16, 1000]))
    lens = rng.integers(0, 40, seqs) * (rng.random(seqs) < 0.7)
    offsets = (int(rng.integers(0, 4)) + np.concatenate([[0], np.cumsum(lens)])).astype(np.uint32)
    first = rng.integers(0, 50, seqs).astype(np.uint32) if seed % 2 else None
    tables = rng.integers(0, 60, (seqs, int(rng.integers(1, 30)))).astype(np.uint32)
    tables[rng.random(tables.shape) < 0.1] = R.NO_ROW
    tables[rng.random(tables.shape) < 0.05] = 0xFFFFFFFE
    n = int(offsets[-1]) + 5
    assert np.array_equal(_slots(slots_lib, n, 50 * page, None, tables, offsets, first, page), R.slots_of(tables, page, offsets, n, 50 * page, first))


@pytest.mark.parametrize("seed", range(30))
def test_broken_offsets_stay_inside_the_tables(slots_lib, seed):
    """offsets in any order: every answer is a slot of the cache, none, or out of range — and no table is read past its end (the tables end in front
    of a guard that would give a slot of its own)"""
    rng = np.random.default_rng(seed)
    seqs, most, page = int(rng.integers(1, 12)), int(rng.integers(1, 6)), int(rng.integers(1, 9))
    tables = np.zeros((seqs + 1, most), np.uint32)
    tables[:seqs] = rng.integers(0, 9, (seqs, most))
    tables[seqs] = 10  # the guard: slots 10 * page and up
    offsets = rng.integers(0, 30, seqs + 1).astype(np.uint32)
    first = rng.choice(np.array([0, 1, 7, 0xFFFFFFFF], np.uint32), seqs)
    got = _slots(slots_lib, 40, 20 * page, None, tables[:seqs], offsets, first, page)
    assert ((got >= -2) & (got < 10 * page)).all()


def test_the_reference_agrees_with_torch():
    """rows_ref's 8-bit type and quantiser against torch's conversion and a formula written apart"""
    torch = pytest.importorskip("torch")
    v = R.e4m3_values()
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v[~np.isnan(v)], t[~np.isnan(t)]) and np.array_equal(np.isnan(v), np.isnan(t))
    x = np.concatenate([np.random.default_rng(0).uniform(-448, 448, 20000), np.random.default_rng(1).normal(0, 0.02, 20000), (v[:126] + v[1:127]) / 2, v[:127], -v[:127]]).astype(np.float32)
    got = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.to_e4m3(x) & 127, got & 127)
    y = np.random.default_rng(2).standard_normal((3, 2, 8)).astype(np.float32)
    c, s = R.quantise(y, "i8", 4)
    a = np.abs(y.reshape(3, 2, 2, 4)).max(-1)
    assert np.array_equal(s, a / np.float32(127)) and np.abs(R.values(c, s, "i8", 4) - y).max() <= a.max() / 127 * 0.5001


def test_the_reference_selection_agrees_with_torch():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).standard_normal((6, 40))
    cum = np.random.default_rng(1).standard_normal(6).astype(np.float32)
    s, r, t = R.select(x, 3, 5, cum)
    z = (torch.log_softmax(torch.from_numpy(x), -1) + torch.from_numpy(cum).double()[:, None]).reshape(2, -1)
    v, i = torch.topk(z, 5)
    assert np.allclose(s, v.numpy(), rtol=1e-13, atol=1e-13)
    assert np.array_equal(r, (i // 40).numpy() + np.array([[0], [3]])) and np.array_equal(t, (i % 40).numpy())

"""CPU: which stream a call runs on that takes no pipeline.  Over a tensor's memory it is torch's current one — a stream of the library's own is ordered with
none of torch's, and the call would read what is still being written — and otherwise one of its own."""
import sys
import types

import pytest

import arrow_gpu_amd as ag
from arrow_gpu_amd import gpu_utils


class Made(Exception):
    pass


class Device:
    ordinal = 3
    _handle = None


class Tensor:
    """what borrow_tensor asks of one"""

    def __init__(self, dtype, shape, item):
        self.dtype, self.shape, self.item, self.device, self.requires_grad = dtype, shape, item, "gpu", False

    def get_device(self):
        return 3

    def data_ptr(self):
        return 4096

    def numel(self):
        n = 1
        for d in self.shape:
            n *= d
        return n

    def element_size(self):
        return self.item

    def is_contiguous(self):
        return True

    def stride(self):
        at, got = 1, []
        for d in reversed(self.shape):
            got.append(at)
            at *= d
        return tuple(reversed(got))


DEV = Device()
FLOATS = lambda n, lent: (ag.Float32ArrayGPU.of_tensor(Tensor("torch.float32", (n,), 4), DEV) if lent else ag.Float32ArrayGPU(ag.DeviceBuffer(DEV, 4096, 4 * n, owned=False), DEV, n, None))  # noqa: E731
INDEX = lambda n, lent: (ag.UInt32ArrayGPU.of_tensor(Tensor("torch.int32", (n,), 4), DEV) if lent else ag.UInt32ArrayGPU(ag.DeviceBuffer(DEV, 4096, 4 * n, owned=False), DEV, n, None))  # noqa: E731
BITS = lambda n, lent: (ag.BooleanArrayGPU.of_tensor(Tensor("torch.uint8", (-(-n // 64) * 8,), 1), DEV, n) if lent else ag.BooleanArrayGPU(ag.DeviceBuffer(DEV, 4096, -(-n // 64) * 8, owned=False), DEV, n, None))  # noqa: E731
ROWS = lambda shape, lent: (ag.RowsGPU.of_tensor(Tensor("torch.float32", shape, 4), DEV) if lent else ag.RowsGPU(ag.DeviceBuffer(DEV, 4096, 1, owned=False), DEV, shape, "f32"))  # noqa: E731


def CACHE(lent):
    if lent:
        return ag.QuantisedRowsGPU.of_tensors(Tensor("torch.uint8", (4, 2, 8), 1), Tensor("torch.float32", (4, 2, 2), 4), DEV, code="i8", heads=2, dim=8, group=4)
    return ag.QuantisedRowsGPU(ag.DeviceBuffer(DEV, 4096, 64, owned=False), ag.DeviceBuffer(DEV, 4096, 64, owned=False), DEV, 4, 2, 8, 4, "i8")


def SELECTION(lent):
    return ag.BeamSelection(*[(FLOATS if i == 0 else INDEX)(4, lent) for i in range(3)], DEV, 2, 2)


def PAGES(*lent):
    i32 = lambda shape, b: ag.RowsGPU.of_tensor(Tensor("torch.int32", shape, 4), DEV) if b else ag.RowsGPU(ag.DeviceBuffer(DEV, 4096, 1, owned=False), DEV, shape, "u32")  # noqa: E731
    return ag.PageMap(i32((2, 2), lent[0]), 1, INDEX(3, lent[1]), INDEX(2, lent[2]))


# call(which): argument `which` lies in a tensor's memory; -1: none
CALLS = {
    "put_quantised": (3, lambda w: ag.put_quantised([CACHE(w == 0)], [ROWS((3, 2, 8), w == 1)], INDEX(3, w == 2))),
    "put_quantised pages": (3, lambda w: ag.put_quantised(CACHE(False), ROWS((3, 2, 8), False), PAGES(w == 0, w == 1, w == 2))),
    "take_quantised": (3, lambda w: ag.take_quantised(CACHE(w == 0), INDEX(3, w == 1), out=ROWS((3, 2, 8), w == 2))),
    "take_rows": (4, lambda w: ag.take_rows([ROWS((3, 5, 2), w == 0)], INDEX(3, w == 1), INDEX(3, w == 2), out=[ROWS((3, 5, 2), w == 3)])),
    "select_beams": (5, lambda w: ag.select_beams(ROWS((4, 64), w == 0), 2, 2, FLOATS(4, w == 1), BITS(64, w == 2), BITS(4, w == 3), out=SELECTION(w == 4))),
    "add": (2, lambda w: FLOATS(9, w == 0).add(FLOATS(9, w == 1))),
    "add_dyn": (2, lambda w: ag.add_dyn(FLOATS(9, w == 0), FLOATS(9, w == 1))),
    "sub_array_dyn": (2, lambda w: ag.sub_array_dyn(FLOATS(9, w == 0), FLOATS(9, w == 1))),
    "sin_dyn": (1, lambda w: ag.sin_dyn(FLOATS(9, w == 0))),
    "sum": (1, lambda w: FLOATS(9, w == 0).sum()),
    "cast": (1, lambda w: FLOATS(9, w == 0).cast(ag.UInt8ArrayGPU)),
    "bitcast_dyn": (1, lambda w: ag.bitcast_dyn(FLOATS(9, w == 0), ag.ArrowType.UInt32Type)),
    "take": (2, lambda w: FLOATS(9, w == 0).take(INDEX(4, w == 1))),
    "take_dyn": (2, lambda w: ag.take_dyn(FLOATS(9, w == 0), INDEX(4, w == 1))),
    "take_columns": (3, lambda w: ag.take_columns([FLOATS(9, w == 0), FLOATS(9, w == 1)], INDEX(4, w == 2))),
    "put": (4, lambda w: FLOATS(9, w == 0).put(INDEX(4, w == 1), FLOATS(9, w == 2), INDEX(4, w == 3))),
    "put_dyn": (4, lambda w: ag.put_dyn(FLOATS(9, w == 0), INDEX(4, w == 1), FLOATS(9, w == 2), INDEX(4, w == 3))),
    "merge_dyn": (3, lambda w: ag.merge_dyn(FLOATS(9, w == 0), FLOATS(9, w == 1), BITS(9, w == 2))),
    "any": (1, lambda w: BITS(9, w == 0).any()),
    "all": (1, lambda w: BITS(9, w == 0).all()),
    "count_set_bits": (1, lambda w: BITS(9, w == 0).count_set_bits()),
    "clone_buffer": (1, lambda w: ag.GpuDevice.clone_buffer(DEV, FLOATS(9, True).data)),
}


@pytest.mark.parametrize("name", CALLS)
def test_calls_over_tensors_run_on_torchs_stream(monkeypatch, name):
    made = []

    def make(device, label=None, hip_stream=None, fuse=None):
        made.append(hip_stream)
        raise Made

    asked = []
    fake = types.SimpleNamespace(cuda=types.SimpleNamespace(is_initialized=lambda: True, is_current_stream_capturing=lambda: False, current_stream=lambda ordinal: (asked.append(ordinal), types.SimpleNamespace(cuda_stream=0))[1]))
    monkeypatch.setitem(sys.modules, "torch", fake)
    monkeypatch.setattr(gpu_utils, "ArrowComputePipeline", make)
    arguments, call = CALLS[name]
    for which in range(arguments):
        with pytest.raises(Made):
            call(which)
        assert made.pop() == 0 and not made and asked.pop() == 3, which  # torch's default stream is the handle 0
    if name != "clone_buffer":
        with pytest.raises(Made):
            call(-1)
        assert made.pop() is None and not made and not asked


def test_fused_chains_over_tensors_run_on_torchs_stream(monkeypatch):
    made = []

    def make(device, label=None, hip_stream=None, fuse=None):
        made.append(hip_stream)
        raise Made

    monkeypatch.setitem(sys.modules, "torch", types.SimpleNamespace(cuda=types.SimpleNamespace(is_initialized=lambda: True, is_current_stream_capturing=lambda: False, current_stream=lambda o: types.SimpleNamespace(cuda_stream=5))))
    monkeypatch.setattr(gpu_utils, "ArrowComputePipeline", make)
    for head, step, other in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        chain = ag.FusedChain(FLOATS(9, head)).add(FLOATS(9, step))
        with pytest.raises(Made):
            chain.gt(FLOATS(9, other))
        assert made.pop() == (5 if head or step or other else None)
        with pytest.raises(Made):
            chain.finish()
        assert made.pop() == (5 if head or step else None)


def test_reading_back_waits_for_torchs_stream(monkeypatch):
    waited = []
    fake = types.SimpleNamespace(cuda=types.SimpleNamespace(is_initialized=lambda: True, is_current_stream_capturing=lambda: False, current_stream=lambda o: types.SimpleNamespace(cuda_stream=5, synchronize=lambda: waited.append(o))))
    monkeypatch.setitem(sys.modules, "torch", fake)

    def download(*a, **k):
        raise Made

    monkeypatch.setattr(gpu_utils.capi, "call", download)
    device = Device()
    device.retrive_data = lambda *a: gpu_utils.GpuDevice.retrive_data(device, *a)
    device.sync = download
    for thing in (FLOATS(9, True), BITS(9, True), FLOATS(9000, True), ROWS((3, 4), True)):
        thing.gpu_device = device
        with pytest.raises(Made):
            thing.values()
        assert waited.pop() == 3 and not waited
    mine = FLOATS(9, False)
    mine.gpu_device = device
    with pytest.raises(Made):
        mine.values()
    assert not waited


@pytest.mark.parametrize("own_stream", [True, False])
def test_a_pipeline_of_its_own_holds_the_tensors_of_its_calls(monkeypatch, own_stream):
    """their memory would otherwise go back to torch while a kernel on a stream that torch does not know still uses it; torch's own stream keeps its order"""
    import arrow_gpu_amd.kernels.rows as K

    kept = []
    monkeypatch.setattr(K.capi, "call", lambda *a: None)
    pipe = types.SimpleNamespace(device=DEV, _handle=None, keep=lambda *b: kept.extend(b), own_stream=own_stream)
    cache, rows, index, pages = CACHE(True), ROWS((3, 2, 8), True), INDEX(3, True), PAGES(True, True, True)
    state, out, parents, lengths = ROWS((3, 5, 2), True), ROWS((3, 5, 2), True), INDEX(3, True), INDEX(3, True)
    logits, scores, mask, sel = ROWS((4, 64), True), FLOATS(4, True), BITS(64, True), SELECTION(True)
    sel.workspace, sel._workspace_of = ag.DeviceBuffer(DEV, 4096, 1 << 20, owned=False), (2, 64)
    for call, things in ((lambda: ag.put_quantised_op(cache, rows, index, pipe), (cache.codes, cache.scales, rows.data, index.data)),
                         (lambda: ag.take_quantised_op(cache, pages, pipe, out=rows), (cache.codes, cache.scales, rows.data, pages.tables.data, pages.offsets.data, pages.first.data)),
                         (lambda: ag.take_rows_op(state, parents, pipe, lengths=lengths, out=out), (state.data, out.data, parents.data, lengths.data)),
                         (lambda: ag.select_beams_op(logits, 2, 2, pipe, scores=scores, allowed=mask, out=sel),
                          (logits.data, scores.data, mask.data, sel.scores.data, sel.parents.data, sel.tokens.data))):
        call()
        lent = [b for b in kept if isinstance(b, gpu_utils.BorrowedBuffer)]
        assert {id(b) for b in lent} == ({id(b) for b in things} if own_stream else set())
        kept.clear()


def test_a_tensor_that_requires_gradients_is_refused():
    """its graph would end here without a word"""
    def made(dtype, shape, item):
        t = Tensor(dtype, shape, item)
        t.requires_grad = True
        return t

    plain = Tensor("torch.float32", (4, 2, 2), 4)
    for bad in (lambda: ag.RowsGPU.of_tensor(made("torch.float32", (3, 4), 4), DEV), lambda: ag.Float32ArrayGPU.of_tensor(made("torch.float32", (3,), 4), DEV),
                lambda: ag.QuantisedRowsGPU.of_tensors(Tensor("torch.uint8", (4, 2, 8), 1), made("torch.float32", (4, 2, 2), 4), DEV, code="i8", heads=2, dim=8, group=4)):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            bad()
        assert e.value.status == ag._capi.ERR_ARG and "detach" in str(e.value)
    ag.QuantisedRowsGPU.of_tensors(Tensor("torch.uint8", (4, 2, 8), 1), plain, DEV, code="i8", heads=2, dim=8, group=4)
    torch = pytest.importorskip("torch")
    for t in (torch.ones(3, 4, requires_grad=True), torch.ones(3, 4, requires_grad=True) * 2):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            ag.RowsGPU.of_tensor(t, DEV)
        assert "detach" in str(e.value)
    with pytest.raises(ag.ArrowErrorGPU) as e:
        ag.RowsGPU.of_tensor(torch.ones(3, 4, requires_grad=True).detach(), DEV)
    assert "GPU 3" in str(e.value)  # (a host tensor, the next complaint)


def test_a_tensor_of_truth_values_is_no_bitmap():
    """one a byte: read as packed bits it would be a mask of other rows, without an error"""
    for dtype, item in (("torch.bool", 1), ("torch.float8_e4m3fn", 1), ("torch.int32", 4)):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            ag.BooleanArrayGPU.of_tensor(Tensor(dtype, (64,), item), DEV, 64)
        assert e.value.status == ag._capi.ERR_ARG
    for dtype in ("torch.uint8", "torch.int8"):
        assert ag.BooleanArrayGPU.of_tensor(Tensor(dtype, (64,), 1), DEV).len == 512
        assert ag.BooleanArrayGPU.of_tensor(Tensor(dtype, (64,), 1), DEV, 100).len == 100
        for bits in (513, -1):
            with pytest.raises(ag.ArrowErrorGPU):
                ag.BooleanArrayGPU.of_tensor(Tensor(dtype, (64,), 1), DEV, bits)


def test_a_call_that_waits_is_refused_while_torch_captures(monkeypatch):
    fake = types.SimpleNamespace(cuda=types.SimpleNamespace(is_initialized=lambda: True, is_current_stream_capturing=lambda: True, current_stream=lambda o: 1 / 0))
    monkeypatch.setitem(sys.modules, "torch", fake)
    for call in (lambda: ag.take_quantised(CACHE(True), INDEX(3, True), out=ROWS((3, 2, 8), True)), lambda: FLOATS(9, True).add(FLOATS(9, False)),
                 lambda: gpu_utils.GpuDevice.retrive_data(DEV, FLOATS(9, True).data)):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            call()
        assert e.value.status == ag._capi.ERR_ARG and "captures" in str(e.value)


def test_tensors_of_another_library(monkeypatch):
    """torch not loaded, or loaded for the CPU alone: a pipeline of the call's own, and torch is not woken"""
    made = []

    def make(device, label=None, hip_stream=None, fuse=None):
        made.append(hip_stream)
        raise Made

    monkeypatch.setattr(gpu_utils, "ArrowComputePipeline", make)
    for torch in (None, types.SimpleNamespace(cuda=types.SimpleNamespace(is_initialized=lambda: False, current_stream=lambda o: 1 / 0, is_current_stream_capturing=lambda: 1 / 0))):
        monkeypatch.setitem(sys.modules, "torch", torch)
        with pytest.raises(Made):
            FLOATS(9, True).add(FLOATS(9, True))
        assert made.pop() is None
        gpu_utils.settle(DEV, FLOATS(9, True))

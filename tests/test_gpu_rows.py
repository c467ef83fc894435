"""GPU: operators on whole rows — the quantised cache (put_quantised, take_quantised, by slots and through page tables), take_rows and select_beams —
against their definitions in numpy (tests/rows_ref.py), and a run of them together as a beam search makes it."""
import ctypes as C

import numpy as np
import pytest

import rows_ref as R
from arrow_gpu_amd import _capi as capi

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]
CODES = ["i8", "i4", "e4m3"]


@pytest.fixture(scope="module")
def dev():
    import gc

    import arrow_gpu_amd as ag

    d = ag.GpuDevice(0)
    yield d
    gc.collect()  # what the tests past 32 bits reserved goes back for the modules behind this one
    capi.call("agpu_device_trim", d._handle)


@pytest.fixture()
def p(dev):
    import arrow_gpu_amd as ag

    return ag.ArrowComputePipeline(dev, "rows")


def u32(values, dev):
    import arrow_gpu_amd as ag

    return ag.UInt32ArrayGPU.from_slice(np.asarray(values, dtype=np.uint32), dev)


def bits(flags, dev):
    import arrow_gpu_amd as ag

    flags = np.asarray(flags, dtype=bool).reshape(-1)
    packed = np.zeros((len(flags) + 63) // 64 * 8, np.uint8)
    packed[:(len(flags) + 7) // 8] = np.packbits(flags, bitorder="little")
    return ag.BooleanArrayGPU(dev.create_gpu_buffer_with_data(packed), dev, len(flags), None)


def up(x, kind, dev):
    import arrow_gpu_amd as ag

    return ag.RowsGPU.from_numpy(x, dev, kind)


def stored(store, dev):
    """(codes, scales) of a cache on the host, in their layouts."""
    n, h, d, g = store.n_slots, store.heads, store.dim, store.group
    codes = dev.retrive_data(store.codes).reshape(-1)
    scales = dev.retrive_data(store.scales).view(np.float32)
    if store.code == "i4":
        return codes[:n * h * d // 2].reshape(n, h, d // 2), scales[:2 * n * h * d // g].reshape(n, h, d // g, 2)
    return codes[:n * h * d].reshape(n, h, d), scales[:n * h * d // g].reshape(n, h, d // g)


def assert_codes(got, want, code, scales):
    """Codes of groups whose scale is a number; a group that holds none reads back as NaN whatever its codes are."""
    ok = ~np.isnan(scales[..., 0] if code == "i4" else scales)
    n, h = got.shape[:2]
    g, w = got.reshape(n, h, ok.shape[2], -1)[ok], want.reshape(n, h, ok.shape[2], -1)[ok]
    if code == "e4m3":  # the sign of a zero is no value
        g, w = np.where(g == 128, 0, g), np.where(w == 128, 0, w)
    assert np.array_equal(g, w), (np.argwhere(g != w)[:4], g[g != w][:4], w[g != w][:4])


def assert_values(got, want64, kind):
    """One rounding to f32 and, for the 16-bit types, one more: at most half a step each."""
    assert np.array_equal(np.isnan(got), np.isnan(want64))
    top = {"f32": 3.4028235e38, "f16": 65504.0, "bf16": 3.3895314e38}[kind]
    fine = np.isfinite(want64) & (np.abs(want64) < top)
    tol = np.abs(want64) * (R.HALF_STEP["f32"] + (R.HALF_STEP[kind] if kind != "f32" else 0)) * (1 + 2.0**-10)
    tiny = {"f32": 2.0**-150, "f16": 2.0**-25, "bf16": 2.0**-134}[kind]  # half a step of the subnormal numbers
    off = np.abs(got.astype(np.float64) - want64)
    assert (off[fine] <= tol[fine] + tiny).all(), (off[fine] / np.abs(want64[fine])).max()


def activations(rng, shape, kind):
    x = rng.standard_normal(shape).astype(np.float32) * np.where(rng.random(shape[1:]) > 0.9, 9, 1).astype(np.float32)
    return R.rounded(x, kind)


SHAPES = [(1, 1, 2, 2), (1, 8, 128, 128), (3, 2, 6, 2), (65, 5, 80, 80), (33, 2, 96, 48), (130, 4, 64, 32), (17, 3, 256, 256), (9, 1, 576, 576), (7, 2, 1024, 1024),
          (2, 1, 2048, 2048), (21, 3, 24, 8), (300, 2, 128, 16), (11, 7, 36, 36), (1025, 1, 64, 64)]


@pytest.mark.parametrize("n,heads,dim,group", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("code", CODES)
def test_put_and_take(dev, p, code, kind, n, heads, dim, group):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(n * 131 + dim + group)
    x = activations(rng, (n, heads, dim), kind)
    slots = rng.permutation(n + 7)[:n]
    store = ag.QuantisedRowsGPU.empty(n + 7, heads, dim, dev, code=code, group=group)
    ag.put_quantised_op(store, up(x, kind, dev), u32(slots, dev), p)
    got = ag.take_quantised_op(store, u32(slots, dev), p, kind)[0]
    p.sync()
    codes, scales = stored(store, dev)
    want_codes, want_scales = R.quantise(x, code, group)
    assert np.array_equal(scales[slots].view(np.uint32), want_scales.view(np.uint32))
    assert_codes(codes[slots], want_codes, code, want_scales)
    left = np.setdiff1d(np.arange(n + 7), slots)
    assert not codes[left].any() and not scales[left].any()
    want = R.values(want_codes, want_scales, code, group)
    assert_values(got.values(), want, kind)
    # half a step of the group's scale (e4m3: of the value) off the input, and the rounding of what comes back
    scale = np.repeat((want_scales[..., 0] if code == "i4" else want_scales).astype(np.float64), group, axis=-1).reshape(x.shape)
    step = np.maximum(np.abs(x) * 2.0**-4, scale * 2.0**-10) if code == "e4m3" else scale / 2
    assert (np.abs(want - x) <= step * (1 + 2.0**-12) + np.abs(x) * 2.0**-21).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dim,group", [(64, 32), (40, 10)])
def test_groups_at_the_ends_of_the_range(dev, p, code, kind, dim, group):
    """zeros, one value alone, subnormals, the smallest live span, the largest values, NaN and infinities, minus zero"""
    import arrow_gpu_amd as ag

    big = {"f32": 3.0e38, "f16": 6.0e4, "bf16": 3.0e38}[kind]
    small = {"f32": 1.2e-38, "f16": 6e-8, "bf16": 1.2e-38}[kind]
    rng = np.random.default_rng(5)
    x = np.zeros((20, 2, dim), np.float32)
    x[1] = 3.25
    x[2] = -7.5
    x[3, :, 1] = -1.0
    x[4] = small * rng.standard_normal((2, dim))
    x[5] = 1e-36 * rng.standard_normal((2, dim)) if kind != "f16" else 1e-6
    x[6] = big * rng.uniform(0.5, 1, (2, dim))
    x[7] = big * rng.uniform(-1, 1, (2, dim))   # i4 in f32 / bf16: a span that overflows
    x[8] = rng.standard_normal((2, dim))
    x[8, 0, 3] = np.nan
    x[9] = rng.standard_normal((2, dim))
    x[9, 1, dim - 1] = np.inf
    x[10, :, 0] = -np.inf
    x[11] = -0.0
    x[12, :, ::2] = big
    x[13] = rng.integers(-1, 2, (2, dim))
    x[14] = np.arange(dim) % 16
    x[15] = (np.arange(dim) % 16) * 0.5 + 100
    x[16:] = rng.standard_normal((4, 2, dim)) * 10.0 ** rng.integers(-4, 4, (4, 2, dim))
    x = R.rounded(x, kind)
    store = ag.QuantisedRowsGPU.empty(20, 2, dim, dev, code=code, group=group)
    ag.put_quantised_op(store, up(x, kind, dev), u32(np.arange(20), dev), p)
    got = {k: ag.take_quantised_op(store, u32(np.arange(20), dev), p, k)[0] for k in KINDS}
    p.sync()
    codes, scales = stored(store, dev)
    want_codes, want_scales = R.quantise(x, code, group)
    first = want_scales[..., 0] if code == "i4" else want_scales
    mine = scales[..., 0] if code == "i4" else scales
    assert np.array_equal(np.isnan(mine), np.isnan(first))
    live = ~np.isnan(first)
    assert np.array_equal(mine[live].view(np.uint32), first[live].view(np.uint32))
    assert_codes(codes, want_codes, code, want_scales)
    want = R.values(want_codes, want_scales, code, group)
    for k in KINDS:
        assert_values(got[k].values(), want, k)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("code", CODES)
def test_slices_and_odd_addresses(dev, p, code, kind):
    """keys out of a fused projection [rows, heads of all, dim], a start that is not on 16 bytes, rows read back into a wider tensor"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(11)
    n, heads, dim, group = 37, 3, 64, 32
    for at, width in ((0, 64), (3 * 64, 64), (1, 65), (8, 72)):
        whole = activations(rng, (n, 7, width), kind)
        flat = up(whole.reshape(n, -1), kind, dev)
        item = flat.item_size
        view = ag.RowsGPU(flat.data, dev, (n, heads, dim), kind, (7 * width, width, 1), flat.ptr + at * item)
        x = np.lib.stride_tricks.as_strided(whole.reshape(-1)[at:], (n, heads, dim), [7 * width * 4, width * 4, 4])
        store = ag.QuantisedRowsGPU.empty(64, heads, dim, dev, code=code, group=group)
        slots = u32(rng.permutation(64)[:n], dev)
        ag.put_quantised_op(store, view, slots, p)
        wide = up(np.full((n, 7 * width), 5.0, np.float32), kind, dev)
        into = ag.RowsGPU(wide.data, dev, (n, heads, dim), kind, (7 * width, width, 1), wide.ptr + at * item)
        ag.take_quantised_op(store, slots, p, out=into)
        p.sync()
        want_codes, want_scales = R.quantise(np.ascontiguousarray(x), code, group)
        codes, scales = stored(store, dev)
        assert_codes(codes[slots.raw_values()], want_codes, code, want_scales)
        assert_values(into.values(), R.values(want_codes, want_scales, code, group), kind)
        held = wide.values().reshape(-1)
        mask = np.ones(held.size, bool)
        mask[(at + np.arange(n)[:, None, None] * 7 * width + np.arange(heads)[:, None] * width + np.arange(dim)).reshape(-1)] = False
        assert (held[mask] == 5.0).all()


@pytest.mark.parametrize("dim,group", [(64, 64), (20, 10)])
@pytest.mark.parametrize("code", CODES)
def test_slots_that_are_none_or_out_of_range(dev, p, code, dim, group):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(3)
    n = 50
    x = activations(rng, (n, 2, dim), "f16")
    slots = rng.permutation(80)[:n].astype(np.int64)
    none, bad = [0, 7, 49], [1, 20]
    slots[none] = R.NO_ROW
    slots[bad] = [80, 0xFFFFFFFE]
    good = np.setdiff1d(np.arange(n), none + bad)
    store = ag.QuantisedRowsGPU.empty(80, 2, dim, dev, code=code, group=group)
    ag.put_quantised_op(store, up(x, "f16", dev), u32(slots, dev), p)
    with pytest.raises(ag.ArrowErrorGPU) as e:
        p.sync()
    assert e.value.status == capi.ERR_SHAPE
    p.sync()  # reported once
    want_codes, want_scales = R.quantise(x[good], code, group)
    codes, scales = stored(store, dev)
    assert_codes(codes[slots[good]], want_codes, code, want_scales)
    untouched = np.setdiff1d(np.arange(80), slots[good])
    assert not codes[untouched].any() and not scales[untouched].any()
    out = up(np.full((n, 2, dim), 9.0, np.float32), "f16", dev)
    with pytest.raises(ag.ArrowErrorGPU):
        ag.take_quantised(store, u32(slots, dev), out=out)
    got = out.values()
    assert_values(got[good], R.values(want_codes, want_scales, code, group), "f16")
    assert (got[none] == 9.0).all() and (got[bad] == 0.0).all()
    only_none = u32(np.full(n, R.NO_ROW), dev)
    ag.put_quantised(store, up(x, "f16", dev), only_none)  # nothing stored, nothing reported
    assert np.array_equal(stored(store, dev)[0], codes)


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("code,dim,group", [("i8", 64, 32), ("i4", 96, 96), ("e4m3", 12, 6)])
def test_pages(dev, p, code, dim, group, page):
    """ragged sequences, empty ones first, last and between, that end inside pages; rows before the first and behind the last are left"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(page)
    lens = [0, 5, 1, 0, 0, 3 * page, 70, 17, 0]
    lead, behind = 3, 6
    offsets = lead + np.concatenate([[0], np.cumsum(lens)])
    n = int(offsets[-1]) + behind
    first = rng.integers(0, 2 * page + 1, len(lens))
    most = -(-(max(lens) + 2 * page) // page) + 1
    tables = rng.permutation(len(lens) * most).reshape(len(lens), most).astype(np.uint32)
    slots_n = len(lens) * most * page
    tables[6, 1] = R.NO_ROW
    x = activations(rng, (n, 2, dim), "bf16")
    pages = ag.PageMap(ag.RowsGPU.from_numpy(tables, dev), page, u32(offsets, dev), u32(first, dev))
    store = ag.QuantisedRowsGPU.empty(slots_n, 2, dim, dev, code=code, group=group)
    ag.put_quantised_op(store, up(x, "bf16", dev), pages, p)
    out = up(np.full((n, 2, dim), 9.0, np.float32), "bf16", dev)
    ag.take_quantised_op(store, pages, p, out=out)
    p.sync()
    slots = R.slots_of(tables, page, offsets, n, slots_n, first)
    some = slots >= 0
    want_codes, want_scales = R.quantise(x[some], code, group)
    codes, scales = stored(store, dev)
    assert_codes(codes[slots[some]], want_codes, code, want_scales)
    untouched = np.setdiff1d(np.arange(slots_n), slots[some])
    assert not codes[untouched].any() and not scales[untouched].any()
    got = out.values()
    assert_values(got[some], R.values(want_codes, want_scales, code, group), "bf16")
    assert (got[~some] == 9.0).all()
    again = ag.take_quantised_op(store, pages, p, "f32", n_rows=n)[0]
    p.sync()
    assert_values(again.values()[some], R.values(want_codes, want_scales, code, group), "f32")


@pytest.mark.parametrize("code,dim,group", [("i8", 64, 32), ("i4", 96, 96), ("e4m3", 12, 6)])
def test_a_slot_named_twice(dev, p, code, dim, group):
    """what the slot holds then may come from either row, group by group or mixed; the other slots are right"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(31)
    n, heads = 300, 3
    x = activations(rng, (n, heads, dim), "f32")
    slots = rng.permutation(n + 20)[:n]
    slots[200:260] = slots[7]
    store = ag.QuantisedRowsGPU.empty(n + 20, heads, dim, dev, code=code, group=group)
    ag.put_quantised_op(store, up(x, "f32", dev), u32(slots, dev), p)
    p.sync()
    codes, scales = stored(store, dev)
    want_codes, want_scales = R.quantise(x, code, group)
    once = np.array([s != slots[7] for s in slots])
    assert np.array_equal(scales[slots[once]].view(np.uint32), want_scales[once].view(np.uint32))
    assert_codes(codes[slots[once]], want_codes[once], code, want_scales[once])
    left = np.setdiff1d(np.arange(n + 20), slots)
    assert not codes[left].any() and not scales[left].any()
    assert np.isin(scales[slots[7]].reshape(heads, -1), want_scales[~once].reshape(61, heads, -1)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_4_bit_values_are_rounded_once_and_the_same_each_time(dev, p, kind):
    """code * scale + lowest with one rounding to f32 (a rounded product would be off by up to half a step of the product, which can be many of the value's),
    then one to the rows' type; other rows through the same kernels between two runs change nothing"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(13)
    n, heads, dim, group = 96, 8, 128, 64
    x, other = (activations(rng, (n, heads, dim), "bf16") for _ in range(2))
    slots, back = u32(rng.permutation(4096)[:n], dev), []
    store = ag.QuantisedRowsGPU.empty(4096, heads, dim, dev, code="i4", group=group)
    for rows in (x, other, x, other, x):
        ag.put_quantised_op(store, up(rows, "bf16", dev), slots, p)
        back.append(ag.take_quantised_op(store, slots, p, kind)[0])
    p.sync()
    got = [b.values().astype(np.float32) for b in back]
    codes, scales = R.quantise(x, "i4", group)
    # a code of 4 bits times a scale of 24 is exact in 64 bits, the sum is within 2^-53 of it: no f32 border is that near for these rows
    want = R.values(codes, scales, "i4", group).astype(np.float32)
    assert np.array_equal(got[0].view(np.uint32), R.rounded(want, kind).view(np.uint32))
    assert np.array_equal(got[0], got[2]) and np.array_equal(got[0], got[4]) and np.array_equal(got[1], got[3])


def test_pages_out_of_range(dev, p):
    import arrow_gpu_amd as ag

    tables = np.array([[0, 1], [5, 2]], np.uint32)  # page 5 lies behind the cache
    offsets = np.array([0, 6, 9], np.uint32)        # sequence 0: two positions more than its pages hold
    store = ag.QuantisedRowsGPU.empty(8, 1, 16, dev)
    pages = ag.PageMap(ag.RowsGPU.from_numpy(tables, dev), 2, u32(offsets, dev))
    x = R.rounded(np.random.default_rng(0).standard_normal((9, 1, 16)), "f32")
    ag.put_quantised_op(store, up(x, "f32", dev), pages, p)
    with pytest.raises(ag.ArrowErrorGPU):
        p.sync()
    out = up(np.full((9, 1, 16), 9.0, np.float32), "f32", dev)
    ag.take_quantised_op(store, pages, p, out=out)
    with pytest.raises(ag.ArrowErrorGPU):
        p.sync()
    slots = R.slots_of(tables, 2, offsets, 9, 8)
    assert slots.tolist() == [0, 1, 2, 3, -2, -2, -2, -2, 4]
    got = out.values()
    assert (got[slots == -2] == 0).all()
    c, s = R.quantise(x[slots >= 0], "i8", 16)
    assert_values(got[slots >= 0], R.values(c, s, "i8", 16), "f32")


def test_many_caches_in_one_call(dev, p):
    """caches of different codes, groups, types and sizes by one slot column, as the layers of a model"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(9)
    n, cases = 41, [("i8", "bf16", 4, 64, 64), ("i8", "bf16", 4, 64, 64), ("i4", "bf16", 4, 64, 32), ("e4m3", "f32", 2, 48, 24), ("i8", "f16", 1, 10, 5)] + [("i8", "bf16", 4, 64, 64)] * 40
    slots = rng.permutation(64)[:n]
    xs = [activations(rng, (n, h, d), kind) for _, kind, h, d, _ in cases]
    stores = [ag.QuantisedRowsGPU.empty(64 + 3 * (i % 5), h, d, dev, code=code, group=g) for i, (code, _, h, d, g) in enumerate(cases)]
    ag.put_quantised_op(stores, [up(x, c[1], dev) for x, c in zip(xs, cases)], u32(slots, dev), p)
    out = [ag.RowsGPU.empty((n, c[2], c[3]), c[1], dev) for c in cases]
    ag.take_quantised_op(stores, u32(slots, dev), p, out=out)
    p.sync()
    for x, store, o, (code, kind, _, _, g) in zip(xs, stores, out, cases):
        c, s = R.quantise(x, code, g)
        assert_codes(stored(store, dev)[0][slots], c, code, s)
        assert_values(o.values(), R.values(c, s, code, g), kind)


def test_no_rows_and_no_caches(dev, p):
    import arrow_gpu_amd as ag

    store = ag.QuantisedRowsGPU.empty(4, 1, 16, dev)
    ag.put_quantised_op([], [], u32([], dev), p)
    assert ag.take_quantised_op([], u32([], dev), p) == []
    ag.put_quantised_op(store, ag.RowsGPU.empty((0, 1, 16), "f32", dev), u32([], dev), p)
    assert len(ag.take_quantised_op(store, u32([], dev), p)[0]) == 0
    assert ag.take_rows_op([], u32([1], dev), p) == []
    assert len(ag.take_rows_op(up(np.ones((3, 4), np.float32), "f32", dev), u32([], dev), p)[0]) == 0
    sel = ag.select_beams_op(ag.RowsGPU.empty((0, 10), "f32", dev), 2, 3, p)
    assert sel.values()[0].shape == (0, 3)
    p.sync()


def test_a_cache_past_32_bits(dev, p):
    """slots whose codes lie more than 4 GiB behind the first"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(2)
    n_slots, heads, dim = 5_000_000, 8, 128
    store = ag.QuantisedRowsGPU.empty(n_slots, heads, dim, dev, code="i8", group=128)
    slots = np.concatenate([rng.integers(0, n_slots - 8, 20), np.arange(n_slots - 8, n_slots)])
    slots = np.unique(slots)
    x = activations(rng, (len(slots), heads, dim), "bf16")
    ag.put_quantised_op(store, up(x, "bf16", dev), u32(slots, dev), p)
    got = ag.take_quantised_op(store, u32(slots, dev), p, "f32")[0]
    pages = ag.PageMap(ag.RowsGPU.from_numpy(np.array([[n_slots // 8 - 1]], np.uint32), dev), 8, u32([0, 8], dev))
    tail = ag.take_quantised_op(store, pages, p, "f32", n_rows=8)[0]
    p.sync()
    c, s = R.quantise(x, "i8", 128)
    want = R.values(c, s, "i8", 128)
    assert_values(got.values(), want, "f32")
    assert_values(tail.values(), want[-8:], "f32")


# ------------------------------------------------------------------------------------------------------------- take_rows
@pytest.mark.parametrize("type_,shape", [("bf16", (8, 4, 33, 64)), ("u8", (5, 3, 7, 11)), ("f32", (16, 5)), ("u32", (3, 1000)), ("i64", (4, 9)), ("f16", (2, 1, 1, 1)),
                                         ("u8", (40, 4099)), ("bf16", (6, 17, 80)), ("f32", (1, 8, 64, 32)), ("u8", (300, 16)), ("i8", (9, 2, 5, 8))])
def test_take_rows(dev, p, type_, shape):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(shape[0] + shape[-1])
    wide = {"bf16": np.uint16, "u8": np.uint8, "i8": np.uint8, "f32": np.uint32, "u32": np.uint32, "i64": np.uint64, "f16": np.uint16}[type_]
    make = lambda s: rng.integers(0, np.iinfo(wide).max, s, dtype=wide, endpoint=True)  # noqa: E731 — every bit pattern, NaN among them
    view = lambda a: ag.RowsGPU(dev.create_gpu_buffer_with_data(a), dev, a.shape, type_)  # noqa: E731
    raw = lambda r: dev.retrive_data(r.data).view(wide)[:int(np.prod(r.shape))].reshape(r.shape)  # noqa: E731
    a, b = make(shape), make(shape)
    idx = rng.integers(0, shape[0], shape[0] + 3)
    got = ag.take_rows_op([view(a), view(b)], u32(idx, dev), p)
    p.sync()
    assert np.array_equal(raw(got[0]), a[idx]) and np.array_equal(raw(got[1]), b[idx])
    # rows that are none are left, rows out of range are zeros
    odd = idx.copy()
    odd[0], odd[-1] = R.NO_ROW, shape[0]
    before = make((len(idx),) + shape[1:])
    out = view(before)
    ag.take_rows_op(view(a), u32(odd, dev), p, out=out)
    with pytest.raises(ag.ArrowErrorGPU):
        p.sync()
    want = a[np.where(odd < shape[0], odd, 0)]
    want[0], want[-1] = before[0], 0
    assert np.array_equal(raw(out), want)
    if len(shape) > 2:
        most = shape[-2]
        lengths = rng.integers(0, most + 3, len(idx))
        lengths[0] = 0
        lengths[1] = 0xFFFFFFFF
        out = view(before)
        ag.take_rows_op(view(a), u32(idx, dev), p, lengths=u32(lengths, dev), out=out)
        p.sync()
        live = np.arange(most) < lengths[:, None]
        live = live[:, None, :, None] if len(shape) == 4 else live[:, :, None]
        assert np.array_equal(raw(out), np.where(live, a[idx], before))


@pytest.mark.parametrize("at,pitch", [(0, 80), (1, 81), (2, 96), (8, 72)])
def test_take_rows_of_slices(dev, p, at, pitch):
    """a state inside a wider one (rows and pieces further apart than they are long), on 16, 4, 2 byte starts"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(at)
    rows, pieces, dim = 6, 3, 64
    whole = rng.integers(0, 65536, (rows, 2 * pieces, pitch), dtype=np.uint16)
    src = dev.create_gpu_buffer_with_data(whole)
    into = dev.create_gpu_buffer_with_data(np.full((rows, 2 * pieces, pitch), 7, np.uint16))
    view = lambda buf: ag.RowsGPU(buf, dev, (rows, pieces, dim), "f16", (2 * pieces * pitch, pitch, 1), buf.ptr + 2 * at)  # noqa: E731
    idx = rng.integers(0, rows, rows)
    ag.take_rows_op(view(src), u32(idx, dev), p, out=view(into))
    p.sync()
    got = dev.retrive_data(into).view(np.uint16)[:whole.size].reshape(whole.shape)
    want = np.full_like(whole, 7)
    np.lib.stride_tricks.as_strided(want.reshape(-1)[at:], (rows, pieces, dim), [4 * pieces * pitch, 2 * pitch, 2])[:] = \
        np.lib.stride_tricks.as_strided(whole.reshape(-1)[at:], (rows, pieces, dim), [4 * pieces * pitch, 2 * pitch, 2])[idx]
    assert np.array_equal(got, want)


@pytest.mark.parametrize("type_,wide", [("u8", np.uint8), ("bf16", np.uint16), ("f32", np.uint32)])
def test_take_rows_whose_positions_lie_apart(dev, p, type_, wide):
    """(rows, positions, values) with a gap behind each position: into dense rows that the call allocates, and from dense rows into gaps that stay as they were"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(12)
    rows, positions, values, pitch = 7, 9, 21, 26
    whole = rng.integers(0, np.iinfo(wide).max, (rows, positions, pitch), dtype=wide, endpoint=True)
    raw = lambda b, shape: dev.retrive_data(b).view(wide)[:int(np.prod(shape))].reshape(shape)  # noqa: E731
    apart = lambda b: ag.RowsGPU(b, dev, (rows, positions, values), type_, (positions * pitch, pitch, 1))  # noqa: E731
    idx = rng.integers(0, rows, rows)
    got = ag.take_rows_op(apart(dev.create_gpu_buffer_with_data(whole)), u32(idx, dev), p)[0]
    p.sync()
    assert np.array_equal(raw(got.data, (rows, positions, values)), whole[idx][..., :values])
    into = dev.create_gpu_buffer_with_data(np.full_like(whole, 7))
    ag.take_rows_op(got, u32(idx, dev), p, out=apart(into))
    p.sync()
    want = np.full_like(whole, 7)
    want[..., :values] = whole[idx][idx][..., :values]
    assert np.array_equal(raw(into, whole.shape), want)


def test_states_that_lie_interleaved_in_one_allocation(dev, p):
    """[rows, (old keys, new keys, old values, new values), heads, values]: taken from their places into those beside them"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(17)
    rows, heads, values = 9, 3, 21
    whole = rng.integers(0, 65536, (rows, 4, heads, values), dtype=np.uint16)
    buf = dev.create_gpu_buffer_with_data(whole)
    part = lambda i: ag.RowsGPU(buf, dev, (rows, heads, values), "f16", (4 * heads * values, values, 1), buf.ptr + 2 * i * heads * values)  # noqa: E731
    idx = rng.integers(0, rows, rows)
    ag.take_rows_op([part(0), part(2)], u32(idx, dev), p, out=[part(1), part(3)])
    p.sync()
    want = whole.copy()
    want[:, 1], want[:, 3] = whole[idx, 0], whole[idx, 2]
    assert np.array_equal(dev.retrive_data(buf).view(np.uint16)[:whole.size].reshape(whole.shape), want)
    for states, out in (([part(0)], [part(0)]), ([part(0), part(2)], [part(1), part(1)]), ([part(0), part(1)], [part(2), part(0)])):
        with pytest.raises(ag.ArrowErrorGPU) as e:
            ag.take_rows_op(states, u32(idx, dev), p, out=out)
        assert e.value.status == capi.ERR_ARG


def test_take_rows_past_32_bits(dev, p):
    """a state of more than 4 GiB"""
    import arrow_gpu_amd as ag

    rows, width = 5, 1 << 28  # 5 rows of 1 GiB
    src = ag.RowsGPU.empty((rows, width), "f32", dev)
    out = ag.RowsGPU.empty((rows, width), "f32", dev)
    for r in range(rows):
        capi.call("agpu_synth_i32", p._handle, C.c_void_p(src.ptr + 4 * r * width), width, 77, r * width, 0xFFFFFFFF)
    idx = [4, 4, 0, 3, 1]
    ag.take_rows_op(src, u32(idx, dev), p, out=out)
    p.sync()
    for r, i in enumerate(idx):
        for c in (0, 12345, width - 4096):
            a = ag.DeviceBuffer(dev, src.ptr + 4 * (i * width + c), 16384, owned=False)
            b = ag.DeviceBuffer(dev, out.ptr + 4 * (r * width + c), 16384, owned=False)
            assert np.array_equal(dev.retrive_data(a), dev.retrive_data(b))


# ---------------------------------------------------------------------------------------------------------- select_beams
# The largest relative error of a sum of positive terms is the largest of a term's and its additions' together: a term 2^f, f rounded twice below 1/2
# (2 · 2^-26, times ln 2), by an instruction within one unit of f32 (2^-23); groups of 16 terms added pair by pair, 4 roundings of 2^-24 each; the groups
# in f64.  The logarithm's error is that.
LOG_SUM = 2.0**-23 + np.log(2) * 2.0**-25 + 4 * 2.0**-24 + 1e-12


def assert_selection(sel, want, tol=None):
    """parents and tokens are whole numbers; a score is rounded to f32 once, and its log-sum is off by less than LOG_SUM"""
    s, r, t = sel.values()
    ws, wr, wt = want
    assert np.array_equal(r, wr) and np.array_equal(t, wt), (np.argwhere((r != wr) | (t != wt))[:4], s[(r != wr) | (t != wt)][:4], ws[(r != wr) | (t != wt)][:4])
    assert np.array_equal(np.isfinite(s), np.isfinite(ws)) and np.array_equal(s[~np.isfinite(ws)], ws[~np.isfinite(ws)])
    fine = np.isfinite(ws)
    assert (np.abs(s[fine] - ws[fine]) <= np.abs(ws[fine]) * R.HALF_STEP["f32"] * (1 + 2.0**-10) + LOG_SUM).all()


def logits(rng, rows, vocab, kind):
    x = rng.standard_normal((rows, vocab)).astype(np.float32) * 2
    x[np.arange(rows)[:, None], rng.integers(0, vocab, (rows, min(vocab, 12)))] += 8
    return R.rounded(x, kind)


@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 1, 1, 1), (1, 1, 2, 2), (1, 4, 7, 28), (2, 3, 63, 6), (3, 5, 64, 10), (1, 2, 65, 64), (2, 8, 1000, 16), (1, 4, 32000, 8),
                                                 (4, 3, 50257, 6), (1, 1, 128256, 64), (7, 2, 4097, 4), (1, 64, 513, 64), (33, 1, 8192, 1), (2, 1024, 5, 64)])
@pytest.mark.parametrize("kind", KINDS)
def test_select(dev, p, kind, batch, beams, vocab, k):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(batch * 7 + vocab)
    x = logits(rng, batch * beams, vocab, kind)
    cum = -np.float32(15) * rng.random(batch * beams).astype(np.float32)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev))
    again = ag.select_beams_op(up(x, kind, dev), beams, k, p)
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), beams, k, cum))
    assert_selection(again, R.select(x.astype(np.float64), beams, k))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [64, 50, 999, 4099, 20011])
def test_select_masked_and_finished(dev, p, kind, vocab):
    """per-row bitmaps that leave much, little, one token and nothing; NaN, infinities and the type's extremes in masked places"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(vocab)
    batch, beams, k = 4, 5, 10
    rows, pitch = batch * beams, (vocab + 63) // 64 * 64
    x = logits(rng, rows, vocab, kind)
    allowed = np.zeros((rows, pitch), bool)
    allowed[:, :vocab] = rng.random((rows, vocab)) < rng.choice([0.02, 0.5, 0.97], (rows, 1))
    allowed[0] = False
    allowed[2] = False
    allowed[2, vocab - 1] = True
    allowed[5:10] = False          # request 1: nothing at all
    allowed[10:15] = False         # request 2: one token in all
    allowed[13, vocab // 2] = True
    x[~allowed[:, :vocab]] = R.rounded(rng.choice(np.array([np.nan, np.inf, -np.inf, 6e4, -6e4], np.float32), (~allowed[:, :vocab]).sum()), kind)
    allowed[:, vocab:] = True      # the padding's bits say nothing
    finished = rng.random(rows) < 0.2
    finished[13] = False
    cum = -np.float32(15) * rng.random(rows).astype(np.float32)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev), allowed=bits(allowed, dev), finished=bits(finished, dev),
                             end_token=vocab - 1)
    shared = ag.select_beams_op(up(np.where(allowed[3, :vocab], logits(rng, rows, vocab, kind), 1), kind, dev), beams, k, p, allowed=bits(allowed[3], dev))
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), beams, k, cum, allowed[:, :vocab], finished, vocab - 1))
    assert shared.values()[0].shape == (batch, k)
    assert allowed[3, shared.values()[2][shared.values()[0] > -np.inf]].all()


def test_select_ties_and_rows_without_a_distribution(dev, p):
    import arrow_gpu_amd as ag

    vocab, beams, k = 9000, 4, 12
    x = np.zeros((16, vocab), np.float32)                # request 0: every score equal → the first tokens of the first row
    x[4:8] = (np.arange(vocab) % 7 == 3) * 2.0           # request 1: many at the top
    x[8] = np.nan                                        # request 2: one row without a distribution for each reason, one with
    x[9, 77] = np.inf
    x[10] = -np.inf
    x[11, 5:] = -np.inf                                  # five live tokens in all: the rest in order
    x[11, :5] = [0, -1, 0, -2, -0.0]
    x[12:16] = -np.inf                                   # request 3: nothing
    for kind in KINDS:
        sel = ag.select_beams_op(up(x, kind, dev), beams, k, p)
        p.sync()
        want = R.select(x.astype(np.float64), beams, k)
        assert want[2][0].tolist() == list(range(k)) and set(want[1][2][:5]) == {11} and want[2][2][5:].tolist() == list(range(7))
        assert_selection(sel, want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("k", [1, 5, 16, 64])
@pytest.mark.parametrize("low", [0.0, -1e4, -3e38, -2.5])
def test_select_very_many_equal_logits(dev, p, kind, k, low):
    """rows in which all but a few logits hold one value (a mask's lowest number), the few anywhere; and rows of a few values many times"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(k)
    low = max(low, -6e4) if kind == "f16" else low
    beams, vocab = 2, 40009
    x = np.full((10, vocab), low, np.float32)
    for r in range(6):
        at = rng.integers(0, vocab, r * 4)
        x[r, at] = np.maximum(low, 0) + 3 * rng.random(len(at))
    x[4, ::2] = low + 0.5
    x[6] = rng.integers(0, 3, vocab) - 1.0
    x[7, vocab - 20:] = rng.random(20) * 5 + np.maximum(low, 0)
    x[8] = np.where(rng.random(vocab) < 0.999, low, low + 1)
    x[9] = np.minimum(np.arange(vocab) // 64, 500)       # rising
    x = R.rounded(x, kind)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p)
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), beams, k))


@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 32, 5000, 64), (2, 64, 777, 64), (1, 1, 150001, 64), (3, 4, 12345, 33), (2, 9, 33000, 50), (1, 1024, 40, 64)])
@pytest.mark.parametrize("kind", KINDS)
def test_select_many_beams_and_a_large_k(dev, p, kind, batch, beams, vocab, k):
    """thousands of entries to join for a request"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(beams + k)
    x = logits(rng, batch * beams, vocab, kind)
    cum = -np.float32(3) * rng.random(batch * beams).astype(np.float32)
    cum[:beams] = 0.0
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev))
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), beams, k, cum))


def test_select_candidates_beside_each_other(dev, p):
    """640 tokens of a row are all that is above -infinity, 16 in each of some stretches of 1024: no bound is known before they are joined"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(3)
    x = np.full((2, 262144), -np.inf, np.float32)
    for j in (0, 12, 19, 24, 31):
        for seg in range(8 * j, 8 * j + 8):
            at = seg * 1024 + rng.choice(1024, 16, replace=False)
            x[0, at] = 5 * rng.random(16)
            x[1, at] = rng.integers(0, 40, 16)           # and many equal ones
    for k in (16, 40, 64):
        sel = ag.select_beams_op(up(x, "f32", dev), 1, k, p)
        p.sync()
        assert_selection(sel, R.select(x.astype(np.float64), 1, k))


def test_select_rows_of_one_row(dev, p):
    """one row of logits for all beams (stride 0), as at a request's first step"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(8)
    x = logits(rng, 1, 5001, "bf16")
    flat = up(x, "bf16", dev)
    view = ag.RowsGPU(flat.data, dev, (6, 5001), "bf16", (0, 1))
    cum = -3 * rng.random(6).astype(np.float32)
    sel = ag.select_beams_op(view, 3, 9, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev))
    p.sync()
    assert_selection(sel, R.select(np.repeat(x, 6, 0).astype(np.float64), 3, 9, cum))


@pytest.mark.parametrize("vocab,pitch", [(5001, 5003), (999, 1000), (50257, 50257), (13, 17), (70001, 70016)])
@pytest.mark.parametrize("kind", KINDS)
def test_select_equal_rows_have_equal_scores(dev, p, kind, vocab, pitch):
    """wherever in memory the rows begin: of equal scores the lower row's comes first"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(vocab)
    beams, k = 7, 12
    x = np.repeat(logits(rng, 2, vocab, kind), beams, 0)
    wide = np.zeros((2 * beams, pitch), np.float32)
    wide[:, :vocab] = x
    base = up(wide, kind, dev)
    view = ag.RowsGPU(base.data, dev, (2 * beams, vocab), kind, (pitch, 1))
    allowed = np.tile(rng.random((1, (vocab + 63) // 64 * 64)) < 0.6, (2 * beams, 1))
    for mask in (None, allowed):
        sel = ag.select_beams_op(view, beams, k, p, allowed=bits(mask, dev) if mask is not None else None)
        p.sync()
        want = R.select(x.astype(np.float64), beams, k, allowed=mask[:, :vocab] if mask is not None else None)
        assert want[1][0, :beams].tolist() == list(range(beams))
        assert_selection(sel, want)


@pytest.mark.parametrize("kind", KINDS)
def test_select_forced_tokens_keep_the_scores(dev, p, kind):
    """rows whose mask leaves one token: its log-softmax is 0, the running score stays what it was"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(4)
    beams, vocab, k = 6, 30011, 6
    x = logits(rng, 2 * beams, vocab, kind)
    allowed = np.zeros((2 * beams, (vocab + 63) // 64 * 64), bool)
    only = rng.integers(0, vocab, 2 * beams)
    allowed[np.arange(2 * beams), only] = True
    cum = np.repeat(-np.float32(3) * rng.random(4).astype(np.float32), 3)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev), allowed=bits(allowed, dev))
    x[~allowed[:, :vocab]] = -np.inf
    bare = ag.select_beams_op(up(x, kind, dev), beams, k, p)
    p.sync()
    s, r, t = sel.values()
    for b in range(2):
        order = np.argsort(-cum[b * beams:(b + 1) * beams], kind="stable") + b * beams
        assert np.array_equal(s[b], cum[order]) and np.array_equal(r[b], order) and np.array_equal(t[b], only[order])
    s, r, t = bare.values()
    assert not s.any() and np.array_equal(r.reshape(-1), np.arange(2 * beams)) and np.array_equal(t.reshape(-1), only)


def test_select_scores_at_the_ends(dev, p):
    """the first step (one live beam), NaN and infinite running scores, also of finished rows"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(1)
    beams, vocab, k = 4, 500, 8
    x = logits(rng, 24, vocab, "bf16")
    cum = np.zeros(24, np.float32)
    cum[1:4] = -np.inf
    cum[4:8] = -np.inf
    cum[8], cum[9] = np.nan, np.inf
    cum[12:14] = np.inf
    cum[16:20] = [3e38, -3e38, 0, 1]
    finished = np.zeros(24, bool)
    finished[[2, 4, 8, 13, 17, 20, 21, 22, 23]] = True
    sel = ag.select_beams_op(up(x, "bf16", dev), beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev), finished=bits(finished, dev), end_token=3)
    p.sync()
    with np.errstate(over="ignore"):
        assert_selection(sel, R.select(x.astype(np.float64), beams, k, cum, None, finished, 3))


@pytest.mark.parametrize("at,pitch", [(0, 1000), (1, 1001), (3, 1031), (8, 1024)])
@pytest.mark.parametrize("kind", KINDS)
def test_select_from_slices(dev, p, kind, at, pitch):
    """logits inside a wider tensor, rows on every alignment; what lies beside them is NaN"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(at)
    beams, vocab, k = 3, 997, 6
    whole = np.full((9, pitch + 8), np.nan, np.float32)
    x = logits(rng, 9, vocab, kind)
    whole.reshape(-1)[at:at + 9 * pitch].reshape(9, pitch)[:, :vocab] = x
    flat = up(whole, kind, dev)
    view = ag.RowsGPU(flat.data, dev, (9, vocab), kind, (pitch, 1), flat.ptr + at * flat.item_size)
    sel = ag.select_beams_op(view, beams, k, p)
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), beams, k))


def test_select_past_32_bits(dev, p):
    """rows whose logits lie more than 4 GiB behind the first; nearly all of them equal"""
    import arrow_gpu_amd as ag

    vocab, beams, k = 800_000_011, 3, 5
    x = ag.RowsGPU.empty((beams, vocab), "bf16", dev)
    capi.call("agpu_memset", p._handle, C.c_void_p(x.ptr), 0, 2 * beams * vocab)
    places = [(2, vocab - 1, 9.0), (1, vocab // 2, 6.0), (0, 7, 3.0)]
    for r, t, v in places:
        bits16 = np.array([v], np.float32).view(np.uint32) >> 16
        half = np.ascontiguousarray(bits16.astype(np.uint16))
        capi.call("agpu_upload", p._handle, C.c_void_p(x.ptr + 2 * (r * vocab + t)), C.c_void_p(half.ctypes.data), 2)
    cum = np.array([0.0, -1.0, -2.0], np.float32)
    sel = ag.select_beams_op(x, beams, k, p, scores=ag.Float32ArrayGPU.from_slice(cum, dev))
    p.sync()
    lse = {r: np.log(vocab - 1 + np.exp(v)) for r, _, v in places}
    want = [cum[r] + (v - lse[r]) for r, _, v in places] + [-lse[0], -lse[0]]
    assert_selection(sel, (np.array([want]), np.array([[2, 1, 0, 0, 0]]), np.array([[vocab - 1, vocab // 2, 7, 0, 1]])))


def test_select_far_apart_logits(dev, p):
    """logits over the whole range of f32: the sum's terms vanish, one by one"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(4)
    x = (rng.standard_normal((6, 3001)) * 10.0 ** rng.integers(-6, 37, (6, 3001))).astype(np.float32)
    x[3] = 3.4e38
    x[4] = -3.4e38
    x[5] = np.where(np.arange(3001) < 2000, -3.4e38, 3.4e38)
    sel = ag.select_beams_op(up(x, "f32", dev), 1, 20, p)
    p.sync()
    assert_selection(sel, R.select(x.astype(np.float64), 1, 20))


# ------------------------------------------------------------------------------------------------------- a run of them
def _search(ag, dev, p, steps, state, inputs, want=None):
    """One step of a beam search over a paged, quantised cache: new rows in, context out, selection, tables and states by the parents."""
    for x, lg in inputs[:steps]:
        ag.put_quantised_op(state["stores"], x, state["slots"], p)
        state["read"] = ag.take_quantised_op(state["stores"], state["pages"], p, out=state["context"])
        state["sel"] = ag.select_beams_op(lg, state["beams"], state["beams"], p, scores=state["scores"], out=state["sel"])
        ag.take_rows_op(state["states"], state["sel"].parents, p, lengths=state["lengths"], out=state["next"])


def _search_state(ag, dev, rng):
    batch, beams, vocab, heads, dim, page = 2, 4, 1003, 2, 64, 8
    rows = batch * beams
    state = {"beams": beams, "vocab": vocab, "rows": rows}
    state["stores"] = [ag.QuantisedRowsGPU.empty(rows * 2 * page, heads, dim, dev, code=c, group=32) for c in ("i8", "i4")]
    tables = rng.permutation(rows * 2).reshape(rows, 2).astype(np.uint32)
    lens = rng.integers(1, 2 * page, rows)
    state["slots_np"] = tables[np.arange(rows), (lens - 1) // page] * page + (lens - 1) % page
    state["slots"] = u32(state["slots_np"], dev)
    offsets = np.concatenate([[0], np.cumsum(lens)])
    state["map"] = R.slots_of(tables, page, offsets, int(offsets[-1]), rows * 2 * page)
    state["tables"] = ag.RowsGPU.from_numpy(tables, dev)
    state["pages"] = ag.PageMap(state["tables"], page, u32(offsets, dev))
    state["context"] = [ag.RowsGPU.empty((int(offsets[-1]), heads, dim), "f32", dev) for _ in range(2)]
    state["scores_np"] = -5 * rng.random(rows).astype(np.float32)
    state["scores"] = ag.Float32ArrayGPU.from_slice(state["scores_np"], dev)
    state["held"] = rng.standard_normal((rows, heads, 10, dim)).astype(np.float32)
    state["lengths_np"] = rng.integers(0, 11, rows)
    state["lengths"] = u32(state["lengths_np"], dev)
    state["states"] = [ag.RowsGPU.from_numpy(state["held"], dev)]
    state["next"] = [ag.RowsGPU.from_numpy(np.zeros_like(state["held"]), dev)]
    state["sel"] = ag.BeamSelection.empty(batch, beams, dev)
    return state


def _check_search(state, x, lg):
    for store, code, got, xv in zip(state["stores"], ("i8", "i4"), state["context"], x):
        cache = np.zeros((store.n_slots, store.heads, store.dim))
        c, s = R.quantise(xv, code, 32)
        cache[state["slots_np"]] = R.values(c, s, code, 32)
        assert_values(got.values(), cache[state["map"]], "f32")
    want = R.select(lg.astype(np.float64), state["beams"], state["beams"], state["scores_np"])
    assert_selection(state["sel"], want)
    live = (np.arange(10) < state["lengths_np"][:, None])[:, None, :, None]
    assert np.array_equal(state["next"][0].values(), np.where(live, state["held"][want[1].reshape(-1)], 0))


def test_a_step_of_a_search(dev, p):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(21)
    state = _search_state(ag, dev, rng)
    x = [activations(rng, (state["rows"], 2, 64), "bf16") for _ in range(2)]
    lg = logits(rng, state["rows"], state["vocab"], "bf16")
    _search(ag, dev, p, 1, state, [([up(v, "bf16", dev) for v in x], up(lg, "bf16", dev))])
    p.sync()
    _check_search(state, x, lg)


def test_a_step_captured_and_replayed(dev, p):
    """the step as a graph, replayed over new inputs, with eager work and waits between the replays"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(22)
    state = _search_state(ag, dev, rng)
    rows, vocab = state["rows"], state["vocab"]
    dx = [up(np.zeros((rows, 2, 64), np.float32), "f32", dev) for _ in range(2)]
    dl = up(np.zeros((rows, vocab), np.float32), "f32", dev)
    _search(ag, dev, p, 1, state, [(dx, dl)])  # once before the capture: the selection's workspace is there
    p.sync()
    g = C.c_void_p()
    capi.call("agpu_pipeline_begin_capture", p._handle)
    _search(ag, dev, p, 1, state, [(dx, dl)])
    capi.call("agpu_pipeline_end_capture", p._handle, C.byref(g))
    for _ in range(4):
        x = [activations(rng, (rows, 2, 64), "f32") for _ in range(2)]
        lg = logits(rng, rows, vocab, "f32")
        for d, v in zip(dx + [dl], x + [lg]):
            v = np.ascontiguousarray(v, dtype=np.float32)
            capi.call("agpu_upload", p._handle, C.c_void_p(d.ptr), C.c_void_p(v.ctypes.data), v.nbytes)
        capi.call("agpu_memset", p._handle, C.c_void_p(state["next"][0].ptr), 0, state["held"].nbytes)
        capi.call("agpu_graph_launch", g, p._handle)
        p.sync()
        _check_search(state, x, lg)
        eager = ag.select_beams(dl, state["beams"], state["beams"], scores=state["scores"])  # on a pipeline of its own
        assert_selection(eager, R.select(lg.astype(np.float64), state["beams"], state["beams"], state["scores_np"]))
    capi.call("agpu_graph_destroy", g)


def test_rows_of_columns_that_a_fusing_pipeline_has_only_recorded(dev):
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(41)
    a = rng.standard_normal(64 * 96).astype(np.float32)
    pipe = ag.ArrowComputePipeline(dev, "fusing", fuse=True)
    two, three = (ag.Float32ArrayGPU.from_slice([v], dev) for v in (2.0, 3.0))
    x = ag.add_scalar_op_dyn(ag.mul_scalar_op_dyn(ag.Float32ArrayGPU.from_slice(a, dev), two, pipe), three, pipe)
    store = ag.QuantisedRowsGPU.empty(64, 1, 96, dev)
    slots = u32(rng.permutation(64), dev)
    ag.put_quantised_op(store, ag.RowsGPU.of_array(x, (64, 1, 96)), slots, pipe)
    got = ag.take_quantised_op(store, slots, pipe)[0]
    pipe.finish()
    pipe.sync()
    want = (a * np.float32(2) + np.float32(3)).reshape(64, 1, 96)
    codes, scales = R.quantise(want, "i8", 96)
    assert_values(got.values(), R.values(codes, scales, "i8", 96), "f32")


def test_two_pipelines_at_once(dev):
    """the same calls on two streams, each with its own cache and selection"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(23)
    ps = [ag.ArrowComputePipeline(dev, f"rows {i}") for i in range(2)]
    states = [_search_state(ag, dev, rng) for _ in ps]
    inputs = []
    for s in states:
        inputs.append(([activations(rng, (s["rows"], 2, 64), "f16") for _ in range(2)], logits(rng, s["rows"], s["vocab"], "f16")))
    on_gpu = [([up(v, "f16", dev) for v in x], up(lg, "f16", dev)) for x, lg in inputs]
    for _ in range(20):
        for pipe, s, i in zip(ps, states, on_gpu):
            _search(ag, dev, pipe, 1, s, [i])
    for pipe in ps:
        pipe.sync()
    for s, (x, lg) in zip(states, inputs):
        _check_search(s, x, lg)


def test_torch_tensors():
    """tensors of torch on its streams, without copies: in a process of its own, where torch has loaded the GPU runtime before this library does"""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, os.path.join(here, "torch_rows_check.py")], capture_output=True, text=True, timeout=110, cwd=os.path.dirname(here))
    assert r.returncode == 0 and "torch rows OK" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]

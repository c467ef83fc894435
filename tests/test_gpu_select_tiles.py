"""GPU: select_beams where a wave's segment is more than one tile of 1024 logits — selections of about 8 million logits and more — against the definition
in 64 bits (tests/rows_ref.py): every type, masks, finished rows, rows without a distribution, ties and ascending rows over tiles, far logits."""
import numpy as np
import pytest

import rows_ref as R
from test_gpu_rows import KINDS, LOG_SUM, assert_selection, bits, dev, p, up  # noqa: F401 — dev and p: fixtures

pytestmark = pytest.mark.gpu


def tiles(rows, vocab):
    """of a segment: as many, up to 8, as leave 4096 segments"""
    t = 8
    while t > 1 and rows * -(-vocab // (1024 * t)) < 4096:
        t //= 2
    return t


def logits(rng, rows, vocab, kind):
    x = rng.standard_normal((rows, vocab), dtype=np.float32) * np.float32(2)
    x[np.arange(rows)[:, None], rng.integers(0, vocab, (rows, 12))] += 8
    return R.rounded(x, kind)


def f32(values, dev):  # noqa: F811
    import arrow_gpu_amd as ag

    return ag.Float32ArrayGPU.from_slice(np.asarray(values, np.float32), dev)


def assert_near(sel, want, x, cum):
    """assert_selection() where rows compete whose log-sums are equal, or nearly so, in exact arithmetic (an ascending row and a descending one).  A row's
    scores are all off by one error, at most LOG_SUM: the i-th of the scores so moved is at most LOG_SUM from the i-th of the exact ones, and the exact score of
    the token that stands there at most LOG_SUM from its moved one.  So the token's exact score is at most 2 LOG_SUM from the i-th exact score; and the
    tokens of one row, all moved alike, stand in the exact order."""
    s, r, t = sel.values()
    ws, wr, wt = want
    fine = np.isfinite(ws)
    assert np.array_equal(np.isfinite(s), fine)
    assert (np.abs(s[fine] - ws[fine]) <= np.abs(ws[fine]) * R.HALF_STEP["f32"] * (1 + 2.0**-10) + LOG_SUM).all()
    for b in np.nonzero(((r != wr) | (t != wt)).any(-1))[0]:
        lse = {}
        for row in set(r[b].tolist()):
            v = x[row].astype(np.float64)
            lse[row] = v.max() + np.log(np.exp(v - v.max()).sum())
            mine = t[b][r[b] == row]
            assert np.array_equal(mine, np.lexsort((np.arange(len(v)), -v))[:len(mine)])
        score = np.array([float(cum[p]) + (float(x[p, q]) - lse[p]) for p, q in zip(r[b].tolist(), t[b].tolist())])
        assert fine[b].all() and (np.abs(score - ws[b]) <= 2 * LOG_SUM).all()


LOWEST = {"f32": -3.4028235e38, "f16": -65504.0, "bf16": -3.3895314e38}


@pytest.mark.parametrize("hole", ["masked", "-inf", "lowest"])
@pytest.mark.parametrize("kind", KINDS)
def test_low_logits_behind_a_first_tile_that_holds_none(dev, p, kind, hole):  # noqa: F811
    """a segment whose first tile has no ordinary maximum, its live logits anywhere between -75 and 10: log-sums as near as everywhere, and a row with
    one live token keeps its score"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(len(hole))
    rows, vocab, beams, k = 4096, 8192, 4, 6
    assert tiles(rows, vocab) == 8
    dead = {"masked": 1.0, "-inf": -np.inf, "lowest": LOWEST[kind]}[hole]
    x = np.full((rows, vocab), dead, np.float32)
    allowed = np.zeros((rows, vocab), bool) if hole == "masked" else None
    level = np.repeat(-np.arange(-10, 75.5, 0.5), beams)[np.arange(rows) % (171 * beams)]  # of a request; near one another, as competing rows are
    live = np.where(np.arange(rows) // beams % 2 == 0, 1, 40)
    for r in range(rows):
        at = 1024 + rng.choice(vocab - 1024, live[r], replace=False)
        x[r, at] = level[r] + (rng.random(live[r]) if live[r] > 1 else 0)
        if allowed is not None:
            allowed[r, at] = True
    x = R.rounded(x, kind)
    cum = -np.float32(3) * rng.random(rows).astype(np.float32)
    cum[::beams] = cum[1::beams]  # equal scores too: the lower row's comes first
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev), allowed=bits(allowed, dev) if allowed is not None else None)
    p.sync()
    want = R.select_many(x, beams, k, cum, allowed)
    s, r, t = sel.values()
    lone = live[::beams] == 1
    assert np.array_equal(s[lone][:, :beams], np.sort(cum.reshape(-1, beams)[lone])[:, ::-1])  # exactly
    fine = np.isfinite(want[0])
    assert (np.abs(s[fine] - want[0][fine]) <= np.abs(want[0][fine]) * R.HALF_STEP["f32"] * (1 + 2.0**-10) + LOG_SUM).all(), np.abs(s[fine] - want[0][fine]).max()
    assert_selection(sel, want)


@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("kind", KINDS)
def test_logits_about_the_largest_reference(dev, p, kind, sign):  # noqa: F811
    """a reference is an ordinary number up to 16384: tiles below and above -16384 and 16384 in one segment, close to each other and far apart"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(5 + sign)
    rows, vocab, beams, k = 4096, 8192, 4, 8
    assert tiles(rows, vocab) == 8
    x = sign * np.float32(16384) + rng.random((rows, vocab), dtype=np.float32) * 2
    for r in range(0, rows, beams):  # tile by tile a level of its own, the same in all of a request's rows
        reach = (2.0, 20.0, 100.0, 3000.0)[r // beams % 4]
        x[r:r + beams] += np.repeat(rng.uniform(-reach, reach, vocab // 1024), 1024).astype(np.float32)
    x = R.rounded(x, kind)
    cum = -np.float32(3) * rng.random(rows).astype(np.float32)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev))
    p.sync()
    assert_near(sel, R.select_many(x, beams, k, cum), x, cum)


@pytest.mark.parametrize("rows,vocab,beams,k,of", [(2100, 4001, 7, 14, 2), (1040, 16001, 8, 16, 4), (820, 40003, 4, 64, 8), (4100, 8190, 1, 1, 8), (256, 128256, 8, 16, 8)])
@pytest.mark.parametrize("kind", KINDS)
def test_a_batch(dev, p, kind, rows, vocab, beams, k, of):  # noqa: F811
    """ordinary logits; then with masks that leave much, little, one token and nothing, and whole tiles out, NaN and infinities under them, rows finished"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(rows + vocab)
    assert tiles(rows, vocab) == of
    x = logits(rng, rows, vocab, kind)
    cum = -np.float32(15) * rng.random(rows).astype(np.float32)
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev))
    p.sync()
    assert_selection(sel, R.select_many(x, beams, k, cum))

    pitch = (vocab + 63) // 64 * 64
    allowed = np.zeros((rows, pitch), bool)
    for r in range(rows):
        allowed[r, :vocab] = rng.random(vocab, dtype=np.float32) < (0.001, 0.02, 0.5, 0.97)[r % 4]
    for r in range(0, rows, 3):  # whole tiles, the segment's first among them
        allowed[r, :vocab] &= np.repeat((np.arange(-(-vocab // 1024)) > 0) & (rng.random(-(-vocab // 1024)) < 0.5), 1024)[:vocab]
    allowed[1] = False
    allowed[2] = False
    allowed[2, vocab - 1] = True
    allowed[beams * 5:beams * 6] = False
    some = rng.integers(0, rows * vocab, rows * 40)
    some = some[~allowed[some // vocab, some % vocab]]
    x[some // vocab, some % vocab] = R.rounded(rng.choice(np.array([np.nan, np.inf, -np.inf, 6e4, -6e4], np.float32), len(some)), kind)
    allowed[:, vocab:] = True
    finished = rng.random(rows) < 0.2
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev), allowed=bits(allowed, dev), finished=bits(finished, dev), end_token=vocab // 2)
    p.sync()
    assert_selection(sel, R.select_many(x, beams, k, cum, allowed[:, :vocab], finished, vocab // 2))


@pytest.mark.parametrize("k", [1, 16, 64])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_other_kinds(dev, p, kind, k):  # noqa: F811
    """ascending and descending rows, equal logits, ties that begin in a late tile, spans past a segment's range, rows without a distribution"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(k)
    rows, vocab, beams = 820, 40003, 2
    assert tiles(rows, vocab) == 8
    at = np.arange(vocab)

    def late(n, value, other):
        row = np.full(vocab, other, np.float32)
        row[rng.integers(vocab // 2, vocab, n)] = value
        return row

    def with_one(value, where):
        row = rng.standard_normal(vocab).astype(np.float32)
        row[where] = value
        return row

    make = [lambda: at / 2048.0, lambda: -at / 2048.0, lambda: np.zeros(vocab), lambda: np.full(vocab, LOWEST[kind]), lambda: late(2000, 3.0, 1.0), lambda: late(30, 3.0, LOWEST[kind]),
            lambda: rng.standard_normal(vocab) * 100, lambda: with_one(np.nan, vocab - 1), lambda: with_one(np.inf, vocab - 3000), lambda: np.where(at // 1024 % 8 == 3, rng.random(vocab) * 5 - 60, -np.inf),
            lambda: (at % 509) / 64.0, lambda: np.where(at // 1024 % 2 == 1, 0.5, -0.5), lambda: np.where(at < 9000, -500.0, rng.standard_normal(vocab)), lambda: np.full(vocab, -np.inf),
            lambda: np.where(at // 1024 % 8 == 5, 80.0, 0.0) + rng.random(vocab), lambda: np.floor(rng.random(vocab) * 4) - 2, lambda: np.minimum(at // 1024, 37) * 1.0]
    one = [R.rounded(np.asarray(m(), np.float32), kind) for m in make]
    x = np.stack([one[r // 2 % len(one)] if r // 2 < 2 * len(one) else one[rng.integers(len(one))] for r in range(rows)])
    cum = -np.float32(3) * rng.random(rows).astype(np.float32)
    cum[:rows // 2] = 0  # pairs of equal rows first: of equal scores the lower row's, then its lower tokens
    sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev))
    p.sync()
    assert_near(sel, R.select_many(x, beams, k, cum), x, cum)


@pytest.mark.parametrize("kind", KINDS)
def test_equal_rows_wherever_they_begin(dev, p, kind):  # noqa: F811
    """rows on every alignment, NaN beside them: equal rows have equal scores, the lower row's come first"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(6)
    rows, vocab, pitch, beams, k = 2100, 5001, 5003, 5, 12
    assert tiles(rows, vocab) == 4
    x = np.repeat(logits(rng, rows // beams, vocab, kind), beams, 0)
    wide = np.full((rows, pitch), np.nan, np.float32)
    wide[:, :vocab] = x
    base = up(wide, kind, dev)
    view = ag.RowsGPU(base.data, dev, (rows, vocab), kind, (pitch, 1))
    sel = ag.select_beams_op(view, beams, k, p)
    p.sync()
    want = R.select_many(x, beams, k)
    assert want[1][0, :beams].tolist() == list(range(beams))
    assert_selection(sel, want)


@pytest.mark.parametrize("rows,vocab", [(12, 999), (12, 4099), (2100, 4001)])
@pytest.mark.parametrize("kind", KINDS)
def test_one_mask_for_all_rows(dev, p, kind, rows, vocab):  # noqa: F811
    """a bitmap of one row's tokens: log-sums, scores, parents, order — a vocabulary that is no multiple of 64, and the bitmap's length that or a multiple"""
    import arrow_gpu_amd as ag

    rng = np.random.default_rng(vocab)
    beams, k = 6, 10
    x = logits(rng, rows, vocab, kind)
    allowed = np.zeros((vocab + 63) // 64 * 64, bool)
    allowed[:vocab] = rng.random(vocab) < 0.3
    x[:, ~allowed[:vocab]] = np.inf
    cum = -np.float32(5) * rng.random(rows).astype(np.float32)
    want = R.select_many(x, beams, k, cum, allowed[:vocab])
    assert np.isfinite(want[0]).all()
    for mask in (allowed, allowed[:vocab]):
        sel = ag.select_beams_op(up(x, kind, dev), beams, k, p, scores=f32(cum, dev), allowed=bits(mask, dev))
        p.sync()
        assert_selection(sel, want)

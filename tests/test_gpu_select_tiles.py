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

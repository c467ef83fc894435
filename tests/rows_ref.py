"""The row operators' definitions in plain numpy (include/arrow_gpu.h "rows"): what the kernels are held to.  Factors are f32 by definition; sums,
products and scores in 64 bits."""
from __future__ import annotations

import numpy as np

TOP = {"i8": np.float32(127), "e4m3": np.float32(448), "i4": np.float32(15)}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}  # a rounding's largest relative error
NO_ROW = 0xFFFFFFFF


def e4m3_values() -> np.ndarray:
    """The 256 values of the 8-bit type."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, np.ldexp(1 + m / 8, e - 7), np.ldexp(m, -9)) * np.where(c & 128, -1.0, 1.0)
    return np.where((c & 127) == 127, np.nan, v)


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Codes of the values nearest to x (finite, |x| <= 464), ties to the even code: by search in the table of non-negative values."""
    v = e4m3_values()[:127]
    a = np.abs(x.astype(np.float64))
    hi = np.clip(np.searchsorted(v, a), 1, 126)
    lo = hi - 1
    up, down = v[hi] - a, a - v[lo]
    c = np.where(up < down, hi, np.where(down < up, lo, np.where(lo % 2 == 0, lo, hi)))
    return (c | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def quantise(x: np.ndarray, code: str, group: int):
    """x f32 [n, heads, dim] → (codes as stored, scales as stored)."""
    n, h, d = x.shape
    v = np.ascontiguousarray(x, dtype=np.float32).reshape(n, h, d // group, group)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(v).all(-1)
        lo = np.where(bad, 0, v.min(-1)).astype(np.float32) if code == "i4" else np.zeros(v.shape[:-1], np.float32)
        span = (v.max(-1) - lo).astype(np.float32) if code == "i4" else np.abs(v).max(-1)
        bad |= ~np.isfinite(span)
        live = ~bad & (span >= TOP[code] * np.float32(2.0**-126))
        inv = np.where(live, TOP[code] / np.where(live, span, 1), 0).astype(np.float32)
        scale = np.where(bad, np.nan, np.where(live, span / TOP[code], 0)).astype(np.float32)
        y = np.where(bad[..., None], 0, (v - lo[..., None]).astype(np.float32))
    if code == "e4m3":
        return to_e4m3((y * inv[..., None]).astype(np.float32)).reshape(n, h, d), scale
    q = np.rint(y.astype(np.float64) * inv[..., None].astype(np.float64)).astype(np.int8).reshape(n, h, d)
    if code == "i8":
        return q.view(np.uint8), scale
    q = q.view(np.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), np.stack([scale, lo], -1)


def values(codes: np.ndarray, scales: np.ndarray, code: str, group: int) -> np.ndarray:
    """What the codes stand for, in 64 bits."""
    n, h = codes.shape[:2]
    s = scales.astype(np.float64)
    if code == "i4":
        q = np.empty(codes.shape[:2] + (2 * codes.shape[2],))
        q[..., 0::2], q[..., 1::2] = codes & 15, codes >> 4
        v = q.reshape(n, h, -1, group) * s[..., :1] + s[..., 1:]
    else:
        q = codes.view(np.int8).astype(np.float64) if code == "i8" else e4m3_values()[codes]
        v = q.reshape(n, h, -1, group) * s[..., None]
    return v.reshape(n, h, -1)


def rounded(x: np.ndarray, kind: str) -> np.ndarray:
    """f32 values that an array of `kind` can hold."""
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if kind == "bf16":
        b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
        return np.where(np.isnan(x), np.float32(np.nan), (((b + 0x7FFF + ((b >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32))
    return x.astype(np.float32)


def slots_of(tables, page_rows, offsets, n, n_slots, first=None):
    """Per row its slot, -1 for none, -2 for one out of range."""
    got = np.full(n, -1, np.int64)
    for s in range(len(offsets) - 1):
        for i in range(int(offsets[s]), min(int(offsets[s + 1]), n)):
            t = i - int(offsets[s]) + (int(first[s]) if first is not None else 0)
            if t // page_rows >= tables.shape[1]:
                got[i] = -2
            elif tables[s, t // page_rows] == NO_ROW:
                got[i] = -1
            else:
                at = int(tables[s, t // page_rows]) * page_rows + t % page_rows
                got[i] = at if at < n_slots else -2
    return got


def select(x, beams, k, scores=None, allowed=None, finished=None, end_token=0):
    """x f64 [rows, vocab] → (scores f64, parents, tokens) [batch, k]."""
    rows, vocab = x.shape
    out_s, out_p, out_t = [], [], []
    for b in range(rows // beams):
        s, r, l, t = [], [], [], []
        for row in range(b * beams, (b + 1) * beams):
            cum = 0.0 if scores is None else float(scores[row])
            if finished is not None and finished[row]:
                if not np.isnan(cum):
                    s.append(np.array([cum])), r.append(np.array([row])), l.append(np.zeros(1)), t.append(np.array([end_token]))
                continue
            v = x[row] if allowed is None else np.where(allowed[row], x[row], -np.inf)
            if np.isnan(v).any() or not np.isfinite(v.max()):
                continue
            m = v.max()
            lse = m + np.log(np.exp(v - m).sum())
            s.append(cum + (v - lse)), r.append(np.full(vocab, row)), l.append(v), t.append(np.arange(vocab))
        s, r, l, t = (np.concatenate(z) if z else np.zeros(0) for z in (s, r, l, t))
        live = s > -np.inf  # (NaN: not)
        s, r, l, t = s[live], r[live].astype(np.int64), l[live], t[live].astype(np.int64)
        order = np.lexsort((t, -l, r, -s))[:k]
        s, r, t = s[order], r[order], t[order]
        have, at = {(a - b * beams) * vocab + c for a, c in zip(r.tolist(), t.tolist())}, 0
        s, r, t = s.tolist(), r.tolist(), t.tolist()
        while len(s) < k:
            if at not in have:
                s.append(-np.inf), r.append(b * beams + at // vocab), t.append(at % vocab)
            at += 1
        out_s.append(s), out_p.append(r), out_t.append(t)
    return np.array(out_s), np.array(out_p, np.int64), np.array(out_t, np.int64)


def select_many(x, beams, k, scores=None, allowed=None, finished=None, end_token=0):
    """select() for large inputs: of every row only the k tokens that can be chosen are sorted, a block of rows at a time.  x [rows, vocab] of any float type."""
    rows, vocab = x.shape
    out = [[], [], []]
    block = max(1, (1 << 23) // (beams * vocab)) * beams
    for r0 in range(0, rows, block):
        v = x[r0:r0 + block].astype(np.float64)
        n, each = v.shape[0], min(k, vocab)
        if allowed is not None:
            v = np.where(allowed if allowed.ndim == 1 else allowed[r0:r0 + block], v, -np.inf)
        done = np.zeros(n, bool) if finished is None else np.asarray(finished[r0:r0 + block], bool)
        cum = np.zeros(n) if scores is None else scores[r0:r0 + block].astype(np.float64)
        with np.errstate(all="ignore"):
            m = v.max(-1, keepdims=True)
            lse = (m + np.log(np.exp(v - m).sum(-1, keepdims=True)))[:, 0]
            lse[~np.isfinite(m[:, 0])] = np.nan  # a NaN, +infinity or nothing
            border = np.partition(v, vocab - each, -1)[:, vocab - each, None]
            above, equal = v > border, v == border
            take = above | (equal & (np.cumsum(equal, -1) <= each - above.sum(-1, keepdims=True)))
            row, token = np.nonzero(take)
            logit = v[row, token]
            score = cum[row] + (logit - lse[row])
        live = (score > -np.inf) & ~done[row]
        ends = np.nonzero(done & (cum > -np.inf))[0]
        row, token = np.concatenate([row[live], ends]), np.concatenate([token[live], np.full(len(ends), end_token)])
        logit, score = np.concatenate([logit[live], np.zeros(len(ends))]), np.concatenate([score[live], cum[ends]])
        order = np.lexsort((token, -logit, row, -score, row // beams))
        row, token, score = row[order], token[order], score[order]
        first = np.searchsorted(row // beams, np.arange(n // beams + 1))
        for b in range(n // beams):
            at = slice(first[b], min(first[b] + k, first[b + 1]))
            s, r, t = score[at].tolist(), (row[at] + r0).tolist(), token[at].tolist()
            have, f = {(p - r0 - b * beams) * vocab + q for p, q in zip(r, t)}, 0
            while len(s) < k:
                if f not in have:
                    s.append(-np.inf), r.append(r0 + b * beams + f // vocab), t.append(f % vocab)
                f += 1
            out[0].append(s), out[1].append(r), out[2].append(t)
    return np.array(out[0]), np.array(out[1], np.int64), np.array(out[2], np.int64)

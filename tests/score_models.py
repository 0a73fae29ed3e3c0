"""numpy statements of the 4-bit cache, of attention with shaped scores and of log probabilities, in 64 bits (no code of the package)."""
from __future__ import annotations

import numpy as np

import kv_models as M

ULP = 2.0 ** -24             # half a step of fp32, relative to the value
KINDS = ("f16", "q8", "q4")


def part_bytes(kind: str, dim: int, page: int) -> int:
    return page * dim // 2 + page * dim // 16 if kind == "q4" else M.part_bytes(kind == "q8", dim, page)


def fours_at(which: int, dim: int, page: int):
    """(byte, shift) of every token's and element's four bits in a part of keys (0) or values (1)."""
    token, element = np.arange(page)[:, None], np.arange(dim)[None]
    if which == 0:
        return token * (dim // 2) + element // 2, np.broadcast_to(element % 2 * 4, (page, dim))
    return (token // 4 * (dim // 4) + element // 4) * 8 + token % 4 * 2 + element % 4 // 2, np.broadcast_to(element % 2 * 4, (page, dim))


def decode_pool(raw: np.ndarray, kind: str, pages: int, heads: int, dim: int, page: int) -> np.ndarray:
    """[2][pages][heads][page][dim] in float64 of a cache's bytes."""
    if kind != "q4":
        return M.decode_pool(raw, kind == "q8", pages, heads, dim, page)
    raw = np.ascontiguousarray(raw, np.uint8).reshape(2, pages, heads, part_bytes(kind, dim, page))
    d = raw[..., page * dim // 2:].copy().view(np.float16).reshape(2, pages, heads, dim // 32, page).astype(np.float64)
    d = np.repeat(np.swapaxes(d, -1, -2), 32, -1)
    out = np.empty((2, pages, heads, page, dim))
    for which in (0, 1):
        at, shift = fours_at(which, dim, page)
        with np.errstate(over="ignore", invalid="ignore"):
            out[which] = (((raw[which][..., at] >> shift.astype(np.uint8) & 15).astype(np.float64) - 8) * d[which]).astype(np.float16)
    return out


def encode_fours(x: np.ndarray):
    """(n, d, distance from the nearest border) of blocks of 32 of float64 values: n as if in unbounded precision."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        size = np.where(np.isnan(y), -1, np.abs(y))
        largest = np.take_along_axis(y, size.argmax(-1)[..., None], -1)
        largest = np.where(size.max(-1, keepdims=True) < 0, 0, largest)
        d = np.clip(largest * -0.125, -65504, 65504).astype(np.float16).astype(np.float64)
        t = np.where((d != 0) & ~np.isnan(y), y / d, 0)
        n = np.clip(np.rint(t), -8, 7) + 8
    return n.reshape(x.shape), d[..., 0], np.abs(np.abs(t - np.floor(t)) - 0.5).reshape(x.shape)


def random_pool(rng, kind, pages, heads, dim, page, spread=1.0):
    """A cache's bytes: normal values, or blocks of uniform numbers with scales of their own."""
    if kind == "f16":
        return (spread * rng.standard_normal((2, pages, heads, page * dim))).astype(np.float16).view(np.uint8).reshape(-1)
    codes = page * dim // (1 if kind == "q8" else 2)
    raw = rng.integers(0, 256, (2, pages, heads, part_bytes(kind, dim, page))).astype(np.uint8)
    if kind == "q8":
        raw[..., :codes] = np.where(raw[..., :codes] == 128, 0, raw[..., :codes])
    lo, hi = (0.004, 0.03) if kind == "q8" else (0.06, 0.4)
    d = spread * rng.uniform(lo, hi, (2, pages, heads, page * dim // 32))
    if kind == "q4":
        d *= rng.choice([-1, 1], d.shape)
    raw[..., codes:] = d.astype(np.float16).view(np.uint8).reshape(2, pages, heads, -1)
    return raw.reshape(-1)


def attend(pool, q, positions, requests_of, table, scale, window=0, cap=0.0, slopes=None, first=None, end=None):
    """(out, bound): attention in float64, and how far fp32 arithmetic may be off.

    An element is sum p v.  A score s = scale q.k is off by the rounding of the 2 dim products and sums of its two binary16
    parts, (2 dim + 8) half steps of scale * sum |q k|; a cap leaves that as it is at most, and its tanh, product and
    quotient add 2^-21 + 4 half steps of the score, 12 in all; the bias three half steps of itself (the distance, the
    slope's scaling, the product), and the two sums one of what is summed.  Weights are off by twice that (their own and
    the sum's) and the power's 8, the sums over n tokens by n + 64 half steps of sum p |v|.  And each by 2^-38 of the
    largest, whatever its own size: it is held 2^13 times as large as the largest is 1, as two binary16 parts, the smaller
    of which is off by up to 2^-25, half a step of binary16's subnormal numbers: what an
    element is where all larger weights meet values of 0."""
    _, pages, kv, page, dim = pool.shape
    rows, heads = q.shape[:2]
    out, bound = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    for i in range(rows):
        r = i if requests_of is None else int(requests_of[i])
        p = int(positions[i])
        if p < 0 or not 0 <= r < table.shape[0]:
            continue
        room = table.shape[1] * page
        stop = min(p + 1 if end is None else int(end[i]), room)
        begin = max(0, p - window + 1) if window else 0
        if first is not None:
            begin = max(begin, int(first[i]))
        j = np.arange(begin, max(stop, begin))
        at = table[r, j // page]
        ok = (at >= 0) & (at < pages)
        j, at = j[ok], at[ok]
        if not len(j):
            continue
        for h in range(heads):
            k, v = (pool[w, at, h // (heads // kv), j % page] for w in (0, 1))
            qh = q[i, h].astype(np.float64)
            s = scale * (k @ qh)
            off = (2 * dim + 8) * np.abs(scale) * (np.abs(k) @ np.abs(qh))
            if cap:
                s = cap * np.tanh(s / cap)
                off = off + 12 * np.abs(s)
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(p - j)
                off = off + 3 * np.abs(bias) + np.abs(s)
                s = s - bias
            off = off + 2 * (np.abs(s) + np.abs(s).min()) + 2 * np.abs(s.max()) if cap or slopes is not None else off
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ v
            size = w @ np.abs(v)
            bound[i, h] = ULP * ((w * off) @ np.abs(v) + (w @ off) * size + (16 + len(j) + 64) * size) + 2.0 ** -38 * w.max() * np.abs(v).sum(0)
    return out, bound


def logprobs(logits, scale=1.0, cap=0.0):
    """(log p, entropy) in float64 of rows of fp32 logits; -inf is left out whatever the cap."""
    x = logits.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if cap:
            x = np.where(np.isneginf(x), x, cap * np.tanh(x / cap))
        m = x.max(-1, keepdims=True)
        m = np.where(np.isneginf(m), 0, m)
        e = np.exp(scale * (x - m))
        total = e.sum(-1, keepdims=True)
        with np.errstate(divide="ignore"):
            logp = scale * (x - m) - np.where(total == 0, 0, np.log(total))
        p = e / np.where(total == 0, 1, total)
        entropy = -np.where(p > 0, p * np.where(p > 0, logp, 0), np.where(np.isnan(p), np.nan, 0)).sum(-1)
    return logp, entropy


def ranked(logits, top):
    """Tokens of the largest logits, the largest first, equal ones by their number; -1 where NaN leaves none."""
    x = np.where(np.isnan(logits), np.float32(0), logits) + np.float32(0)
    out = np.full((len(x), top), -1)
    for i, row in enumerate(x):
        order = np.lexsort((np.arange(len(row)), -row.astype(np.float64)))
        order = order[~np.isnan(logits[i][order])][:top]
        out[i, :len(order)] = order
    return out

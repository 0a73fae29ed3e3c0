"""numpy statements of the paged key-value cache and its operators, in 64 bits (no code of the package)."""
from __future__ import annotations

import numpy as np


def part_bytes(q8: bool, dim: int, page: int) -> int:
    return page * dim + page * dim // 16 if q8 else 2 * page * dim


def decode_pool(raw: np.ndarray, q8: bool, pages: int, heads: int, dim: int, page: int) -> np.ndarray:
    """[2][pages][heads][page][dim] in float64 of a cache's bytes."""
    raw = np.ascontiguousarray(raw, np.uint8).reshape(2, pages, heads, part_bytes(q8, dim, page))
    if not q8:
        return raw.view(np.float16).reshape(2, pages, heads, page, dim).astype(np.float64)
    quants = raw[..., :page * dim].copy().view(np.int8).reshape(2, pages, heads, page, dim // 32, 32).astype(np.float64)
    d = raw[..., page * dim:].copy().view(np.float16).reshape(2, pages, heads, dim // 32, page).astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        return (quants * np.swapaxes(d, -1, -2)[..., None]).astype(np.float16).astype(np.float64).reshape(2, pages, heads, page, dim)


def encode_blocks(x: np.ndarray):
    """(bytes, scales) of blocks of 32 of float64 values, and how near each byte came to its neighbour: the
    distance of x / d from the nearest half."""
    y = x.reshape(*x.shape[:-1], -1, 32)
    d = np.minimum(np.abs(y).max(-1) / 127, 65504).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        t = np.where(d[..., None] > 0, y / d[..., None], 0)
    return np.clip(np.rint(t), -127, 127).reshape(x.shape), d, np.abs(np.abs(t - np.floor(t)) - 0.5).reshape(x.shape)


def rotate(x: np.ndarray, positions: np.ndarray, frequencies: np.ndarray, halves: bool, norm=None, eps: float = 0.0) -> np.ndarray:
    """x [rows][heads][dim] normalised and turned, in float64."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    pairs = len(frequencies)
    out = x.copy()
    angle = positions.astype(np.float64)[:, None] * frequencies
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    first = np.arange(pairs) if halves else 2 * np.arange(pairs)
    second = first + pairs if halves else first + 1
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., first] * sin + x[..., second] * cos
    return out


def attend(pool: np.ndarray, q: np.ndarray, positions, requests_of, table: np.ndarray, scale: float, window: int = 0):
    """(out, slack): attention in float64 and, per output, sum p |v| and the largest scale * sum |q k| of its
    row and head -- what a rounding error of fp32 arithmetic is in proportion to."""
    _, pages, kv, page, dim = pool.shape
    rows, heads = q.shape[:2]
    out, weight = np.zeros((rows, heads, dim)), np.zeros((rows, heads, dim))
    reach = np.zeros((rows, heads))
    for i in range(rows):
        r = i if requests_of is None else int(requests_of[i])
        if positions[i] < 0 or not 0 <= r < table.shape[0]:
            continue
        end = min(int(positions[i]) + 1, table.shape[1] * page)
        begin = max(0, int(positions[i]) - window + 1) if window else 0
        j = np.arange(begin, end)
        at = table[r, j // page]
        ok = (at >= 0) & (at < pages)
        j, at = j[ok], at[ok]
        if not len(j):
            continue
        for h in range(heads):
            k, v = (pool[w, at, h // (heads // kv), j % page] for w in (0, 1))
            qh = q[i, h].astype(np.float64)
            s = scale * (k @ qh)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], weight[i, h] = p @ v, p @ np.abs(v)
            reach[i, h] = scale * (np.abs(k) @ np.abs(qh)).max()
    return out, weight, reach


def plan(past, fresh, pages: int, page: int, ring, free, table, max_rows: int):
    """The step's pages one request after the other; returns a dict of the call's results."""
    requests, stride = table.shape
    table, ring = table.copy(), ring.copy()
    head, count = (int(v) for v in free)
    if not (0 <= head < pages and 0 <= count <= pages):
        head = count = 0
    slots, positions, rows_of = (np.full(max_rows, -1, np.int64) for _ in range(3))
    lengths, starts = np.array(past, np.int64), [0]
    taken = asked = back = row = 0
    before = table.copy()
    for r in range(requests):
        p, f = int(past[r]), int(fresh[r])
        held = 0 <= p <= min(stride * page, 2**31 - 1)
        had = -(-p // page) if held else 0
        if f < 0:
            lengths[r] = 0
            for b in range(had):
                if back < pages - count:
                    ring[(head + count + back) % pages] = before[r, b]
                    back += 1
        f = max(f, 0)
        ok = held and row + f <= max_rows and p + f <= min(stride * page, 2**31 - 1)
        if ok and f:
            need = -(-(p + f) // page) - had
            asked += need
            ok = need == 0 or asked <= count
            if ok:
                for b in range(had, had + need):
                    table[r, b] = ring[(head + taken) % pages]
                    taken += 1
                lengths[r] = p + f
        for i in range(f):
            if row + i >= max_rows:
                break
            rows_of[row + i] = r
            if ok:
                positions[row + i] = p + i
                at = table[r, (p + i) // page]
                if 0 <= at < pages:
                    slots[row + i] = at * page + (p + i) % page
        row += f
        starts.append(min(row, max_rows))
    return {"lengths": lengths, "rowStarts": np.array(starts), "table": table, "pageRing": ring,
            "freePages": np.array([(head + taken) % pages, count - taken + back]), "slots": slots, "positions": positions,
            "rowRequests": rows_of}

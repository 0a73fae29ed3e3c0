"""The 4-bit cache and attention with capped, biased and masked scores on the GPU, against numpy in 64 bits."""
import numpy as np
import pytest

import kv_models as M
import score_models as S
import test_gpu_kv as K
from gpu_util import say

pytestmark = pytest.mark.gpu

HALF, ULP = 2.0 ** -11, 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    from jitllm_amd.runtime import Context
    c = Context(0)
    yield c
    c.close()


def kv_type(kind):
    from jitllm_amd.attention import KvType
    return {"f16": KvType.F16, "q8": KvType.Q8_0, "q4": KvType.Q4_0}[kind]


def cache_of(ctx, kind, pages, heads, dim, page, raw):
    from jitllm_amd.attention import PagedKvCache
    memory = ctx.raw_buffer(raw.nbytes)
    memory.upload(raw)
    return PagedKvCache(ctx, kv_type(kind), pages, heads, dim, page, memory=memory)


def pool_of(cache, kind):
    raw = cache.memory.download(np.uint8, cache.nbytes)
    return S.decode_pool(raw, kind, cache.pages, cache.kvHeads, cache.headDim, cache.pageTokens)


# ---- the 4-bit cache: written, read --------------------------------------------------------------

APPENDS = [
    # rows, heads, kv, dim, page, halves, turned, norm, context
    (1, 32, 8, 64, 16, False, 64, False, 1000), (1, 14, 2, 64, 16, True, 64, False, 5), (3, 28, 4, 128, 32, True, 128, False, 131072),
    (64, 32, 8, 128, 32, True, 128, True, 8192), (65, 5, 5, 96, 16, False, 96, True, 700), (33, 3, 1, 96, 64, True, 48, True, 900),
    (17, 8, 2, 192, 128, True, 96, False, 100000), (40, 16, 4, 256, 16, False, 256, True, 4096), (7, 71, 1, 64, 256, False, 32, False, 60),
    (300, 4, 2, 128, 64, False, 128, False, 2000000), (20, 8, 8, 128, 16, False, 0, False, 50), (9, 0, 4, 128, 16, True, 64, True, 77)]


@pytest.mark.parametrize("rows,heads,kv,dim,page,halves,turned,norm,context", APPENDS)
def test_append_fours(ctx, rows, heads, kv, dim, page, halves, turned, norm, context):
    say("append fours", rows, heads, kv, dim, page, halves, turned, norm, context)
    rng = np.random.default_rng(rows + dim + page)
    pages = rows // page + 3
    x = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float32)
    x[:, :, 3] *= 20                                           # a channel that stands out, as keys have
    x[rows // 2, heads + 2 * kv - 1, :32] = 0                  # a block of zeros
    raw = S.random_pool(rng, "q4", pages, kv, dim, page)
    cache = cache_of(ctx, "q4", pages, kv, dim, page, raw)
    slots = rng.permutation(pages * page)[:rows]
    positions = rng.integers(0, context, rows)
    freq = 500000.0 ** (-np.arange(0, turned, 2) / turned) if turned else np.zeros(0)
    qn, kn = (1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)) if norm else (None, None)
    if rows > 2:
        slots[1], positions[2] = -1, -1                        # no page; no token at all
    if rows > 3:
        slots[3] = pages * page                                # a slot behind the cache's last
    apart = rows % 2 == 1
    got = K.run_append(ctx, cache, x, heads, kv, dim, positions, slots, freq, halves, qn, kn, 1e-6, apart=apart, pad=0 if apart else 8)
    before, after = S.decode_pool(raw, "q4", pages, kv, dim, page), pool_of(cache, "q4")
    live = positions >= 0
    # what comes in front of the rounding to fp32 is in double precision: half a step of it, and a thousandth for the sums
    step = 1.001 * ULP
    if heads:
        q = M.rotate(x[:, :heads], np.maximum(positions, 0), freq, halves, qn, 1e-6)
        assert (np.abs(got - q) <= step * np.abs(q) + 1e-9 * np.abs(q).max(-1, keepdims=True))[live].all()
    k = M.rotate(x[:, heads:heads + kv], np.maximum(positions, 0), freq, halves, kn, 1e-6)
    written = np.zeros((pages, page), bool)
    for which, y in ((0, k.astype(np.float32).astype(np.float64)), (1, x[:, heads + kv:].astype(np.float64))):
        n, d, border = S.encode_fours(y)
        want = ((n - 8) * np.repeat(d, 32, -1)).astype(np.float16).astype(np.float64)
        for i in range(rows):
            if not live[i] or not 0 <= slots[i] < pages * page:
                continue
            written[slots[i] // page, slots[i] % page] = True
            at = after[which, slots[i] // page, :, slots[i] % page]
            if which == 1:                                     # nothing but copies in front of it: the same but where the
                sure = border[i] > 1e-6                        # fp32 quotient may fall on the other side of a border
                assert np.array_equal(at[sure], want[i][sure])
            # half a step of the block's scale; the largest value's neighbours on the other side end at 7 of 8, half a step
            # more; the scale and the value are rounded to binary16
            assert (np.abs(at - y[i]) <= np.repeat(np.abs(d[i]), 32, -1) * (1 + 8 * HALF) + 2 * HALF * np.abs(y[i]) + 2.0 ** -24).all()
            inside = np.abs(n[i] - 8) < 7
            assert (np.abs(at - y[i]) <= np.repeat(np.abs(d[i]), 32, -1) * (0.5 + 8 * HALF) + 2 * HALF * np.abs(y[i]) + 2.0 ** -24)[inside].all()
    keep = np.broadcast_to(~written[None, :, None, :, None], after.shape)
    assert np.array_equal(after[keep], before[keep])


def test_append_fours_special_values(ctx):
    """Infinities, NaN, values past binary16, values below its smallest, equal largest ones of both signs."""
    dim, page = 64, 16
    x = np.zeros((8, 3, dim), np.float32)
    x[0, 2, :] = 1e6
    x[1, 2, :] = np.nan
    x[2, 2, 0], x[2, 2, 1], x[2, 2, 2] = np.inf, -np.inf, 5
    x[3, 2, :] = 1e-9
    x[4, 2, :32], x[4, 2, 5] = 2, np.nan
    x[5, 2, :] = np.linspace(-1e38, 1e38, dim)
    x[6, 2, 9], x[6, 2, 17], x[6, 2, 18] = 4, -4, 1            # the first of the largest is the one that d goes by
    x[7, 2, 17], x[7, 2, 9], x[7, 2, 18] = 4, -4, 1
    cache = cache_of(ctx, "q4", 2, 1, dim, page, np.zeros(2 * 2 * S.part_bytes("q4", dim, page), np.uint8))
    say("append fours special")
    K.run_append(ctx, cache, x, 1, 1, dim, np.zeros(8, int), np.arange(8), np.zeros(0), False, None, None, 0.0)
    v = pool_of(cache, "q4")[1, 0, 0]
    assert (v[0] == np.inf).all()                               # -65504 x -8, beyond binary16
    assert (v[1] == 0).all()                                    # nothing but NaN: a scale of 0
    assert v[2, 0] == np.inf and v[2, 1] == -np.inf and v[2, 2] == 0
    assert (v[3] == 0).all()
    assert v[4, 5] == 0 and np.array_equal(np.delete(v[4, :32], 5), np.full(31, 2.0))
    assert np.isinf(v[5][[0, -1]]).all()
    assert v[6, 9] == 4 and v[6, 17] == -3.5 and v[6, 18] == 1
    assert v[7, 9] == -4 and v[7, 17] == 3.5 and v[7, 18] == 1


@pytest.mark.parametrize("dim,kv,page", [(64, 3, 16), (96, 2, 256), (128, 8, 32), (192, 1, 64), (256, 5, 128)])
def test_read_fours(ctx, dim, kv, page):
    say("read fours", dim, kv, page)
    rng = np.random.default_rng(dim)
    pages, rows = 5, 23
    raw = S.random_pool(rng, "q4", pages, kv, dim, page)
    cache = cache_of(ctx, "q4", pages, kv, dim, page, raw)
    slots = rng.integers(0, pages * page, rows)
    slots[4], slots[9], slots[11] = -1, pages * page, 2**31 - 1
    pool = S.decode_pool(raw, "q4", pages, kv, dim, page)
    ok = (slots >= 0) & (slots < pages * page)
    at = np.where(ok, slots, 0)
    for make in (ctx.half_array, ctx.float_array):
        k, v = make(rows * kv * dim), make(rows * kv * dim)
        cache.read(K.ints(ctx, slots), rows, k, v)
        ctx.sync()
        for which, a in enumerate((k, v)):
            want = np.where(ok[:, None, None], pool[which, at // page, :, at % page], 0)
            assert np.array_equal(a.get().astype(np.float64).reshape(rows, kv, dim), want)


# ---- attention -----------------------------------------------------------------------------------

def run(ctx, cache, q, positions, requests_of, table, window=0, half=False, pad=0, cap=0.0, slopes=None, first=None, end=None, scale=None,
        attention=None):
    from jitllm_amd.attention import PagedAttention, Rows
    rows, heads, dim = q.shape
    attention = attention or PagedAttention(ctx, rows, heads, cache.kvHeads, dim)
    stride = heads * dim + pad
    flat = np.full((rows, stride), np.nan, np.float32)
    flat[:, :heads * dim] = q.reshape(rows, -1)
    out = (ctx.half_from_numpy if half else ctx.from_numpy)(np.full((rows + 2) * stride, -5.5))
    qa = ctx.from_numpy(flat)
    ints = lambda x: None if x is None else K.ints(ctx, x)      # noqa: E731
    attention.attend(cache, Rows(qa, stride), rows, ints(positions), ints(table), Rows(out, stride), requests=table.shape[0],
                     rowRequests=ints(requests_of), scale=scale, window=window, cap=cap,
                     slopes=None if slopes is None else ctx.from_numpy(slopes), firstTokens=ints(first), endTokens=ints(end))
    ctx.sync()
    got = out.get().reshape(rows + 2, stride)
    assert (got[rows:] == -5.5).all() and (got[:, heads * dim:] == -5.5).all()   # rows behind, columns between
    return got[:rows, :heads * dim].astype(np.float64).reshape(rows, heads, dim)


def check(got, want, bound, half=False):
    """Each element within its bound; all together within a hundredth of the bounds' sum, or 2e-6 of their norm: roundings
    are of either sign, and one operand rounded to binary16 would pass that ten times over."""
    assert np.isfinite(got).all()
    each = bound + (HALF * np.abs(want) + 2.0 ** -25 if half else 0)
    assert (np.abs(got - want) <= each).all(), np.max(np.abs(got - want) / np.maximum(each, 1e-300))
    if not half:
        assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want) + 0.01 * np.linalg.norm(bound) + 1e-12


FOURS = [
    # lengths, heads, kv, dim, page, window, half
    ([201], 32, 8, 64, 16, 0, False), ([1], 14, 2, 64, 16, 0, True), ([1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 65], 4, 2, 128, 16, 0, False),
    ([127, 128, 129, 255, 256, 257, 1000], 28, 4, 128, 32, 0, False), ([950, 3, 511, 512, 513], 6, 6, 128, 16, 0, True),
    ([4096], 16, 4, 256, 16, 1024, False), ([700, 40, 90], 16, 4, 256, 64, 100, False), ([333, 1, 77], 9, 3, 96, 16, 0, False),
    ([1300, 64], 3, 3, 96, 128, 1, False), ([260, 511], 24, 2, 192, 256, 0, True), ([900, 5], 12, 2, 192, 16, 17, False),
    ([2000, 7], 71, 1, 64, 32, 0, False), ([129], 48, 1, 128, 16, 0, True), ([9000], 32, 8, 128, 64, 0, False),
    ([5000, 1, 300], 8, 8, 64, 16, 0, False), ([40, 3], 300, 300, 256, 16, 0, False)]


@pytest.mark.parametrize("lengths,heads,kv,dim,page,window,half", FOURS)
def test_attend_over_fours(ctx, lengths, heads, kv, dim, page, window, half):
    say("attend fours", lengths, heads, kv, dim, page, window, half)
    rng = np.random.default_rng(sum(lengths) + dim)
    rows = len(lengths)
    table, pages = K.make_tables(rng, lengths, page)
    raw = S.random_pool(rng, "q4", pages, kv, dim, page)
    cache = cache_of(ctx, "q4", pages, kv, dim, page, raw)
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    positions = np.array(lengths) - 1
    got = run(ctx, cache, q, positions, None, table, window, half, pad=8 if rows > 1 else 0)
    check(got, *S.attend(S.decode_pool(raw, "q4", pages, kv, dim, page), q, positions, None, table, dim ** -0.5, window), half)


@pytest.mark.parametrize("rows,longest,heads,kv,dim", [(70, 400, 8, 2, 64), (300, 60, 4, 4, 128), (1030, 20, 4, 1, 64), (40, 3000, 7, 1, 128)])
def test_attend_over_fours_ragged(ctx, rows, longest, heads, kv, dim):
    say("attend fours ragged", rows, longest, heads, kv, dim)
    rng = np.random.default_rng(rows)
    page = 16
    lengths = (longest * rng.random(rows) ** 2).astype(int)
    lengths[rng.integers(0, rows)] = longest
    requests = rows + 5
    requests_of = rng.permutation(requests)[:rows]
    table, pages = K.make_tables(rng, lengths, page, requests_of, requests)
    raw = S.random_pool(rng, "q4", pages, kv, dim, page)
    cache = cache_of(ctx, "q4", pages, kv, dim, page, raw)
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    got = run(ctx, cache, q, lengths - 1, requests_of, table)
    check(got, *S.attend(S.decode_pool(raw, "q4", pages, kv, dim, page), q, lengths - 1, requests_of, table, dim ** -0.5))
    assert (got[lengths == 0] == 0).all()


def documents_of(rng, positions, requests_of, most):
    """The first token of each row's document, documents of a random length beginning where they do in each request."""
    starts = {r: np.unique(np.concatenate([[0], rng.integers(0, max(int(n), 1), 1 + int(n) // 40)])) for r, n in enumerate(most)}
    return np.array([starts[r][np.searchsorted(starts[r], max(p, 0), side="right") - 1] if r in starts else 0 for p, r in zip(positions, requests_of)])


SCORED = [
    # runs (request, first position, rows), requests, heads, kv, dim, page, kind, window, half, cap, slopes, documents, prefix
    ([(0, 200, 1)], 1, 32, 8, 64, 16, "f16", 0, False, 30.0, False, False, 0), ([(0, 0, 1)], 1, 4, 2, 128, 16, "q4", 0, False, 0.0, True, False, 0),
    ([(0, 3000, 1), (1, 17, 1), (2, 511, 1)], 3, 16, 8, 256, 16, "f16", 0, False, 50.0, False, False, 0),
    ([(r, 90 * r, 1) for r in range(11)], 11, 8, 8, 128, 32, "f16", 0, True, 0.0, True, False, 0),
    ([(r, 90 * r, 1) for r in range(11)], 11, 28, 4, 96, 16, "q8", 200, False, 20.0, True, False, 0),
    ([(0, 5000, 1)], 1, 12, 2, 192, 64, "q4", 0, True, 4.0, True, False, 0), ([(0, 0, 300)], 1, 8, 2, 64, 16, "f16", 0, False, 0.0, False, True, 0),
    ([(0, 0, 257)], 1, 4, 4, 128, 64, "q4", 0, False, 0.0, False, False, 130), ([(0, 0, 150), (1, 0, 77)], 2, 6, 2, 96, 16, "q8", 0, True, 30.0, False, False, 64),
    ([(0, 700, 40), (1, 0, 5), (2, 33, 64)], 3, 16, 1, 64, 32, "f16", 50, False, 10.0, True, True, 0),
    ([(0, 0, 130), (1, 100, 65), (-1, 3, 5)], 2, 16, 4, 256, 16, "q4", 0, False, 50.0, False, True, 120),
    ([(0, 40, 17)], 1, 9, 1, 128, 16, "q8", 0, False, 0.0, True, False, 0), ([(0, 0, 200)], 1, 2, 1, 192, 128, "f16", 0, False, 0.0, True, True, 0),
    ([(0, 0, 5), (1, 7, 2)], 2, 600, 600, 64, 16, "f16", 0, False, 30.0, False, False, 4), ([(0, 0, 40)], 1, 40, 1, 64, 16, "q4", 0, False, 30.0, True, False, 0)]


@pytest.mark.parametrize("runs,requests,heads,kv,dim,page,kind,window,half,cap,slopes,documents,prefix", SCORED)
def test_attend_scored(ctx, runs, requests, heads, kv, dim, page, kind, window, half, cap, slopes, documents, prefix):
    """Rows that decode, prompts, both; each with what its own call asks for; and the rows in another order."""
    say("attend scored", runs[:4], heads, kv, dim, page, kind, window, half, cap, slopes, documents, prefix)
    rng = np.random.default_rng(len(runs) + dim + heads)
    requests_of = np.concatenate([np.full(n, r) for r, _, n in runs])
    positions = np.concatenate([np.arange(first, first + n) for _, first, n in runs])
    real = (requests_of >= 0) & (requests_of < requests)
    most = np.ones(requests, int)
    np.maximum.at(most, requests_of[real], positions[real] + 1)
    table, pages = K.make_tables(rng, most, page)
    raw = S.random_pool(rng, kind, pages, kv, dim, page)
    cache = cache_of(ctx, kind, pages, kv, dim, page, raw)
    pool = S.decode_pool(raw, kind, pages, kv, dim, page)
    first = documents_of(rng, positions, requests_of, most) if documents else None
    end = np.maximum(positions + 1, np.minimum(prefix, np.where(real, most[np.clip(requests_of, 0, requests - 1)], 0))) if prefix else None
    m = (2.0 ** (-8 * np.arange(1, heads + 1) / heads)).astype(np.float32) if slopes else None
    if len(positions) > 30:
        positions[rng.random(len(positions)) < 0.05] = -1
    for turn in range(2):
        q = (5 * rng.standard_normal((len(positions), heads, dim))).astype(np.float32)
        got = run(ctx, cache, q, positions, requests_of, table, window, half, 8, cap, m, first, end)
        check(got, *S.attend(pool, q, positions, requests_of, table, dim ** -0.5, window, cap, m, first, end), half)
        assert (got[~real | (positions < 0)] == 0).all()
        positions, requests_of, real = positions[::-1].copy(), requests_of[::-1].copy(), real[::-1].copy()
        first, end = (None if x is None else x[::-1].copy() for x in (first, end))


PROMPTS = [
    # enough rows that they go in blocks: of one request, of several of odd lengths, beside rows that decode over long and short
    # contexts, beside rows of nothing
    ([(0, 0, 1400)], 1, 8, 2, 64, 16, "q4", 0, False, 0.0, False, False, 0), ([(0, 0, 500), (1, 900, 333), (2, 3, 70)], 3, 12, 4, 96, 16, "f16", 0, True, 20.0, True, True, 0),
    ([(0, 0, 300)] + [(1 + r, 1000 + 13 * r, 1) for r in range(40)] + [(41, 40, 35)], 42, 32, 8, 128, 32, "q8", 0, False, 30.0, False, False, 100),
    ([(0, 0, 300)] + [(1 + r, 1000 + 13 * r, 1) for r in range(40)] + [(-1, 5, 30)], 41, 32, 8, 64, 64, "q4", 0, False, 0.0, False, False, 0),
    ([(r, 11 * r, 9) for r in range(60)], 60, 16, 8, 64, 16, "f16", 0, False, 0.0, True, False, 0), ([(0, 50, 620)], 1, 7, 7, 128, 16, "q4", 200, True, 5.0, False, False, 0),
    ([(0, 0, 330), (1, 700, 90)], 2, 14, 7, 192, 16, "q8", 0, False, 0.0, False, True, 0), ([(0, 0, 130), (1, 0, 75)], 2, 48, 16, 256, 32, "f16", 64, False, 50.0, False, False, 40),
    ([(0, 0, 90)], 1, 96, 4, 256, 16, "q4", 0, False, 0.0, True, False, 60), ([(0, 10, 1300), (-1, 0, 2400), (1, 0, 400)], 2, 32, 1, 64, 16, "f16", 30, False, 0.0, True, False, 0),
    # ... and enough that there are several workgroups to a compute unit
    ([(0, 0, 500), (1, 300, 250)], 2, 32, 8, 128, 16, "q4", 0, False, 30.0, False, False, 64), ([(0, 0, 300), (1, 700, 333), (2, 3, 70)], 3, 24, 8, 96, 16, "q8", 100, True, 20.0, True, True, 0),
    ([(0, 0, 1100)], 1, 16, 8, 64, 32, "q8", 0, False, 0.0, False, False, 0), ([(0, 50, 520), (-1, 5, 30), (1, 0, 90)], 2, 28, 7, 128, 16, "f16", 0, False, 8.0, True, False, 0),
    ([(0, 0, 300), (1, 60, 120)], 2, 48, 12, 96, 16, "f16", 70, False, 0.0, False, True, 0), ([(0, 0, 600)], 1, 32, 16, 96, 64, "q4", 0, True, 0.0, False, False, 0),
    ([(0, 0, 2100)], 1, 8, 4, 64, 16, "q8", 0, False, 25.0, False, False, 100), ([(0, 30, 2050)], 1, 8, 4, 128, 64, "q4", 0, True, 0.0, False, False, 0),
    ([(0, 9, 600), (1, 0, 50)], 2, 32, 16, 64, 16, "q4", 0, False, 50.0, True, False, 0), ([(0, 0, 560)], 1, 32, 8, 128, 128, "q8", 0, False, 0.0, True, False, 30)]


@pytest.mark.parametrize("runs,requests,heads,kv,dim,page,kind,window,half,cap,slopes,documents,prefix", PROMPTS)
def test_attend_prompts(ctx, runs, requests, heads, kv, dim, page, kind, window, half, cap, slopes, documents, prefix):
    test_attend_scored(ctx, runs, requests, heads, kv, dim, page, kind, window, half, cap, slopes, documents, prefix)


@pytest.mark.parametrize("kind,kv", [(kind, kv) for kv in (4, 8) for kind in S.KINDS])
def test_attend_prompts_of_values_that_are_not_finite(ctx, kind, kv):
    """Infinities, NaN and, in four bits, a scale that takes its multiples past binary16, at tokens that some rows of a block
    see: those may get NaN, the others are what they are without; and pages outside the cache."""
    rng = np.random.default_rng(21)
    heads, dim, page, rows = kv, 64, 16, 3000
    table, pages = K.make_tables(rng, [rows], page)
    table[0, 7], table[0, 100] = -1, pages
    raw = S.random_pool(rng, kind, pages, kv, dim, page)
    bad_tokens = [37, 640, 1001, 2999]
    dirty = raw.reshape(2, pages, kv, -1).copy()
    for t, bad in zip(bad_tokens, (np.inf, np.nan, 30000 if kind == "q4" else -np.inf, np.nan)):
        p, o = table[0, t // page], t % page
        if kind == "f16":
            dirty.view(np.float16).reshape(2, pages, kv, page, dim)[1, p, :, o, 5::7] = bad
        else:
            codes = page * dim // (1 if kind == "q8" else 2)
            scales = dirty[..., codes:].view(np.float16).reshape(2, pages, kv, dim // 32, page)
            scales[1, p, :, 1, o] = np.float16(bad)
            dirty[..., codes:] = scales.view(np.uint8).reshape(2, pages, kv, -1)
    cache = cache_of(ctx, kind, pages, kv, dim, page, dirty.reshape(-1))
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    positions, of = np.arange(rows), np.zeros(rows, int)
    say("attend prompts not finite", kind, kv)
    window = 20
    got = run(ctx, cache, q, positions, of, table, window, cap=20.0)
    hit = np.array([any(i - window < t <= i for t in bad_tokens) for i in range(rows)])
    want, bound = S.attend(S.decode_pool(raw, kind, pages, kv, dim, page), q, positions, of, table, dim ** -0.5, window, 20.0)
    check(got[~hit], want[~hit], bound[~hit])
    assert hit.sum() == 3 * window + 1 and not np.isfinite(got[hit]).all()


@pytest.mark.parametrize("rows_together", [False, True])
def test_attend_scored_ranges_that_leave_nothing(ctx, rows_together):
    """Ends before their beginnings, behind the table's last token, below 0; documents that begin behind the row."""
    rng = np.random.default_rng(3)
    heads, kv, dim, page = 4, 2, 64, 16
    first = np.array([0, 5, 60, 0, -7, 2**31 - 1, 3, 99, 0, 50])
    end = np.array([0, 5, 50, -3, 9, 40, 2**31 - 1, 100, -2**31, 51])
    positions = np.array([4, 4, 4, 4, 4, 4, 2**31 - 1, 4, 4, -1])
    rows = len(first)
    table, pages = K.make_tables(rng, [100] if rows_together else [100] * rows, page)
    requests_of = np.zeros(rows, int) if rows_together else np.arange(rows)
    for kind in S.KINDS:
        raw = S.random_pool(rng, kind, pages, kv, dim, page)
        cache = cache_of(ctx, kind, pages, kv, dim, page, raw)
        pool = S.decode_pool(raw, kind, pages, kv, dim, page)
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        say("attend nothing", rows_together, kind)
        got = run(ctx, cache, q, positions, requests_of, table, first=first, end=end)
        check(got, *S.attend(pool, q, positions, requests_of, table, dim ** -0.5, first=first, end=end))
        assert (got[[0, 1, 2, 3, 5, 8, 9]] == 0).all() and (got[[4, 6, 7]] != 0).any(-1).all()
        got = run(ctx, cache, q, positions, requests_of, table, first=first)
        check(got, *S.attend(pool, q, positions, requests_of, table, dim ** -0.5, first=first))


@pytest.mark.parametrize("kind,scored", [("q4", False)] + [(kind, True) for kind in S.KINDS])
def test_masked_places_have_no_influence(ctx, kind, scored):
    """NaN and infinities outside every row's tokens; and inside some rows' only, where those may get NaN and no others do."""
    rng = np.random.default_rng(11)
    heads, kv, dim, page = 4, 2, 96, 16
    rows, tokens = 33, 150
    table, pages = K.make_tables(rng, [tokens], page)
    raw = S.random_pool(rng, kind, pages, kv, dim, page)
    more = dict(cap=20.0, slopes=np.full(heads, 0.01, np.float32)) if scored else {}
    positions = np.arange(70, 70 + rows)
    first = np.where(np.arange(rows) < 15, 10, 75) if scored else None
    end = np.minimum(positions + 4, 100) if scored else None
    lo, hi = (first, end) if scored else (np.zeros(rows, int), positions + 1)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    for bad_tokens in ([t for t in range(tokens) if t < lo.min() or t >= hi.max()], [72, 101 if scored else 90]):
        for bad in (np.nan, np.inf, -np.inf):
            dirty = raw.reshape(2, pages, kv, -1).copy()
            for t in bad_tokens:
                p, o = table[0, t // page], t % page
                for which in (0, 1):
                    if kind == "f16":
                        dirty.view(np.float16).reshape(2, pages, kv, page, dim)[which, p, :, o, 5::7] = bad
                    else:
                        codes = page * dim // (1 if kind == "q8" else 2)
                        scales = dirty[..., codes:].view(np.float16).reshape(2, pages, kv, dim // 32, page)
                        scales[which, p, :, 1, o] = np.float16(bad)
                        dirty[..., codes:] = scales.view(np.uint8).reshape(2, pages, kv, -1)
            clean = cache_of(ctx, kind, pages, kv, dim, page, raw)
            other = cache_of(ctx, kind, pages, kv, dim, page, dirty.reshape(-1))
            say("attend masked", kind, scored, len(bad_tokens), bad)
            for together in (False, True):
                of, t = (np.zeros(rows, int), table) if together else (None, np.repeat(table, rows, 0))
                a, b = (run(ctx, c, q, positions, of, t, first=first, end=end, **more) for c in (clean, other))
                hit = np.array([any(lo[i] <= x < hi[i] for x in bad_tokens) for i in range(rows)])
                assert np.isfinite(a).all() and np.isfinite(b[~hit]).all()
                # (tiles in which some row sees such a value are added in another order; elsewhere the very bits)
                check(b[~hit], *(w[~hit] for w in S.attend(S.decode_pool(raw, kind, pages, kv, dim, page), q, positions, of, t, dim ** -0.5,
                                                           first=first, end=end, cap=more.get("cap", 0.0), slopes=more.get("slopes"))))


def test_values_past_binary16_in_fours(ctx):
    """A finite scale whose multiples pass binary16: rows that do not see that token are what they are without it."""
    rng = np.random.default_rng(12)
    heads, kv, dim, page, rows = 2, 1, 64, 16, 24
    table, pages = K.make_tables(rng, [64], page)
    raw = S.random_pool(rng, "q4", pages, kv, dim, page).reshape(2, pages, kv, -1)
    scales = raw[..., page * dim // 2:].view(np.float16).reshape(2, pages, kv, dim // 32, page)
    scales[1, table[0, 2], :, 1, 3] = 30000                   # token 35: 30000 x -8 ... 7
    raw[..., page * dim // 2:] = scales.view(np.uint8).reshape(2, pages, kv, -1)
    cache = cache_of(ctx, "q4", pages, kv, dim, page, raw.reshape(-1))
    pool = S.decode_pool(raw, "q4", pages, kv, dim, page)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    positions = np.arange(24, 48)
    say("attend past binary16")
    got = run(ctx, cache, q, positions, np.zeros(rows, int), table)
    blind = positions < 35
    want, bound = S.attend(pool, q, positions, np.zeros(rows, int), table, dim ** -0.5)
    check(got[blind], want[blind], bound[blind])
    assert np.isfinite(got[~blind][..., :32]).all()            # the other block's columns
    assert np.array_equal(np.isfinite(got[~blind]), np.isfinite(want[~blind]))


@pytest.mark.parametrize("kind", S.KINDS)
def test_scored_scores_of_all_sizes(ctx, kind):
    """Scores far beyond a cap and far below it, on both sides of where tanh's two forms meet; slopes of either sign, of zero."""
    rng = np.random.default_rng(13)
    heads, kv, dim, page, n = 6, 2, 64, 16, 400
    table, pages = K.make_tables(rng, [n] * 6, page)
    raw = S.random_pool(rng, kind, pages, kv, dim, page)
    pool = S.decode_pool(raw, kind, pages, kv, dim, page)
    cache = cache_of(ctx, kind, pages, kv, dim, page, raw)
    q = rng.standard_normal((6, heads, dim)).astype(np.float32)
    q *= np.array([0, 1e-6, 0.3, 8, 300, 1e6], np.float32)[:, None, None]
    positions = np.full(6, n - 1)
    slopes = np.array([0, 0.5, -0.02, 1e-6, 20, -1e-4], np.float32)
    for cap in (1e-3, 1.0, 30.0, 1e4):
        say("attend sizes", kind, cap)
        for m in (None, slopes):
            got = run(ctx, cache, q, positions, None, table, cap=cap, slopes=m)
            keep = slice(0, 5)                                 # (1e6: what fp32 says of a score between -cap and cap is tested by finiteness)
            want, bound = S.attend(pool, q, positions, None, table, dim ** -0.5, cap=cap, slopes=m)
            check(got[keep], want[keep], bound[keep])
            assert np.isfinite(got).all()


def test_scored_without_anything_is_the_plain_call(ctx):
    """The entry point with nothing asked for says what jl_kv_attention says, up to a factor's place."""
    from jitllm_amd import _lib as L
    from jitllm_amd.attention import PagedAttention
    rng = np.random.default_rng(15)
    heads, kv, dim, page = 8, 2, 128, 32
    lengths = [700, 3, 64]
    table, pages = K.make_tables(rng, lengths, page)
    raw = S.random_pool(rng, "f16", pages, kv, dim, page)
    cache = cache_of(ctx, "f16", pages, kv, dim, page, raw)
    q = rng.standard_normal((3, heads, dim)).astype(np.float32)
    attention = PagedAttention(ctx, 3, heads, kv, dim)
    qa, out, pos, t = ctx.from_numpy(q), ctx.float_array(3 * heads * dim, fill=1.0), K.ints(ctx, np.array(lengths) - 1), K.ints(ctx, table)
    say("attend scored, nothing asked")
    L.check(ctx._lib.jl_kv_attention_scored(ctx.handle, cache.handle, qa.ptr, heads, heads * dim, 3, pos.ptr, None, t.ptr, 3, table.shape[1],
                                            dim ** -0.5, 0, 0.0, None, None, None, out.ptr, 0, heads * dim, attention.workspace.ptr, attention.workspace.nbytes))
    ctx.sync()
    check(out.get().astype(np.float64).reshape(3, heads, dim), *S.attend(S.decode_pool(raw, "f16", pages, kv, dim, page), q, np.array(lengths) - 1, None, table, dim ** -0.5))


def test_scored_is_the_same_every_time(ctx):
    rng = np.random.default_rng(14)
    lengths = np.array([5000, 12, 800, 0, 3333])
    table, pages = K.make_tables(rng, lengths, 16)
    for kind in S.KINDS:
        raw = S.random_pool(rng, kind, pages, 2, 128, 16)
        cache = cache_of(ctx, kind, pages, 2, 128, 16, raw)
        q = rng.standard_normal((5, 8, 128)).astype(np.float32)
        say("attend repeats", kind)
        runs = [run(ctx, cache, q, lengths - 1, None, table, cap=30.0, slopes=np.full(8, 0.01, np.float32)) for _ in range(4)]
        assert all(np.array_equal(r, runs[0]) for r in runs[1:])


def test_fours_past_32_bit_offsets(ctx):
    """A cache of over 4 GiB of four-bit blocks: its last pages are written, read and attended to where they lie."""
    from jitllm_amd.attention import PagedKvCache
    rng = np.random.default_rng(15)
    kv, dim, page, heads = 8, 256, 256, 8
    pages = 9000                                               # 288 KiB a page for k, and for v
    say("fours past 4 GiB")
    cache = PagedKvCache(ctx, kv_type("q4"), pages, kv, dim, page)
    assert cache.nbytes > 1 << 32
    rows = 40
    x = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float32)
    slots = (pages - 1 - np.arange(rows) // 8 * 1700) * page + np.arange(rows) % 8
    table = (pages - 1 - np.arange(5) * 1700).reshape(5, 1)
    K.run_append(ctx, cache, x, heads, kv, dim, np.arange(rows) % 8, slots, np.zeros(0), False, None, None, 0.0)
    k, v = ctx.float_array(rows * kv * dim), ctx.float_array(rows * kv * dim)
    cache.read(K.ints(ctx, slots), rows, k, v)
    out = run(ctx, cache, np.ascontiguousarray(x[7::8, :heads]), np.full(5, 7), None, table, cap=30.0)
    pool = np.zeros((2, 5, kv, page, dim))
    for which, (a, y) in enumerate(((k, x[:, heads:heads + kv]), (v, x[:, heads + kv:]))):
        kept = a.get().astype(np.float64).reshape(rows, kv, dim)
        n, d, border = S.encode_fours(y.astype(np.float64))
        sure = border > 1e-6
        assert np.array_equal(kept[sure], ((n - 8) * np.repeat(d, 32, -1)).astype(np.float16).astype(np.float64)[sure])
        pool[which, :, :, :8] = kept.reshape(5, 8, kv, dim).transpose(0, 2, 1, 3)
    check(out, *S.attend(pool, x[7::8, :heads], np.full(5, 7), None, np.arange(5).reshape(5, 1), dim ** -0.5, cap=30.0))
    cache.free()


@pytest.mark.parametrize("rows", [9, 340])
@pytest.mark.parametrize("kind", S.KINDS)
def test_scored_rows_of_extreme_queries(ctx, kind, rows):
    """Rows that go together, few and a prompt's block, each with scores of another size: thousands apart, all equal, below
    binary16; one with an infinity and one with NaN in a head, which are those heads' alone."""
    rng = np.random.default_rng(rows)
    dim, page, kv, heads, n = 64, 16, 16, 32, 400
    table, pages = K.make_tables(rng, [n], page)
    raw = S.random_pool(rng, kind, pages, kv, dim, page)
    positions, of = np.arange(n - rows, n), np.zeros(rows, int)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    q *= np.array([1, 300, 0, 1e-9, 2.0 ** -140, 40], np.float32)[np.arange(rows) % 6, None, None]
    q[7::6] *= np.exp(rng.uniform(-20, 5, (len(q[7::6]), heads, dim))).astype(np.float32)
    cache = cache_of(ctx, kind, pages, kv, dim, page, raw)
    pool = S.decode_pool(raw, kind, pages, kv, dim, page)
    slopes = (2.0 ** (-8 * np.arange(1, heads + 1) / heads)).astype(np.float32)
    for cap, m in ((0.0, slopes), (30.0, None), (5.0, slopes)):
        say("attend scored extreme", kind, rows, cap)
        clean = run(ctx, cache, q, positions, of, table, cap=cap, slopes=m, window=150)
        check(clean, *S.attend(pool, q, positions, of, table, dim ** -0.5, 150, cap, m))
        bad = q.copy()
        bad[rows // 2, 5, 3], bad[rows // 3, 30, 60] = np.inf, np.nan
        got = run(ctx, cache, bad, positions, of, table, cap=cap, slopes=m, window=150)
        lost = np.zeros(got.shape[:2], bool)
        lost[rows // 2, 5] = lost[rows // 3, 30] = True
        assert np.array_equal(got[~lost], clean[~lost]) and not np.isfinite(got[rows // 3, 30]).any()

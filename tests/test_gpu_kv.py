"""The paged key-value cache's operators on the GPU against numpy in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import kv_models as M
from gpu_util import say

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -11            # half a step of binary16, relative to the value
ULP = 2.0 ** -24             # ... of fp32


@pytest.fixture(scope="module")
def ctx():
    from jitllm_amd.runtime import Context
    c = Context(0)
    yield c
    c.close()


def ints(ctx, values):
    from jitllm_amd.attention import IntArray
    values = np.asarray(values, np.int32).reshape(-1)
    a = IntArray(ctx, max(1, values.size))
    if values.size:
        a.upload(values)
    a.size = values.size
    return a


def random_pool(rng, q8, pages, heads, dim, page, spread=1.0):
    """A cache's bytes: normal values, or blocks of uniform bytes with scales of their own."""
    per = M.part_bytes(q8, dim, page)
    if not q8:
        return (spread * rng.standard_normal((2, pages, heads, page * dim))).astype(np.float16).view(np.uint8).reshape(-1)
    raw = np.empty((2, pages, heads, per), np.uint8)
    raw[..., :page * dim] = rng.integers(-127, 128, (2, pages, heads, page * dim)).astype(np.int8).view(np.uint8)
    d = (spread * rng.uniform(0.004, 0.03, (2, pages, heads, page * dim // 32))).astype(np.float16)
    raw[..., page * dim:] = d.view(np.uint8).reshape(2, pages, heads, -1)
    return raw.reshape(-1)


def cache_of(ctx, q8, pages, heads, dim, page, raw):
    from jitllm_amd.attention import KvType, PagedKvCache
    memory = ctx.raw_buffer(raw.nbytes)
    memory.upload(raw)
    return PagedKvCache(ctx, KvType.Q8_0 if q8 else KvType.F16, pages, heads, dim, page, memory=memory)


def pool_bytes(cache):
    return cache.memory.download(np.uint8, cache.nbytes)


# ---- jl_kv_plan ----------------------------------------------------------------------------------

NAMES = ("lengths", "rowStarts", "table", "pageRing", "freePages", "slots", "positions", "rowRequests")


def run_plan(ctx, past, fresh, pages, page, ring, free, table, max_rows, in_place=False):
    from jitllm_amd.attention import BlockTables
    requests, stride = table.shape
    t = BlockTables(ctx, requests, stride, pages, page, max_rows)
    t.table.set(table), t.pageRing.set(ring)
    if in_place:
        t.lengths.set(past), t.freePages.set(free)
        t.plan(ints(ctx, fresh))
    else:
        t.plan(ints(ctx, fresh), past=ints(ctx, past), freeIn=ints(ctx, free))
    ctx.sync()
    return t


def check_plan(ctx, t, want):
    for name in NAMES:
        got = getattr(t, name).get() if getattr(t, name).size else np.zeros(0)
        assert np.array_equal(got, want[name].reshape(-1)), name


def random_step(rng, requests, page, stride, pages=None, prompts=0.1, free_share=1.5):
    past = rng.integers(0, stride * page, requests)
    fresh = rng.choice([1, 1, 1, 1, 1, 0, -1], requests)
    begin = rng.random(requests) < prompts
    past[begin], fresh[begin] = 0, rng.integers(1, stride * page + 1, int(begin.sum()))
    had = -(-past // page)
    need = np.maximum(0, -(-(past + np.maximum(fresh, 0)) // page) - had)
    free = int(need.sum() * free_share)
    pages = pages or int(had.sum()) + free + 3
    order = rng.permutation(pages)
    table = np.full((requests, stride), -1)
    table[np.arange(stride) < had[:, None]] = order[:had.sum()]
    head = int(rng.integers(0, pages))
    ring = np.full(pages, -1)
    ring[(head + np.arange(free)) % pages] = order[had.sum():had.sum() + free]
    return past, fresh, pages, ring, np.array([head, free]), table


@pytest.mark.parametrize("requests,page,stride,max_rows,free_share", [
    (1, 16, 4, 64, 1.5), (64, 16, 256, 512, 1.5), (65, 32, 7, 300, 0.5), (1023, 64, 5, 20000, 1.0), (1025, 128, 9, 40000, 0.4),
    (2500, 16, 3, 2500, 1.1), (4096, 256, 4, 131072, 1.5), (8192, 16, 2, 9000, 0.9), (200, 64, 100, 131072, 1.2)])
def test_plan_is_the_sequential_one(ctx, requests, page, stride, max_rows, free_share):
    say("plan", requests, page, stride, max_rows, free_share)
    rng = np.random.default_rng(requests + page)
    past, fresh, pages, ring, free, table = random_step(rng, requests, page, stride, free_share=free_share)
    want = M.plan(past, fresh, pages, page, ring, free, table, max_rows)
    t = run_plan(ctx, past, fresh, pages, page, ring, free, table, max_rows)
    check_plan(ctx, t, want)
    # the same call over what it left leaves the same
    t.plan(ints(ctx, fresh), past=ints(ctx, past), freeIn=ints(ctx, free))
    ctx.sync()
    check_plan(ctx, t, want)
    check_plan(ctx, run_plan(ctx, past, fresh, pages, page, ring, free, table, max_rows, in_place=True), want)


PLAN_EDGES = {
    # past, fresh, pages, ring, free, blocks a request, max_rows
    "nothing waits": ([0, 0], [0, 0], 4, [0, 1, 2, 3], [0, 4], 2, 4),
    "no rows": ([3], [1], 4, [1, 2, 3, 0], [0, 3], 2, 0),
    "a page's last token, its first, the table's last": ([15, 16, 31, 32], [1, 1, 1, 1], 12, range(12), [0, 12], 2, 8),
    "a prompt as long as the table row, one longer": ([0, 0], [32, 33], 8, range(8), [6, 8], 2, 80),
    "ring empty: none but those with room go on": ([16, 5, 0, 7], [1, 1, 3, 2], 4, range(4), [2, 0], 2, 9),
    "one page for two": ([16, 16, 3], [1, 1, 1], 4, range(4), [3, 1], 2, 9),
    "a large request in front of small ones": ([0, 0, 0], [40, 3, 3], 8, range(8), [0, 2], 4, 64),
    "lengths that no row holds": ([-1, 33, -5, 2**31 - 1], [1, 1, -1, 1], 8, range(8), [0, 8], 2, 8),
    "a fresh of 2^31 - 1": ([0, 4], [2**31 - 1, 1], 8, range(8), [0, 8], 2, 8),
    "no such ring": ([0, 4, 20], [1, 1, -1], 8, range(8), [9, 4], 2, 8),
    "no such ring either": ([0, 4, 20], [1, 1, -1], 8, range(8), [1, 9], 2, 8),
    "negative": ([0, 4, 20], [1, 1, -1], 8, range(8), [-1, 4], 2, 8),
    "more comes back than was missing": ([32, 32, 32], [-1, -1, -1], 5, range(5), [4, 2], 2, 8),
    "all end": ([32, 1, 0, 17], [-1, -7, -1, -2**31], 12, range(12), [5, 0], 2, 8),
    "rows that pass the step's end": ([0, 0, 0], [5, 6, 2], 8, range(8), [0, 8], 2, 8),
}


@pytest.mark.parametrize("name", PLAN_EDGES)
def test_plan_edges(ctx, name):
    say("plan edge", name)
    past, fresh, pages, ring, free, stride, max_rows = PLAN_EDGES[name]
    requests = len(past)
    # bad entries among the good: pages outside the cache give no slot
    table = (np.arange(requests * stride).reshape(requests, stride) * 7) % (pages + 2) - 1
    ring = np.array(list(ring))
    want = M.plan(past, fresh, pages, 16, ring, free, table, max_rows)
    check_plan(ctx, run_plan(ctx, np.array(past), np.array(fresh), pages, 16, ring, np.array(free), table, max_rows), want)


def test_plan_of_no_requests(ctx):
    from jitllm_amd.attention import BlockTables
    t = BlockTables(ctx, 0, 4, 5, 16, 6)
    t.plan(ints(ctx, []))
    ctx.sync()
    assert t.rowStarts.get().tolist() == [0] and t.freePages.get().tolist() == [0, 5]
    assert t.slots.get().tolist() == t.positions.get().tolist() == t.rowRequests.get().tolist() == [-1] * 6


@pytest.mark.parametrize("requests,stride,page,pages,max_rows", [(40, 8, 16, 150, 400), (300, 8, 16, 1100, 5000)])
def test_plan_many_steps_lose_no_page(ctx, requests, stride, page, pages, max_rows):
    """A server's life: requests begin, decode, wait, end; in place, step after step, against the sequential one."""
    from jitllm_amd.attention import BlockTables
    rng = np.random.default_rng(8)
    t = BlockTables(ctx, requests, stride, pages, page, max_rows)
    state = {"lengths": np.zeros(requests, int), "table": np.full((requests, stride), -1), "pageRing": np.arange(pages), "freePages": np.array([0, pages])}
    for step in range(60):
        fresh = np.where(state["lengths"] == 0, rng.integers(0, 60, requests) * (rng.random(requests) < 0.4),
                         rng.choice([1, 1, 1, 0, -1], requests, p=[0.4, 0.3, 0.15, 0.1, 0.05]))
        say("step", step)
        t.plan(ints(ctx, fresh))
        state = M.plan(state["lengths"], fresh, pages, page, state["pageRing"], state["freePages"], state["table"], max_rows)
        ctx.sync()
        check_plan(ctx, t, state)
        held = [state["table"][r, :-(-state["lengths"][r] // page)] for r in range(requests)]
        free = state["pageRing"][(state["freePages"][0] + np.arange(state["freePages"][1])) % pages]
        assert sorted(np.concatenate(held + [free])) == list(range(pages))


# ---- jl_kv_append and jl_kv_read -----------------------------------------------------------------

def run_append(ctx, cache, x, heads, kv, dim, positions, slots, freq, halves, qn, kn, eps, apart=False, pad=0, in_place=False):
    """x [rows][heads + 2 kv][dim] -> q as the call leaves it."""
    from jitllm_amd.attention import Rope, RopeStyle, Rows
    rows = len(x)
    rope = Rope.of(ctx, freq, RopeStyle.HALVES if halves else RopeStyle.PAIRS) if len(freq) else None
    norms = dict(qNorm=ctx.from_numpy(qn) if qn is not None else None, kNorm=ctx.from_numpy(kn) if kn is not None else None, eps=eps)
    w = heads * dim
    sentinel = np.float32(-77.25)
    if apart:
        q, k, v = (ctx.from_numpy(part) for part in (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]))
        qr, kr, vr = Rows(q, w), Rows(k, kv * dim), Rows(v, kv * dim)
    else:
        stride = (heads + 2 * kv) * dim + pad
        flat = np.full((rows, stride), sentinel, np.float32)
        flat[:, :stride - pad] = x.reshape(rows, -1)
        q = ctx.from_numpy(flat)
        qr, kr, vr = Rows(q, stride), Rows(q, stride, w), Rows(q, stride, w + kv * dim)
    out = q if in_place else ctx.float_array(rows * (w + pad), fill=float(sentinel))
    outr = qr if in_place else Rows(out, w + pad)
    cache.append(kr, vr, ints(ctx, positions), ints(ctx, slots), rows, rope=rope, q=qr if heads else None, qOut=outr if heads else None,
                 heads=heads, **norms)
    ctx.sync()
    got = out.get()
    if not heads:
        return None
    got = np.lib.stride_tricks.as_strided(got, (rows, w), (outr.stride * 4, 4)).copy()
    if pad and not in_place:
        rest = out.get().reshape(rows, -1)[:, w:]
        assert (rest == sentinel).all()
    return got.reshape(rows, heads, dim)


APPENDS = [
    # rows, heads, kv, dim, page, q8, halves, turned, norm, context
    (1, 32, 8, 64, 16, False, False, 64, False, 1000), (1, 14, 2, 64, 16, True, True, 64, False, 5), (3, 28, 4, 128, 32, False, True, 128, False, 131072),
    (64, 32, 8, 128, 32, True, True, 128, True, 8192), (65, 5, 5, 96, 16, True, False, 96, True, 700), (33, 3, 1, 96, 64, False, True, 48, True, 900),
    (17, 8, 2, 192, 128, True, True, 96, False, 100000), (40, 16, 4, 256, 16, True, False, 256, True, 4096), (7, 71, 1, 64, 256, False, False, 32, False, 60),
    (300, 4, 2, 128, 64, False, False, 128, False, 2000000), (20, 8, 8, 128, 16, True, False, 0, False, 50), (9, 0, 4, 128, 16, False, True, 64, True, 77)]


@pytest.mark.parametrize("rows,heads,kv,dim,page,q8,halves,turned,norm,context", APPENDS)
def test_append(ctx, rows, heads, kv, dim, page, q8, halves, turned, norm, context):
    say("append", rows, heads, kv, dim, page, q8, halves, turned, norm, context)
    rng = np.random.default_rng(rows + dim + page)
    pages = rows // page + 3
    x = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float32)
    x[:, :, 3] *= 20                                           # a channel that stands out, as keys have
    x[rows // 2, heads + 2 * kv - 1, :32] = 0                  # a block of zeros
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    slots = rng.permutation(pages * page)[:rows]
    positions = rng.integers(0, context, rows)
    freq = 500000.0 ** (-np.arange(0, turned, 2) / turned) if turned else np.zeros(0)
    qn, kn = (1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)) if norm else (None, None)
    eps = 1e-6
    if rows > 2:
        slots[1], positions[2] = -1, -1                        # no page; no token at all
    if rows > 3:
        slots[3] = pages * page                                # a slot behind the cache's last
    apart = rows % 2 == 1
    got = run_append(ctx, cache, x, heads, kv, dim, positions, slots, freq, halves, qn, kn, eps, apart=apart, pad=0 if apart else 8)
    after = M.decode_pool(pool_bytes(cache), q8, pages, kv, dim, page)
    before = M.decode_pool(raw, q8, pages, kv, dim, page)
    live = positions >= 0
    # A turned value is two products and a sum over cos and sin that are exact to fp32 but for the rounding of
    # an angle below pi (2^-24 pi of it) and the functions' own few units: 10 ulp of |a| + |b| cover them, and
    # a norm's sum of dim squares, division, root and products another dim / 2 + 8 of the value.
    step = (10 + (dim / 2 + 8 if norm else 0)) * ULP
    k = M.rotate(x[:, heads:heads + kv], np.maximum(positions, 0), freq, halves, kn, eps)
    size = lambda y: np.abs(y).max(-1, keepdims=True) * 2      # noqa: E731  (|a| + |b| of any pair of the head)
    if heads:
        q = M.rotate(x[:, :heads], np.maximum(positions, 0), freq, halves, qn, eps)
        assert (np.abs(got - q) <= step * size(q))[live].all()
        assert (got[~live] == -77.25).all()
    v = x[:, heads + kv:].astype(np.float64)
    written = np.zeros((pages, page), bool)
    for which, y, slack in ((0, k, step * size(k)), (1, v, 0.0 * size(v))):
        for i in range(rows):
            if not live[i] or not 0 <= slots[i] < pages * page:
                continue
            at = after[which, slots[i] // page, :, slots[i] % page]
            written[slots[i] // page, slots[i] % page] = True
            if not q8:
                assert (np.abs(at - y[i]) <= slack[i] + HALF * np.abs(y[i]) + 2.0 ** -25).all()
                continue
            kept, d, _ = M.encode_blocks(y[i])
            # half a step of the block's scale, which is half a binary16 step off max / 127 (an end is clamped by that);
            # the value itself is rounded to binary16
            d = np.repeat(d, 32, -1)
            assert (np.abs(at - y[i]) <= d / 2 * (1 + 2 * HALF) + slack[i] + 2 * HALF * np.abs(y[i]) + 2.0 ** -24).all()
            if which == 1:                                     # nothing but copies in front of it: the very bytes
                assert np.array_equal(at, (kept * d).astype(np.float16).astype(np.float64))
    keep = np.broadcast_to(~written[None, :, None, :, None], after.shape)
    assert np.array_equal(after[keep], before[keep])


def test_append_in_place_is_the_same(ctx):
    rng = np.random.default_rng(3)
    for halves in (False, True):
        for dim, turned in ((64, 64), (96, 64), (256, 256)):
            x = rng.standard_normal((37, 6, dim)).astype(np.float32)
            raw = random_pool(rng, False, 4, 1, dim, 16)
            freq = 1e4 ** (-np.arange(0, turned, 2) / turned)
            slots, positions = np.arange(37), rng.integers(0, 9999, 37)
            say("append in place", halves, dim, turned)
            norm = rng.standard_normal(dim).astype(np.float32)
            two = [run_append(ctx, cache_of(ctx, False, 4, 1, dim, 16, raw), x, 4, 1, dim, positions, slots, freq, halves, norm, None, 1e-5, in_place=p)
                   for p in (False, True)]
            assert np.array_equal(two[0], two[1])


@pytest.mark.parametrize("q8", [False, True])
def test_append_special_values(ctx, q8):
    """Infinities, NaN, values past binary16, values below its smallest."""
    dim, page = 64, 16
    x = np.zeros((6, 3, dim), np.float32)
    x[0, 2, :] = 1e6
    x[1, 2, :] = np.nan
    x[2, 2, 0], x[2, 2, 1], x[2, 2, 2] = np.inf, -np.inf, 5
    x[3, 2, :] = 1e-9
    x[4, 2, :32], x[4, 2, 5] = 2, np.nan
    x[5, 2, :] = np.linspace(-1e38, 1e38, dim)
    cache = cache_of(ctx, q8, 2, 1, dim, page, np.zeros(2 * 2 * M.part_bytes(q8, dim, page), np.uint8))
    say("append special", q8)
    run_append(ctx, cache, x, 1, 1, dim, np.zeros(6, int), np.arange(6), np.zeros(0), False, None, None, 0.0)
    v = M.decode_pool(pool_bytes(cache), q8, 2, 1, dim, page)[1, 0, 0]
    with np.errstate(over="ignore"):
        plain = x[:, 2].astype(np.float16).astype(np.float64)
    if not q8:
        assert np.array_equal(v[:6], plain, equal_nan=True)
        return
    assert (v[0] == np.inf).all()                               # 127 x 7872, beyond binary16
    assert (v[1] == 0).all()                                    # nothing but NaN: a scale of 0
    assert v[2, 0] == np.inf and v[2, 1] == -np.inf and v[2, 2] == 0
    assert (v[3] == 0).all()
    assert v[4, 5] == 0 and np.allclose(np.delete(v[4, :32], 5), 2, rtol=2 * HALF)
    assert np.isinf(v[5][[0, -1]]).all()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("dim,kv,page", [(64, 3, 16), (96, 2, 256), (128, 8, 32), (192, 1, 64), (256, 5, 128)])
def test_read(ctx, q8, dim, kv, page):
    say("read", q8, dim, kv, page)
    rng = np.random.default_rng(dim)
    pages, rows = 5, 23
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    slots = rng.integers(0, pages * page, rows)                # one twice is fine here
    slots[4], slots[9], slots[11] = -1, pages * page, 2**31 - 1
    pool = M.decode_pool(raw, q8, pages, kv, dim, page)
    ok = (slots >= 0) & (slots < pages * page)
    at = np.where(ok, slots, 0)
    want = np.where(ok[:, None, None, None], pool[:, at // page, :, at % page], 0)      # [rows][2][kv][dim]
    if want.shape[0] == 2:
        want = np.swapaxes(want, 0, 1)
    for make in (ctx.half_array, ctx.float_array):
        k, v = make(rows * kv * dim), make(rows * kv * dim)
        cache.read(ints(ctx, slots), rows, k, v)
        ctx.sync()
        for which, a in enumerate((k, v)):
            assert np.array_equal(a.get().astype(np.float64).reshape(rows, kv, dim), want[:, which])
    only = ctx.float_array(rows * kv * dim)
    cache.read(ints(ctx, slots), rows, v=only)
    ctx.sync()
    assert np.array_equal(only.get().astype(np.float64).reshape(rows, kv, dim), want[:, 1])


# ---- jl_kv_attention -----------------------------------------------------------------------------

def make_tables(rng, lengths, page, requests_of=None, requests=None, spare=2):
    """A table whose rows hold the requests' pages in no order, -1 behind them; (table, pages)."""
    rows = len(lengths)
    requests = requests or rows
    need = np.zeros(requests, int)
    for i, n in enumerate(lengths):
        r = i if requests_of is None else requests_of[i]
        need[r] = max(need[r], -(-n // page))
    pages = int(need.sum()) + spare
    table = np.full((requests, max(1, need.max())), -1)
    order = rng.permutation(pages)[:need.sum()]
    table[np.arange(table.shape[1]) < need[:, None]] = order
    return table, pages


def run_attend(ctx, cache, q, positions, requests_of, table, scale=None, window=0, half=False, pad=0, workspace=None, attention=None):
    from jitllm_amd import _lib as L
    from jitllm_amd.attention import PagedAttention, Rows
    rows, heads, dim = q.shape
    attention = attention or PagedAttention(ctx, rows, heads, cache.kvHeads, dim)
    if workspace is not None:
        attention.workspace.upload(np.full(attention.workspace.nbytes, workspace, np.uint8))
        L.check(ctx._lib.jl_kv_attention_workspace_init(ctx.handle, attention.workspace.ptr, attention.workspace.nbytes))
    stride = heads * dim + pad
    flat = np.full((rows, stride), np.nan, np.float32)
    flat[:, :heads * dim] = q.reshape(rows, -1)
    out = (ctx.half_from_numpy if half else ctx.from_numpy)(np.full((rows + 2) * stride, -5.5))
    qa = ctx.from_numpy(flat)
    attention.attend(cache, Rows(qa, stride), rows, ints(ctx, positions), ints(ctx, table), Rows(out, stride), requests=table.shape[0],
                     rowRequests=ints(ctx, requests_of) if requests_of is not None else None, scale=scale, window=window)
    ctx.sync()
    got = out.get().reshape(rows + 2, stride)
    assert (got[rows:] == -5.5).all() and (got[:, heads * dim:] == -5.5).all()   # rows behind, columns between
    return got[:rows, :heads * dim].astype(np.float64).reshape(rows, heads, dim)


def check_attend(got, want, weight, reach, lengths, dim, half=False):
    """An element is sum p v.  A score is off by at most the rounding of the 2 dim products and sums of its two
    binary16 parts, (2 dim + 8) half steps of scale * sum |q k|, and its weight by twice that (itself, and the sum
    of all weights) and the power's own 4; the sums over n tokens add n + 64 half steps of sum p |v|.  Roundings of
    either sign: all outputs together are held to 2e-6 of their norm and a hundredth of the sum of those bounds,
    which one operand rounded to binary16 (2^-11) would pass ten times over."""
    n = np.maximum(np.asarray(lengths, float), 1)[:, None, None]
    bound = ((2 * (2 * dim + 8) * reach[..., None] + 8) + n + 64) * ULP * weight
    if half:
        bound = bound + HALF * np.abs(want) + 2.0 ** -25
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
    if not half:
        assert np.linalg.norm(got - want) <= 2e-6 * np.linalg.norm(want) + 0.01 * np.linalg.norm(bound) + 1e-12


ATTENDS = [
    # lengths, heads, kv, dim, page, q8, window, half
    ([201], 32, 8, 64, 16, False, 0, False), ([1], 14, 2, 64, 16, True, 0, True), ([1, 2, 15, 16, 17, 31, 32, 33, 0, 64, 65], 4, 2, 128, 16, False, 0, False),
    ([127, 128, 129, 255, 256, 257, 1000], 28, 4, 128, 32, True, 0, False), ([950, 3, 511, 512, 513], 6, 6, 128, 16, False, 0, True),
    ([4096], 16, 4, 256, 16, True, 1024, False), ([700, 40, 90], 16, 4, 256, 64, False, 100, False), ([333, 1, 77], 9, 3, 96, 16, True, 0, False),
    ([1300, 64], 3, 3, 96, 128, False, 1, False), ([260, 511], 24, 2, 192, 256, False, 0, True), ([900, 5], 12, 2, 192, 16, True, 17, False),
    ([2000, 7], 71, 1, 64, 32, False, 0, False), ([129], 48, 1, 128, 16, True, 0, True), ([9000], 32, 8, 128, 64, False, 0, False),
    ([5000, 1, 300], 8, 8, 64, 16, True, 0, False), ([3, 0, 20, 17], 1200, 600, 64, 16, False, 0, False), ([40, 3], 300, 300, 256, 16, True, 0, False)]


@pytest.mark.parametrize("lengths,heads,kv,dim,page,q8,window,half", ATTENDS)
def test_attend(ctx, lengths, heads, kv, dim, page, q8, window, half):
    say("attend", lengths, heads, kv, dim, page, q8, window, half)
    rng = np.random.default_rng(sum(lengths) + dim)
    rows = len(lengths)
    table, pages = make_tables(rng, lengths, page)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    positions = np.array(lengths) - 1
    scale = dim ** -0.5
    got = run_attend(ctx, cache, q, positions, None, table, scale, window, half, pad=8 if rows > 1 else 0, workspace=0xff)
    want = M.attend(M.decode_pool(raw, q8, pages, kv, dim, page), q, positions, None, table, scale, window)
    check_attend(got, *want, np.minimum(lengths, window or max(lengths)), dim, half)


@pytest.mark.parametrize("rows,longest,heads,kv,dim,q8", [(70, 400, 8, 2, 64, False), (300, 60, 4, 4, 128, True), (1030, 20, 4, 1, 64, False),
                                                          (40, 3000, 7, 1, 128, False), (5, 20000, 4, 1, 64, True)])
def test_attend_ragged_batches(ctx, rows, longest, heads, kv, dim, q8):
    """Many rows of all lengths, empty ones among them, that read the table's rows in another order."""
    say("attend ragged", rows, longest, heads, kv, dim, q8)
    rng = np.random.default_rng(rows)
    page = 16
    lengths = (longest * rng.random(rows) ** 2).astype(int)
    lengths[rng.integers(0, rows)] = longest
    requests = rows + 5
    requests_of = rng.permutation(requests)[:rows]
    table, pages = make_tables(rng, lengths, page, requests_of, requests)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    q = (2 * rng.standard_normal((rows, heads, dim))).astype(np.float32)
    got = run_attend(ctx, cache, q, lengths - 1, requests_of, table, workspace=0x7f)
    want = M.attend(M.decode_pool(raw, q8, pages, kv, dim, page), q, lengths - 1, requests_of, table, dim ** -0.5)
    check_attend(got, *want, lengths, dim)
    assert (got[lengths == 0] == 0).all()


def test_attend_rows_of_one_request(ctx):
    """A prompt's rows, each up to its own position, and rows of requests that the table does not have."""
    rng = np.random.default_rng(4)
    dim, page, kv, heads = 64, 16, 2, 8
    table, pages = make_tables(rng, [50, 130], page)
    raw = random_pool(rng, False, pages, kv, dim, page)
    cache = cache_of(ctx, False, pages, kv, dim, page, raw)
    positions = np.concatenate([np.arange(50), np.arange(100, 130), [5, 5, -1, -7]])
    requests_of = np.concatenate([np.zeros(50, int), np.ones(30, int), [-1, 2, 0, 1]])
    q = rng.standard_normal((len(positions), heads, dim)).astype(np.float32)
    say("attend prompt rows")
    got = run_attend(ctx, cache, q, positions, requests_of, table)
    want = M.attend(M.decode_pool(raw, False, pages, kv, dim, page), q, positions, requests_of, table, dim ** -0.5)
    check_attend(got, *want, np.maximum(positions + 1, 0), dim)
    assert (got[-4:] == 0).all()


SHARED = [
    # rows of each request in turn, the requests, heads, kv, dim, page, q8, window, half
    ([(0, 0, 40)], 1, 8, 2, 64, 16, False, 0, False), ([(0, 0, 300)], 1, 4, 4, 128, 32, False, 0, False), ([(0, 0, 130)], 1, 14, 2, 64, 64, True, 33, False),
    ([(r, 50 * r, 4) for r in range(20)], 20, 16, 4, 128, 16, True, 0, True), ([(r % 3, 7 * r, 1 + r % 5) for r in range(30)], 3, 6, 2, 96, 16, False, 0, False),
    ([(1, 900, 33), (0, 0, 1), (2, 5, 70), (-1, 3, 5), (3, 3, 3), (1, 10, 2)], 3, 8, 8, 192, 16, False, 100, False), ([(0, 1000, 3)], 1, 16, 2, 256, 128, True, 0, False),
    ([(0, 0, 600), (1, 30, 500)], 2, 5, 1, 64, 16, False, 0, False), ([(0, 500, 17)], 1, 9, 1, 128, 16, False, 0, False), ([(0, 2900, 2), (1, 0, 65)], 2, 24, 8, 256, 16, False, 0, True),
    # more heads than workgroups, rows that fill no block
    ([(0, 20, 3)], 1, 300, 300, 256, 16, False, 0, False), ([(0, 3, 5), (1, 7, 2)], 2, 600, 600, 64, 16, True, 0, False)]


@pytest.mark.parametrize("runs,requests,heads,kv,dim,page,q8,window,half", SHARED)
def test_attend_rows_that_share_requests(ctx, runs, requests, heads, kv, dim, page, q8, window, half):
    """Runs of rows of one request (request, first position, rows), as prompts and drafts have them, of odd lengths and
    beside other requests', some without a token; and the rows of a run in another order."""
    say("attend shared", runs[:6], heads, kv, dim, page, q8, window, half)
    rng = np.random.default_rng(len(runs) + dim + heads)
    requests_of = np.concatenate([np.full(n, r) for r, _, n in runs])
    positions = np.concatenate([np.arange(first, first + n) for _, first, n in runs])
    most = np.ones(requests, int)
    real = (requests_of >= 0) & (requests_of < requests)
    np.maximum.at(most, requests_of[real], positions[real] + 1)
    table, pages = make_tables(rng, most, page)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    pool = M.decode_pool(raw, q8, pages, kv, dim, page)
    positions[rng.random(len(positions)) < 0.05] = -1
    for turn in range(2):
        q = (2 * rng.standard_normal((len(positions), heads, dim))).astype(np.float32)
        got = run_attend(ctx, cache, q, positions, requests_of, table, window=window, half=half, pad=8)
        want = M.attend(pool, q, positions, requests_of, table, dim ** -0.5, window)
        check_attend(got, *want, np.maximum(np.minimum(positions + 1, window or 1 << 30), 0), dim, half)
        assert (got[~real | (positions < 0)] == 0).all()
        positions = positions[::-1].copy()
        requests_of, real = requests_of[::-1].copy(), real[::-1].copy()


@pytest.mark.parametrize("q8", [False, True])
def test_attend_masked_places_have_no_influence(ctx, q8):
    """NaN and infinities behind a row's last token, before its window, and in pages of others."""
    rng = np.random.default_rng(11)
    dim, page, kv, heads = 128, 32, 2, 6
    lengths = np.array([1, 16, 33, 95, 300])
    for window in (0, 40):
        table, pages = make_tables(rng, lengths, page)
        raw = random_pool(rng, q8, pages, kv, dim, page)
        clean = cache_of(ctx, q8, pages, kv, dim, page, raw)
        q = rng.standard_normal((5, heads, dim)).astype(np.float32)
        seen = np.zeros((pages, page), bool)
        for i, n in enumerate(lengths):
            j = np.arange(max(0, n - window) if window else 0, n)
            seen[table[i, j // page], j % page] = True
        dirty = raw.reshape(2, pages, kv, -1).copy()
        if q8:
            scales = dirty[..., page * dim:].view(np.float16).reshape(2, pages, kv, dim // 32, page)
            for which, bad in ((0, np.nan), (1, np.inf)):
                scales[which] = np.where(seen[:, None, None, :], scales[which], np.float16(bad))
        else:
            values = dirty.view(np.float16).reshape(2, pages, kv, page, dim)
            for which, bad in ((0, np.nan), (1, -np.inf)):
                values[which] = np.where(seen[:, None, :, None], values[which], np.float16(bad))
            values[1, ~seen.any(1)] = np.nan
        other = cache_of(ctx, q8, pages, kv, dim, page, dirty.reshape(-1))
        say("attend masked", q8, window)
        a, b = (run_attend(ctx, c, q, lengths - 1, None, table, window=window) for c in (clean, other))
        assert np.array_equal(a, b) and np.isfinite(b).all()


def test_attend_pages_outside_the_cache_count_as_masked(ctx):
    rng = np.random.default_rng(12)
    dim, page, kv, heads = 64, 16, 1, 4
    lengths = [100, 100, 40, 300]
    table, pages = make_tables(rng, lengths, page)
    table[0, [0, 3]], table[1, 6], table[2, :3], table[3, 5:12] = -1, pages, 2**31 - 1, -2**31
    raw = random_pool(rng, False, pages, kv, dim, page)
    cache = cache_of(ctx, False, pages, kv, dim, page, raw)
    q = rng.standard_normal((4, heads, dim)).astype(np.float32)
    positions = np.array([99, 99, 39, 2**31 - 1])              # ... and a position past the table's last token
    say("attend bad pages")
    got = run_attend(ctx, cache, q, positions, None, table)
    want = M.attend(M.decode_pool(raw, False, pages, kv, dim, page), q, positions, None, table, dim ** -0.5)
    check_attend(got, *want, [100, 100, 1, 304], dim)
    assert (got[2] == 0).all()


def test_attend_large_and_extreme_scores(ctx):
    """Scores thousands apart, all equal, of one sign; queries past binary16 and below it; infinities in q."""
    rng = np.random.default_rng(13)
    dim, page, kv = 64, 16, 1
    n = 700
    table, pages = make_tables(rng, [n] * 7, page)
    raw = random_pool(rng, False, pages, kv, dim, page)
    pool = M.decode_pool(raw, False, pages, kv, dim, page)
    cache = cache_of(ctx, False, pages, kv, dim, page, raw)
    q = rng.standard_normal((7, 4, dim)).astype(np.float32)
    q[0] *= 3000
    q[1] = 0
    q[2] *= 1e7
    q[3] *= 1e-9
    q[4] *= np.exp(rng.uniform(-20, 5, (4, dim))).astype(np.float32)
    q[5] = 2.0 ** -140
    say("attend extreme")
    got = run_attend(ctx, cache, q, np.full(7, n - 1), None, table)
    want = M.attend(pool, q, np.full(7, n - 1), None, table, dim ** -0.5)
    # rows whose scores are off by more than a weight can say (1e7 * 64 * 2^-24 ...) are held by their largest weight
    for i in (0, 1, 3, 4, 5, 6):
        check_attend(got[i:i + 1], *(w[i:i + 1] for w in want), [n], dim)
    assert np.isfinite(got[2]).all()
    assert np.abs(got[2] - want[0][2]).max() <= 1e-3           # the winner stands alone: scores are 1e6 apart
    bad = q[:1].copy()
    bad[0, 1, 5], bad[0, 2, 7] = np.inf, np.nan
    got = run_attend(ctx, cache, bad, np.array([n - 1]), None, table[:1])
    assert np.isnan(got[0, 1]).all() and np.isnan(got[0, 2]).all()
    check_attend(got[:, [0, 3]], *(w[:1, [0, 3]] for w in want), [n], dim)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n,every", [(6000, 32), (900, 300)])
def test_attend_weights_far_below_the_largest(ctx, q8, n, every):
    """Tokens that take nearly all the weight and have values of zero (a sequence's first token is often one): the
    result is what the others say, a millionth of the weight each.  Those keep their precision."""
    rng = np.random.default_rng(n)
    dim, page = 64, 16
    table, pages = make_tables(rng, [n], page)
    cache = cache_of(ctx, q8, pages, 1, dim, page, random_pool(rng, q8, pages, 1, dim, page))
    k, v = 0.1 * rng.standard_normal((n, dim)), 1 + 0.5 * rng.random((n, dim))
    k[::every], v[::every] = 0, 0
    k[::every, 3] = 10
    slots = table[0, np.arange(n) // page] * page + np.arange(n) % page
    cache.append(ctx.from_numpy(k), ctx.from_numpy(v), ints(ctx, np.arange(n)), ints(ctx, slots), n)
    ctx.sync()
    q = rng.standard_normal((1, 4, dim)).astype(np.float32)
    q[:, :, 3] = 8 * np.array([1.25, 1.375, 1.4, 1.5])         # scores of 12.5 ... 15: weights of 2^-18 ... 2^-22
    say("attend weak", n, q8)
    got = run_attend(ctx, cache, q, np.array([n - 1]), None, table)
    want = M.attend(M.decode_pool(pool_bytes(cache), q8, pages, 1, dim, page), q, [n - 1], None, table, dim ** -0.5)
    check_attend(got, *want, [n], dim)


def test_attend_is_the_same_every_time_and_with_any_workspace(ctx):
    rng = np.random.default_rng(14)
    lengths = np.array([5000, 12, 800, 0, 3333])
    table, pages = make_tables(rng, lengths, 16)
    raw = random_pool(rng, False, pages, 2, 128, 16)
    cache = cache_of(ctx, False, pages, 2, 128, 16, raw)
    q = rng.standard_normal((5, 8, 128)).astype(np.float32)
    say("attend repeats")
    runs = [run_attend(ctx, cache, q, lengths - 1, None, table, workspace=w) for w in (0, 0xff, 0x7f, None)]
    for r in runs[1:]:
        assert np.array_equal(r, runs[0])


def test_attend_past_32_bit_offsets(ctx):
    """A cache of over 4 GiB: its last pages are read and written where they lie."""
    from jitllm_amd.attention import KvType, PagedAttention, PagedKvCache
    rng = np.random.default_rng(15)
    kv, dim, page, heads = 8, 256, 256, 8
    pages = 2600                                               # 1 MiB a page for k, and for v
    say("attend past 4 GiB")
    cache = PagedKvCache(ctx, KvType.F16, pages, kv, dim, page)
    assert cache.nbytes > 5 << 30
    rows = 40
    x = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float32)
    slots = (pages - 1 - np.arange(rows) // 8 * 500) * page + np.arange(rows) % 8
    table = (pages - 1 - np.arange(5) * 500).reshape(5, 1)
    got_q = run_append(ctx, cache, x, heads, kv, dim, np.arange(rows) % 8, slots, np.zeros(0), False, None, None, 0.0)
    assert np.array_equal(got_q, x[:, :heads])
    out = run_attend(ctx, cache, np.ascontiguousarray(x[7::8, :heads]), np.full(5, 7), None, table)
    kv16 = x[:, heads:].astype(np.float16).astype(np.float64).reshape(5, 8, 2, kv, dim)
    pool = np.zeros((2, 5, kv, page, dim))
    pool[:, :, :, :8] = kv16.transpose(2, 0, 3, 1, 4)
    want = M.attend(pool, x[7::8, :heads], np.full(5, 7), None, np.arange(5).reshape(5, 1), dim ** -0.5)
    check_attend(out, *want, [8] * 5, dim)
    cache.free()


# ---- together ------------------------------------------------------------------------------------

class Layer:
    """A small layer's attention half through the framework, and the same in float64."""

    def __init__(self, ctx, rng, q8, halves, dim=256, heads=4, kv=2, head_dim=64):
        from jitllm_amd import synthetic
        from jitllm_amd.ggml import GGMLType
        self.dim, self.heads, self.kv, self.head_dim = dim, heads, kv, head_dim
        t = GGMLType.Q8_0
        self.raw = [synthetic.weight(t, d, n, seed=int(rng.integers(1 << 30)))
                    for d, n in ((heads * head_dim, dim), (kv * head_dim, dim), (kv * head_dim, dim), (dim, heads * head_dim))]
        self.w = [ctx.load_weight(t, raw, d, n) for raw, (d, n) in
                  zip(self.raw, ((heads * head_dim, dim), (kv * head_dim, dim), (kv * head_dim, dim), (dim, heads * head_dim)))]
        self.dense = [w.dequantize().astype(np.float64) for w in self.w]


@pytest.mark.parametrize("q8,half", [(False, False), (True, False), (False, True)])
def test_decode_steps_through_a_layer(ctx, q8, half):
    """plan -> q|k|v -> append -> attend -> output projection, step after step: prompts of three lengths, decoding,
    one that ends and one that takes its pages; against float64 over the unquantised history."""
    from jitllm_amd.attention import BlockTables, KvType, PagedAttention, PagedKvCache, Rope, RopeStyle, Rows
    from jitllm_amd.projections import QuantizedBatchProjections
    rng = np.random.default_rng(21)
    y = Layer(ctx, rng, q8, True)
    requests, stride, page, pages, max_rows = 4, 6, 16, 14, 64
    w, hd = (y.heads + 2 * y.kv) * y.head_dim, y.heads * y.head_dim
    freq = 1e4 ** (-np.arange(0, y.head_dim, 2) / y.head_dim)
    rope = Rope.of_base(ctx, y.head_dim, 1e4, RopeStyle.HALVES)
    tables = BlockTables(ctx, requests, stride, pages, page, max_rows)
    cache = PagedKvCache(ctx, KvType.Q8_0 if q8 else KvType.F16, pages, y.kv, y.head_dim, page)
    attention = PagedAttention(ctx, max_rows, y.heads, y.kv, y.head_dim)
    proj = QuantizedBatchProjections(ctx, max_rows, max(y.dim, hd), w)
    history = [[] for _ in range(requests)]                    # (k, v) of every token, float64
    steps = [[20, 7, 33, 0], [1, 1, 1, 0], [1, -1, 1, 0], [1, 0, 1, 29], [1, 0, 0, 1], [1, 16, 1, 1]]
    qkv = ctx.float_array(max_rows * w, fill=0.0)
    att = ctx.half_array(max_rows * hd) if half else ctx.float_array(max_rows * hd, fill=0.0)
    for step, fresh in enumerate(steps):
        rows = sum(max(f, 0) for f in fresh)
        x = rng.standard_normal((max_rows, y.dim)).astype(np.float32)
        X, out = ctx.from_numpy(x), ctx.float_array(max_rows * y.dim, fill=0.0)
        say("layer step", step, fresh)
        tables.plan(ints(ctx, fresh))
        proj.fusedQKV(X, qkv, y.w[0], y.w[1], y.w[2], rows)
        cache.append(Rows(qkv, w, hd), Rows(qkv, w, hd + y.kv * y.head_dim), tables.positions, tables.slots, rows, rope=rope,
                     q=Rows(qkv, w), heads=y.heads)
        attention.attend(cache, Rows(qkv, w), rows, tables.positions, tables.table, att, requests=requests, rowRequests=tables.rowRequests)
        proj.projection(att, out, y.w[3], hd, y.dim, False, rows)
        ctx.sync()
        got = out.get().reshape(max_rows, y.dim)[:rows]
        row = 0
        for r, f in enumerate(fresh):
            if f < 0:
                history[r] = []
            for _ in range(max(f, 0)):
                xx = x[row].astype(np.float64)
                pos = np.array([len(history[r])])
                q, k, v = ((m @ xx).reshape(1, -1, y.head_dim) for m in y.dense[:3])
                q, k = M.rotate(q, pos, freq, True), M.rotate(k, pos, freq, True)
                history[r].append((k[0], v[0]))
                K, V = (np.array([h[i] for h in history[r]]) for i in (0, 1))
                o = np.zeros((y.heads, y.head_dim))
                for h in range(y.heads):
                    s = K[:, h // 2] @ q[0, h] * y.head_dim ** -0.5
                    p = np.exp(s - s.max())
                    o[h] = (p / p.sum()) @ V[:, h // 2]
                want = y.dense[3] @ o.reshape(-1)
                # fp16 products inside the projections (2e-3 of the magnitude, as the path is held to) and a cache
                # of 11 or 7 bits, whose scores move by up to that share of a few units
                size = np.abs(y.dense[3]) @ np.abs(o.reshape(-1))
                assert np.abs(got[row] - want).max() <= (0.15 if q8 else 0.03) * size.max(), (step, r, row)
                row += 1
    assert tables.lengths.get().tolist() == [25, 16, 37, 31]   # 20 + 5, 16, 33 + 4, 29 + 2


# ---- graphs, streams, contexts -------------------------------------------------------------------

@pytest.mark.parametrize("q8", [False, True])
def test_a_captured_step_replayed_while_lengths_grow(ctx, q8):
    """plan, append and attend recorded once; every replay after the program's own eager work (inputs uploaded, another
    call through the same workspace, a wait), held to the same step made eagerly over a copy of the state."""
    import bench
    from jitllm_amd.attention import BlockTables, KvType, PagedAttention, PagedKvCache, Rope, Rows
    hip = bench.Hip()
    rng = np.random.default_rng(31)
    requests, stride, page, pages, max_rows, heads, kv, dim = 5, 80, 16, 260, 8, 8, 2, 64
    w = (heads + 2 * kv) * dim
    rope = Rope.of_base(ctx, dim, 1e4)
    attention = PagedAttention(ctx, max_rows, heads, kv, dim)

    class Side:
        def __init__(self):
            self.tables = BlockTables(ctx, requests, stride, pages, page, max_rows)
            self.cache = PagedKvCache(ctx, KvType.Q8_0 if q8 else KvType.F16, pages, kv, dim, page)
            self.fresh, self.qkv = ints(ctx, np.zeros(requests)), ctx.float_array(max_rows * w, fill=0.0)
            self.out = ctx.float_array(max_rows * heads * dim, fill=7.0)

        def step(self):
            t = self.tables
            t.plan(self.fresh)
            self.cache.append(Rows(self.qkv, w, heads * dim), Rows(self.qkv, w, (heads + kv) * dim), t.positions, t.slots, max_rows, rope=rope,
                              q=Rows(self.qkv, w), heads=heads)
            attention.attend(self.cache, Rows(self.qkv, w), max_rows, t.positions, t.table, self.out, requests=requests, rowRequests=t.rowRequests)

    a, b = Side(), Side()
    lengths = np.array([1100, 3, 0, 700, 16])                  # long enough to be cut, short, none, a page's end
    order = rng.permutation(pages)
    need = -(-lengths // page)
    table = np.full((requests, stride), -1)
    table[np.arange(stride) < need[:, None]] = order[:need.sum()]
    raw = random_pool(rng, q8, pages, kv, dim, page)
    raw_at = ctx.raw_buffer(raw.nbytes)
    raw_at.upload(raw)
    for side in (a, b):
        side.tables.table.set(table), side.tables.lengths.set(lengths)
        ring = np.full(pages, -1)
        ring[:pages - need.sum()] = order[need.sum():]
        side.tables.pageRing.set(ring), side.tables.freePages.set([0, pages - need.sum()])
        from jitllm_amd import _lib as L
        host = raw.copy()
        L.check(ctx._lib.jl_upload(ctx.handle, ctx._lib.jl_kv_cache_memory(side.cache.handle), host.ctypes.data, host.nbytes))
    say("captured step", q8)
    a.fresh.set([0] * requests)
    a.step()                                                   # warmed up: nothing new
    ctx.sync()
    exe = hip.capture(ctx.stream, a.step)
    other = PagedKvCache(ctx, KvType.F16, 40, kv, dim, page, memory=raw_at if not q8 else None)
    try:
        for n, fresh in enumerate([[1, 1, 0, 1, 1], [1, 1, 2, 1, 1], [1, -1, 1, 1, 0], [1, 0, 1, 1, 5], [1, 3, 1, -1, 1], [1, 1, 1, 0, 1]]):
            x = rng.standard_normal((max_rows, w)).astype(np.float32)
            for side in (a, b):
                side.fresh.set(fresh), side.qkv.set(x), side.out.init(7.0)
            b.step()
            q = ctx.float_array(heads * dim, fill=0.5)
            attention.attend(other, q, 1, ints(ctx, [600]), ints(ctx, np.arange(40)), ctx.float_array(heads * dim), requests=1)
            ctx.sync()
            hip.launch(exe, ctx.stream)
            ctx.sync()
            assert np.array_equal(a.out.get().view(np.uint32), b.out.get().view(np.uint32)), n
            for name in NAMES:
                assert np.array_equal(getattr(a.tables, name).get(), getattr(b.tables, name).get()), (n, name)
            rows = sum(max(f, 0) for f in fresh)
            assert (a.out.get().reshape(max_rows, -1)[rows:] == 0).all()       # padding: nothing to read
    finally:
        hip.destroy_graph(exe)


def test_two_contexts_at_once(ctx):
    """Two streams, a workspace each, calls in flight side by side: each is what it is alone."""
    from jitllm_amd.attention import KvType, PagedAttention, PagedKvCache
    from jitllm_amd.runtime import Context
    rng = np.random.default_rng(41)
    lengths = np.array([6000, 5, 900, 2500])
    table, pages = make_tables(rng, lengths, 16)
    raw = random_pool(rng, False, pages, 4, 128, 16)
    q = [rng.standard_normal((4, 16, 128)).astype(np.float32) for _ in range(2)]
    say("two contexts")
    with Context(0) as second:
        sides = []
        for c, x in ((ctx, q[0]), (second, q[1])):
            memory = c.raw_buffer(raw.nbytes)
            memory.upload(raw)
            sides.append((c, PagedKvCache(c, KvType.F16, pages, 4, 128, 16, memory=memory), PagedAttention(c, 4, 16, 4, 128), c.from_numpy(x),
                          c.float_array(4 * 16 * 128), ints(c, lengths - 1), ints(c, table)))
        alone = []
        for c, cache, attention, x, out, positions, t in sides:
            attention.attend(cache, x, 4, positions, t, out, requests=4)
            c.sync()
            alone.append(out.get())
        for _ in range(20):
            for c, cache, attention, x, out, positions, t in sides:
                for _ in range(3):
                    attention.attend(cache, x, 4, positions, t, out, requests=4)
            for side, want in zip(sides, alone):
                side[0].sync()
                assert np.array_equal(side[4].get(), want)
        for side in sides:
            side[1].free()
        del sides, cache, attention, x, out, positions, t, memory
    want = M.attend(M.decode_pool(raw, False, pages, 4, 128, 16), q[0], lengths - 1, None, table, 128 ** -0.5)
    check_attend(alone[0].astype(np.float64).reshape(4, 16, 128), *want, lengths, 128)


def test_one_workspace_for_calls_of_several_shapes(ctx):
    """Layers of different heads share the workspace of the widest; what one call leaves in it is the next one's zero."""
    from jitllm_amd.attention import PagedAttention
    rng = np.random.default_rng(43)
    wide = PagedAttention(ctx, 8, 64, 2, 256)
    for lengths, heads, kv, dim, q8 in (([3000, 40], 64, 2, 256, False), ([2000], 8, 1, 64, False), ([5, 900, 1800], 12, 4, 128, True), ([4000], 6, 6, 96, False)) * 2:
        table, pages = make_tables(rng, lengths, 32)
        raw = random_pool(rng, q8, pages, kv, dim, 32)
        cache = cache_of(ctx, q8, pages, kv, dim, 32, raw)
        attention = PagedAttention(ctx, 8, heads, kv, dim)
        assert attention.workspace.nbytes <= wide.workspace.nbytes
        attention.workspace = wide.workspace
        q = rng.standard_normal((len(lengths), heads, dim)).astype(np.float32)
        say("shared workspace", lengths, heads, kv, dim, q8)
        got = run_attend(ctx, cache, q, np.array(lengths) - 1, None, table, attention=attention)
        want = M.attend(M.decode_pool(raw, q8, pages, kv, dim, 32), q, np.array(lengths) - 1, None, table, dim ** -0.5)
        check_attend(got, *want, lengths, dim)


def test_attend_thousands_of_short_rows(ctx):
    rng = np.random.default_rng(44)
    rows, page, dim = 5000, 16, 64
    lengths = rng.integers(0, 4, rows)
    lengths[4321] = 200
    table, pages = make_tables(rng, lengths, page)
    raw = random_pool(rng, False, pages, 1, dim, page)
    cache = cache_of(ctx, False, pages, 1, dim, page, raw)
    q = rng.standard_normal((rows, 2, dim)).astype(np.float32)
    say("attend thousands of rows")
    got = run_attend(ctx, cache, q, lengths - 1, None, table)
    want = M.attend(M.decode_pool(raw, False, pages, 1, dim, page), q, lengths - 1, None, table, dim ** -0.5)
    check_attend(got, *want, lengths, dim)


# ---- rows of one request that go together: what none of them, or only some, may see ---------------

def poisoned(raw, q8, pages, kv, dim, page, at, which, bad, element=None):
    """The cache's bytes with `bad` in k (0) or v (1) at slots `at`: everywhere, or at one element (a block's scale)."""
    dirty = raw.copy().reshape(2, pages, kv, -1)
    for slot in np.atleast_1d(at):
        if q8:
            scales = dirty[..., page * dim:].view(np.float16).reshape(2, pages, kv, dim // 32, page)
            scales[which, slot // page, :, slice(None) if element is None else element // 32, slot % page] = bad
            dirty[..., page * dim:] = scales.reshape(2, pages, kv, -1).view(np.uint8)
        else:
            dirty.view(np.float16).reshape(2, pages, kv, page, dim)[which, slot // page, :, slot % page, slice(None) if element is None else element] = bad
    return dirty.reshape(-1)


def check_where_finite(got, want, weight, reach, lengths, dim):
    """check_attend where the definition says a number; no number where it says none."""
    fine = np.isfinite(want)
    assert not np.isfinite(got[~fine]).any()
    zero = lambda y: np.where(fine, y, 0)                      # noqa: E731
    check_attend(zero(got), zero(want), zero(weight), np.where(np.isfinite(reach), reach, 0), lengths, dim)


GAPS = [
    # positions of one request's rows, window, heads, kv, dim, page
    ([10, 1000], 16, 8, 2, 128, 16), ([700, 5, 701, 3000], 40, 8, 4, 64, 32), ([900, 899, 100, 101, 400, 2, 1, 0], 7, 6, 3, 96, 64),
    ([50, 2000, 50, 2000, 50], 33, 4, 1, 192, 16), ([31, 95, 159], 1, 4, 2, 256, 128), (list(range(100)) + list(range(3000, 3030)), 64, 4, 2, 64, 16)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("positions,window,heads,kv,dim,page", GAPS)
def test_attend_shared_rows_with_a_gap_between_their_windows(ctx, positions, window, heads, kv, dim, page, q8):
    """Rows of one request further apart than the window: what lies between is no row's, and has no influence."""
    say("attend gap", positions[:8], window, heads, kv, dim, page, q8)
    rng = np.random.default_rng(len(positions) + dim)
    positions = np.array(positions)
    rows, n = len(positions), int(positions.max()) + 1
    table, pages = make_tables(rng, [n], page)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    seen = np.zeros(pages * page, bool)
    for i in positions:
        j = np.arange(max(0, i - window + 1), i + 1)
        seen[table[0, j // page] * page + j % page] = True
    dirty = poisoned(raw, q8, pages, kv, dim, page, np.flatnonzero(~seen)[::2], 1, np.nan)
    dirty = poisoned(dirty, q8, pages, kv, dim, page, np.flatnonzero(~seen)[1::2], 1, -np.inf)
    dirty = poisoned(dirty, q8, pages, kv, dim, page, np.flatnonzero(~seen), 0, np.inf)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    got = run_attend(ctx, cache_of(ctx, q8, pages, kv, dim, page, dirty), q, positions, np.zeros(rows, int), table, window=window)
    want = M.attend(M.decode_pool(raw, q8, pages, kv, dim, page), q, positions, np.zeros(rows, int), table, dim ** -0.5, window)
    check_attend(got, *want, np.minimum(positions + 1, window), dim)


LATER = [
    # first position, rows, window, heads, kv, dim, page, poisoned tokens, element of v (None: all)
    (0, 40, 0, 8, 2, 128, 16, [17], None), (0, 40, 0, 8, 2, 128, 16, [5, 30], 77), (20, 64, 0, 4, 4, 64, 32, [50], 9), (0, 33, 9, 6, 3, 96, 64, [12], 70),
    (0, 33, 0, 6, 2, 96, 16, [20], None), (1000, 5, 0, 8, 1, 192, 16, [1002], 150), (3000, 3, 100, 8, 2, 256, 128, [2901, 3001], 200), (6000, 4, 0, 4, 1, 64, 16, [6002], None),
    (60, 10, 3, 16, 1, 256, 16, [64], None), (100, 16, 0, 1, 1, 128, 16, [107, 115], 0)]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("first,rows,window,heads,kv,dim,page,tokens,element", LATER)
def test_attend_shared_rows_keep_to_their_own_tokens(ctx, first, rows, window, heads, kv, dim, page, tokens, element, bad, q8):
    """An infinity or NaN in v at a token that some rows of a prompt see: those lose the columns that it stands in, the
    others -- before it, or past a window behind it -- are what they are without it."""
    say("attend later", first, rows, window, heads, kv, dim, page, tokens, element, bad, q8)
    rng = np.random.default_rng(first + rows + dim)
    positions, requests_of = np.arange(first, first + rows), np.zeros(rows, int)
    table, pages = make_tables(rng, [first + rows], page)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    at = [table[0, t // page] * page + t % page for t in tokens]
    dirty = poisoned(raw, q8, pages, kv, dim, page, at, 1, bad, element)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    clean, got = (run_attend(ctx, cache_of(ctx, q8, pages, kv, dim, page, r), q, positions, requests_of, table, window=window) for r in (raw, dirty))
    pool = M.decode_pool(raw, q8, pages, kv, dim, page)
    out, weight, reach = M.attend(pool, q, positions, requests_of, table, dim ** -0.5, window)
    lost = np.zeros((rows, 1, dim), bool)
    columns = slice(None) if element is None else slice(element // 32 * 32, element // 32 * 32 + 32) if q8 else element
    for t in tokens:
        sees = (positions >= t) & (positions < t + window if window else True)
        lost[sees, :, columns] = True
    lost = np.broadcast_to(lost, out.shape)
    assert lost.any() and not np.isfinite(got[lost]).any()
    assert np.array_equal(got[~lost], clean[~lost])
    check_attend(np.where(lost, 0, got), np.where(lost, 0, out), np.where(lost, 0, weight), reach, np.minimum(positions + 1, window or 1 << 30), dim)


def test_attend_shared_rows_over_8_bit_blocks_whose_values_overflow(ctx):
    """Finite scales whose products with the bytes are infinite in binary16, and scales just below those."""
    rng = np.random.default_rng(51)
    heads, kv, dim, page, rows = 4, 2, 64, 16, 24
    positions, requests_of = np.arange(rows), np.zeros(rows, int)
    table, pages = make_tables(rng, [rows], page)
    raw = random_pool(rng, True, pages, kv, dim, page)
    at = [table[0, t // page] * page + t % page for t in (3, 13, 20)]
    dirty = poisoned(poisoned(raw, True, pages, kv, dim, page, at[:1], 1, 500.0), True, pages, kv, dim, page, at[1:], 1, 5000.0)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    say("attend 8-bit overflow")
    got = run_attend(ctx, cache_of(ctx, True, pages, kv, dim, page, dirty), q, positions, requests_of, table)
    pool = M.decode_pool(dirty, True, pages, kv, dim, page)
    with np.errstate(invalid="ignore"):
        want = M.attend(pool, q, positions, requests_of, table, dim ** -0.5)
    assert np.isfinite(want[0][:13]).all() and not np.isfinite(want[0][13:]).all()
    check_where_finite(got, *want, positions + 1, dim)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("window", [0, 50])
def test_attend_shared_rows_over_bad_pages_and_past_the_table(ctx, window, q8):
    """Pages outside the cache count as masked, positions past the table read what it holds, some rows are of no request."""
    rng = np.random.default_rng(61)
    dim, page, kv, heads = 96, 16, 2, 4
    table, pages = make_tables(rng, [300, 70], page)
    table[0, [0, 3, 17]], table[1, 1:3], table[0, 9:12] = -1, 2**31 - 1, pages
    raw = random_pool(rng, q8, pages, kv, dim, page)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    end = table.shape[1] * page
    positions = np.concatenate([np.arange(30), np.arange(40, 60), np.arange(140, 200), [end - 1, end, end + 1, end + 40, end + 49, end + 50, 2**31 - 1],
                                np.arange(10, 20), [3, -1, 4, 5, -2**31, 6]])
    requests_of = np.concatenate([np.zeros(117, int), np.ones(10, int), [0, 0, 0, -1, 1, 2]])
    q = rng.standard_normal((len(positions), heads, dim)).astype(np.float32)
    say("attend shared bad pages", window, q8)
    got = run_attend(ctx, cache, q, positions, requests_of, table, window=window)
    want = M.attend(M.decode_pool(raw, q8, pages, kv, dim, page), q, positions, requests_of, table, dim ** -0.5, window)
    check_attend(got, *want, np.clip(positions + 1, 0, end), dim)
    assert (got[want[1].max((1, 2)) == 0] == 0).all()


@pytest.mark.parametrize("q8", [False, True])
def test_attend_shared_rows_of_extreme_queries(ctx, q8):
    """Rows that go together, each with scores of another size: thousands apart, all equal, below binary16; one with an
    infinity and one with NaN in a head, which are those heads' alone."""
    rng = np.random.default_rng(62)
    dim, page, kv, heads, rows, n = 64, 16, 2, 4, 24, 500
    table, pages = make_tables(rng, [n], page)
    raw = random_pool(rng, q8, pages, kv, dim, page)
    positions, requests_of = np.arange(n - rows, n), np.zeros(rows, int)
    q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
    q *= np.array([1, 3000, 0, 1e-9, 2.0 ** -140, 40], np.float32)[np.arange(rows) % 6, None, None]
    q[7::6] *= np.exp(rng.uniform(-20, 5, (len(q[7::6]), heads, dim))).astype(np.float32)
    cache = cache_of(ctx, q8, pages, kv, dim, page, raw)
    say("attend shared extreme", q8)
    got = run_attend(ctx, cache, q, positions, requests_of, table)
    pool = M.decode_pool(raw, q8, pages, kv, dim, page)
    out, weight, reach = M.attend(pool, q, positions, requests_of, table, dim ** -0.5)
    # A weight is two binary16 parts of 2^13 times it, the second one off by 2^-25 however small the weight is: n tokens are
    # off by n 2^-38 max |v| together, which is more than check_attend's share of sum p |v| where the token with nearly all
    # of the weight has a v of 0 (an 8-bit block's often is).  Through that check's n + 64 half steps of 2^-24, 2^-14 max |v|
    # more of sum p |v| stand for it.
    want = out, weight + 2.0 ** -14 * np.abs(pool[1]).max(), reach
    check_attend(got, *want, positions + 1, dim)
    bad = q.copy()
    bad[5, 1, 5], bad[18, 2, 7], bad[19, 2, 7] = np.inf, np.nan, -np.inf
    lost = np.zeros((rows, heads), bool)
    lost[[5, 18, 19], [1, 2, 2]] = True
    got = run_attend(ctx, cache, bad, positions, requests_of, table)
    assert np.isnan(got[lost]).all()
    check_attend(np.where(lost[..., None], 0, got), *(np.where(lost[..., None] if w.ndim == 3 else lost, 0, w) for w in want), positions + 1, dim)


def test_attend_shared_rows_are_the_same_every_time_and_with_any_workspace(ctx):
    """Drafts and prompts, cut into parts and whole."""
    rng = np.random.default_rng(63)
    for rows, first, heads, kv, dim, q8 in ((4, 7000, 8, 2, 128, False), (3, 3000, 4, 4, 256, True), (90, 10, 6, 2, 64, False), (16, 2500, 1, 1, 64, True)):
        table, pages = make_tables(rng, [first + rows], 16)
        cache = cache_of(ctx, q8, pages, kv, dim, 16, random_pool(rng, q8, pages, kv, dim, 16))
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        say("attend shared repeats", rows, first, heads, kv, dim, q8)
        runs = [run_attend(ctx, cache, q, np.arange(first, first + rows), np.zeros(rows, int), table, workspace=w) for w in (0, 0xff, 0x7f, None)]
        for r in runs[1:]:
            assert np.array_equal(r, runs[0])


@pytest.mark.parametrize("q8", [False, True])
def test_a_captured_step_whose_rows_go_together(ctx, q8):
    """A step of up to 24 rows for 3 requests, recorded once: prompts, drafts, single tokens, padding; every replay after
    eager work through the same workspace, against the same step made eagerly and against float64."""
    import bench
    from jitllm_amd.attention import BlockTables, KvType, PagedAttention, PagedKvCache, Rows
    hip = bench.Hip()
    rng = np.random.default_rng(64)
    requests, stride, page, pages, max_rows, heads, kv, dim = 3, 12, 16, 30, 24, 4, 2, 64
    w = (heads + 2 * kv) * dim
    attention = PagedAttention(ctx, max_rows, heads, kv, dim)

    class Side:
        def __init__(self):
            self.tables = BlockTables(ctx, requests, stride, pages, page, max_rows)
            self.cache = PagedKvCache(ctx, KvType.Q8_0 if q8 else KvType.F16, pages, kv, dim, page, memory=ctx.raw_buffer(2 * pages * kv * M.part_bytes(q8, dim, page)))
            self.cache.memory.upload(np.full(self.cache.nbytes, 0xff, np.uint8))           # NaN where nothing is written
            self.fresh, self.qkv = ints(ctx, np.zeros(requests)), ctx.float_array(max_rows * w, fill=0.0)
            self.out = ctx.float_array(max_rows * heads * dim, fill=7.0)

        def step(self):
            t = self.tables
            t.plan(self.fresh)
            self.cache.append(Rows(self.qkv, w, heads * dim), Rows(self.qkv, w, (heads + kv) * dim), t.positions, t.slots, max_rows)
            attention.attend(self.cache, Rows(self.qkv, w), max_rows, t.positions, t.table, self.out, requests=requests, rowRequests=t.rowRequests)

    a, b = Side(), Side()
    say("captured step, rows together", q8)
    a.fresh.set([0] * requests)
    a.step()
    ctx.sync()
    exe = hip.capture(ctx.stream, a.step)
    try:
        for n, fresh in enumerate([[20, 3, 0], [1, 1, 1], [4, 4, 4], [1, -1, 9], [5, 0, 1], [24, 0, 0], [1, 17, 5], [0, 0, 0]]):
            x = rng.standard_normal((max_rows, w)).astype(np.float32)
            for side in (a, b):
                side.fresh.set(fresh), side.qkv.set(x), side.out.init(7.0)
            b.step()
            ctx.sync()
            hip.launch(exe, ctx.stream)
            ctx.sync()
            got = a.out.get().reshape(max_rows, heads, dim)
            assert np.array_equal(got.view(np.uint32).reshape(-1), b.out.get().view(np.uint32)), n
            positions, rows_of, table = (getattr(a.tables, k).get() for k in ("positions", "rowRequests", "table"))
            want = M.attend(M.decode_pool(pool_bytes(a.cache), q8, pages, kv, dim, page), x[:, :heads * dim].reshape(max_rows, heads, dim), positions,
                            rows_of, table.reshape(requests, stride), dim ** -0.5)
            check_attend(got.astype(np.float64), *want, positions + 1, dim)
            assert (got[positions < 0] == 0).all()
    finally:
        hip.destroy_graph(exe)


def test_two_contexts_of_rows_that_go_together(ctx):
    """A draft's rows on one stream, a prompt's on another, one cache: each is what it is alone."""
    from jitllm_amd.attention import KvType, PagedAttention, PagedKvCache
    from jitllm_amd.runtime import Context
    rng = np.random.default_rng(65)
    n = 6000
    table, pages = make_tables(rng, [n], 16)
    raw = random_pool(rng, False, pages, 4, 128, 16)
    memory = ctx.raw_buffer(raw.nbytes)
    memory.upload(raw)
    cache = PagedKvCache(ctx, KvType.F16, pages, 4, 128, 16, memory=memory)
    say("two contexts, rows together")
    with Context(0) as second:
        sides = []
        for c, positions in ((ctx, np.arange(n - 4, n)), (second, np.arange(100))):
            rows = len(positions)
            q = rng.standard_normal((rows, 16, 128)).astype(np.float32)
            sides.append((c, PagedAttention(c, rows, 16, 4, 128), c.from_numpy(q), c.float_array(rows * 16 * 128), ints(c, positions), ints(c, table),
                          ints(c, np.zeros(rows)), rows, q, positions))
        for _ in range(20):
            for c, attention, x, out, positions, t, requests_of, rows, _, _ in sides:
                for _ in range(3):
                    attention.attend(cache, x, rows, positions, t, out, requests=1, rowRequests=requests_of)
            for side in sides:
                side[0].sync()
        pool = M.decode_pool(raw, False, pages, 4, 128, 16)
        for side in sides:
            rows, q, positions = side[7:]
            got = side[3].get().astype(np.float64).reshape(rows, 16, 128)
            check_attend(got, *M.attend(pool, q, positions, np.zeros(rows, int), table, 128 ** -0.5), positions + 1, 128)
            assert np.array_equal(got, run_attend(ctx, cache, q, positions, np.zeros(rows, int), table))
        del sides, side, attention, x, out, t, requests_of, c


def test_one_workspace_for_rows_together_and_alone(ctx):
    from jitllm_amd.attention import PagedAttention
    rng = np.random.default_rng(66)
    shared = PagedAttention(ctx, 64, 32, 4, 256)
    for rows, first, requests, heads, kv, dim, q8 in ((4, 3000, 1, 16, 4, 256, False), (2, 2500, 2, 8, 2, 128, True), (33, 0, 1, 8, 8, 64, True), (1, 4000, 1, 32, 4, 192, False)) * 2:
        requests_of = np.arange(rows) % requests
        positions = first + np.arange(rows) // requests
        table, pages = make_tables(rng, positions + 1, 32, requests_of, requests)
        raw = random_pool(rng, q8, pages, kv, dim, 32)
        attention = PagedAttention(ctx, 64, heads, kv, dim)
        attention.workspace = shared.workspace
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        say("one workspace, together and alone", rows, first, requests, heads, kv, dim, q8)
        got = run_attend(ctx, cache_of(ctx, q8, pages, kv, dim, 32, raw), q, positions, requests_of, table, attention=attention)
        check_attend(got, *M.attend(M.decode_pool(raw, q8, pages, kv, dim, 32), q, positions, requests_of, table, dim ** -0.5), positions + 1, dim)


# ---- what the write promises of its precision ----------------------------------------------------

def append_error(x, positions, freq, halves):
    """What double precision leaves of heads [rows][heads][dim] that turned, next to their float64 form: the series of sine
    and cosine end below 2^-45, an angle is rounded four times (product, turns, their fraction, radians) and the products
    and sums, a norm's too, make no 2^-47 together, all of it of |a| + |b| of a pair (at most sqrt 2 times what the pair
    has behind the turn as before it)."""
    slack = np.abs(x) * 2.0 ** -47
    pairs = len(freq)
    first = np.arange(pairs) if halves else 2 * np.arange(pairs)
    second = first + pairs if halves else first + 1
    both = 2 ** 0.5 * (np.abs(x[..., first]) + np.abs(x[..., second])) * (2.0 ** -45 + 2.0 ** -47 + 4 * 2.0 ** -53 * np.abs(positions[:, None, None] * freq))
    slack[..., first], slack[..., second] = both, both
    return slack


@pytest.mark.parametrize("halves", [False, True])
def test_append_where_products_cancel(ctx, halves):
    """a cos - b sin next to zero: the absolute error of the cosine and the sine, in every eighth of a turn."""
    dim, page, rows = 64, 16, 33
    pairs = dim // 2
    freq = np.pi / 4 * (1 + np.linspace(-1e-9, 1e-9, pairs))
    positions = np.arange(rows)
    angle = positions.astype(np.longdouble)[:, None] * freq.astype(np.longdouble)
    cos, sin = np.cos(angle), np.sin(angle)
    a, b = np.ones((rows, pairs)), np.where(cos * sin > 0, 1.0, -1.0)        # near odd eighths |cos| = |sin|
    x = np.zeros((rows, 3, dim), np.float32)
    first = np.arange(pairs) if halves else 2 * np.arange(pairs)
    second = first + pairs if halves else first + 1
    x[:, 0, first], x[:, 0, second] = a, b
    cache = cache_of(ctx, False, 3, 1, dim, page, np.zeros(2 * 3 * M.part_bytes(False, dim, page), np.uint8))
    say("append cancel", halves)
    got = run_append(ctx, cache, x, 1, 1, dim, positions, np.arange(rows), freq, halves, None, None, 0.0)[:, 0]
    want = np.zeros((rows, dim), np.longdouble)
    want[:, first], want[:, second] = a * cos - b * sin, a * sin + b * cos
    slack = append_error(want[:, None].astype(np.float64), positions, freq, halves)[:, 0]
    assert (np.abs(got - want) <= slack + ULP * np.abs(want)).all(), float(np.max(np.abs(got - want) - ULP * np.abs(want)))


@pytest.mark.parametrize("rows,heads,kv,dim,page,q8,halves,turned,norm,context", [a for a in APPENDS if a[1]])
def test_append_rounds_once(ctx, rows, heads, kv, dim, page, q8, halves, turned, norm, context):
    """q is the fp32 value of the float64 form; k and v that, rounded to the cache's type.  (A neighbour where the error of
    double precision reaches over a border: roundings are monotonic.)"""
    say("append rounds", rows, heads, kv, dim, page, q8, halves, turned, norm, context)
    rng = np.random.default_rng(rows * dim + page)
    pages = rows // page + 1
    x = rng.standard_normal((rows, heads + 2 * kv, dim)).astype(np.float32)
    x[:, :, 3] *= 20
    cache = cache_of(ctx, q8, pages, kv, dim, page, np.zeros(2 * pages * kv * M.part_bytes(q8, dim, page), np.uint8))
    slots, positions = rng.permutation(pages * page)[:rows], rng.integers(0, context, rows)
    freq = 500000.0 ** (-np.arange(0, turned, 2) / turned) if turned else np.zeros(0)
    qn, kn = (1 + 0.1 * rng.standard_normal(dim).astype(np.float32) for _ in range(2)) if norm else (None, None)
    eps = np.float32(1e-6)
    got_q = run_append(ctx, cache, x, heads, kv, dim, positions, slots, freq, halves, qn, kn, eps)
    ends = []
    for part, w in ((x[:, :heads], qn), (x[:, heads:heads + kv], kn)):
        y = M.rotate(part, positions, freq, halves, w, float(eps))
        slack = append_error(y, positions, freq, halves) if turned or norm else 0
        ends.append([(y + side * slack).astype(np.float32) for side in (-1, 1)])
    assert ((ends[0][0] <= got_q) & (got_q <= ends[0][1])).all()
    after = M.decode_pool(pool_bytes(cache), q8, pages, kv, dim, page)
    kept = after[:, slots // page, :, slots % page]                                  # [rows][2][kv][dim]
    for got, (low, high) in ((kept[:, 0], ends[1]), (kept[:, 1], [x[:, heads + kv:]] * 2)):
        if not q8:
            assert ((low.astype(np.float16) <= got) & (got <= high.astype(np.float16))).all()
            continue
        blocks = low.reshape(-1, 32)
        sure = (blocks == high.reshape(-1, 32)).all(-1)                              # (fp32 division and rint, as the blocks are defined)
        d = np.minimum(np.abs(blocks).max(-1, keepdims=True) / np.float32(127), np.float32(65504)).astype(np.float16).astype(np.float32)
        want = (np.clip(np.rint(blocks / d), -127, 127) * d).astype(np.float16)
        assert sure.mean() > 0.9 and np.array_equal(got.reshape(-1, 32)[sure], want[sure].astype(np.float64))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attend_shared_rows_over_keys_that_are_not_finite(ctx, bad, q8):
    """... and in k: rows that see the token have no number, the others are what they are without it."""
    rng = np.random.default_rng(67)
    heads, kv, dim, page = 4, 2, 128, 16
    for first, rows, window, token in ((0, 40, 0, 21), (0, 40, 6, 21), (2000, 7, 50, 2003), (2000, 7, 50, 1953)):
        positions, requests_of = np.arange(first, first + rows), np.zeros(rows, int)
        table, pages = make_tables(rng, [first + rows], page)
        raw = random_pool(rng, q8, pages, kv, dim, page)
        dirty = poisoned(raw, q8, pages, kv, dim, page, [table[0, token // page] * page + token % page], 0, bad)
        q = rng.standard_normal((rows, heads, dim)).astype(np.float32)
        say("attend keys", first, rows, window, token, bad, q8)
        clean, got = (run_attend(ctx, cache_of(ctx, q8, pages, kv, dim, page, r), q, positions, requests_of, table, window=window) for r in (raw, dirty))
        sees = (positions >= token) & (positions < token + window if window else True)
        assert sees.any() and (~sees).any() and np.isnan(got[sees]).all()
        # (the others' maximum may be brought forward with that of the rows beside them: the same but for rounding)
        out, weight, reach = M.attend(M.decode_pool(raw, q8, pages, kv, dim, page), q, positions, requests_of, table, dim ** -0.5, window)
        for r in (clean, got):
            check_attend(r[~sees], out[~sees], weight[~sees], reach[~sees], np.minimum(positions + 1, window or 1 << 30)[~sees], dim)

"""The paged key-value cache's calls without a GPU: what they refuse, and in which words.  Every check of an
argument comes before the first call of the HIP runtime, so a context that is only memory serves."""
import ctypes as C

import numpy as np
import pytest

import kv_models as M


@pytest.fixture(scope="module")
def L():
    from jitllm_amd import _lib
    _lib.load()
    return _lib


@pytest.fixture(scope="module")
def lib(L):
    return L.load()


@pytest.fixture(scope="module")
def memory():
    """1 KiB on a 64-byte boundary: addresses that are checked and never followed."""
    raw = C.create_string_buffer(1088)
    at = (C.addressof(raw) + 63) // 64 * 64
    yield at
    del raw


@pytest.fixture(scope="module")
def ctx():
    raw = C.create_string_buffer(4096)                          # a context of device 0
    yield C.addressof(raw)
    del raw


@pytest.fixture(scope="module")
def cache(L, lib, ctx, memory):
    h = C.c_void_p()
    assert lib.jl_kv_cache_wrap(ctx, memory, L.JL_KV_F16, 4, 2, 128, 16, C.byref(h)) == L.JL_OK
    assert lib.jl_kv_cache_memory(h) == memory
    yield h
    assert lib.jl_kv_cache_free(h) == L.JL_OK


def said(lib):
    return lib.jl_last_error().decode()


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_cache_bytes(L, lib, dim, page):
    assert lib.jl_kv_cache_bytes(L.JL_KV_F16, 7, 3, dim, page) == 2 * 7 * 3 * M.part_bytes(False, dim, page)
    assert lib.jl_kv_cache_bytes(L.JL_KV_Q8_0, 7, 3, dim, page) == 2 * 7 * 3 * M.part_bytes(True, dim, page)
    assert lib.jl_kv_cache_bytes(L.JL_KV_F16, 2**22, 8, dim, page) == 2 * 2**22 * 8 * 2 * dim * page


@pytest.mark.parametrize("args,status,words", [
    ((0, 4, 2, 128, 16), "UNSUPPORTED", "type 0"), ((2, 4, 2, 128, 16), "UNSUPPORTED", "type 2"), ((1, 4, 2, 80, 16), "UNSUPPORTED", "80 values"),
    ((1, 4, 2, 0, 16), "UNSUPPORTED", "0 values"), ((8, 4, 2, 512, 16), "UNSUPPORTED", "512 values"), ((1, 4, 2, 128, 8), "INVALID", "pages of 8"),
    ((1, 4, 2, 128, 48), "INVALID", "pages of 48"), ((1, 4, 2, 128, 512), "INVALID", "pages of 512"), ((1, 0, 2, 128, 16), "INVALID", "0 pages"),
    ((1, -3, 2, 128, 16), "INVALID", "-3 pages"), ((1, 2**27, 2, 128, 16), "INVALID", "2^31 - 1 tokens"), ((1, 4, 0, 128, 16), "INVALID", "0 heads"),
    ((1, 4, -1, 128, 16), "INVALID", "-1 heads"), ((1, 4, 1025, 128, 16), "INVALID", "1025 heads")])
def test_cache_refusals(L, lib, ctx, memory, args, status, words):
    want = getattr(L, "JL_ERR_" + status)
    h = C.c_void_p(5)
    assert lib.jl_kv_cache_create(ctx, *args, C.byref(h)) == want and words in said(lib) and not h.value
    h = C.c_void_p(5)
    assert lib.jl_kv_cache_wrap(ctx, memory, *args, C.byref(h)) == want and words in said(lib) and not h.value
    assert lib.jl_kv_cache_bytes(*args) == 0


def test_cache_null_and_unaligned(L, lib, ctx, memory):
    h = C.c_void_p()
    assert lib.jl_kv_cache_wrap(ctx, memory + 8, 1, 4, 2, 128, 16, C.byref(h)) == L.JL_ERR_INVALID and "16-byte" in said(lib)
    assert lib.jl_kv_cache_wrap(ctx, None, 1, 4, 2, 128, 16, C.byref(h)) == L.JL_ERR_INVALID
    assert lib.jl_kv_cache_wrap(None, memory, 1, 4, 2, 128, 16, C.byref(h)) == L.JL_ERR_INVALID
    assert lib.jl_kv_cache_create(ctx, 1, 4, 2, 128, 16, None) == L.JL_ERR_INVALID
    assert lib.jl_kv_cache_free(None) == L.JL_OK and lib.jl_kv_cache_memory(None) is None


PLAN = dict(past=1, fresh=1, requests=4, pages=8, page_tokens=16, page_ring=1, free_in=1, free_out=1, block_table=1, table_stride=2, lengths=1,
            row_starts=1, slots=1, positions=1, row_requests=1, max_rows=4)


@pytest.mark.parametrize("change,words", [
    (dict(requests=-1), "-1 requests"), (dict(requests=8193), "8193 requests"), (dict(pages=0), "0 pages"), (dict(pages=2**27), "2^31 - 1"),
    (dict(page_tokens=0), "pages of 0"), (dict(page_tokens=24), "pages of 24"), (dict(max_rows=-1), "max_rows -1"),
    (dict(max_rows=2**17 + 1), "max_rows 131073"), (dict(table_stride=0), "4 x 0"), (dict(requests=8192, table_stride=2**18), "8192 x 262144")]
    + [({k: None}, "null") for k, v in PLAN.items() if v == 1])
def test_plan_refusals(L, lib, ctx, memory, change, words):
    args = [memory if v == 1 and k not in ("table_stride",) else v for k, v in {**PLAN, **change}.items()]
    assert lib.jl_kv_plan(ctx, *args) == L.JL_ERR_INVALID and words in said(lib), said(lib)


APPEND = dict(q="m", heads=4, ldq=1024, k="m", ldk=1024, v="m", ldv=1024, q_out="m", ldq_out=1024, positions="m", slots="m", rows=0, frequencies="m",
              rotated=128, rope_style=0, q_norm=None, k_norm=None, eps=1e-5)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), "-1 rows"), (dict(rotated=130), "130 values"), (dict(rotated=-16), "-16 values"), (dict(rotated=24), "24 values"),
    (dict(frequencies=None), "null frequencies"), (dict(rope_style=2), "style 2"), (dict(heads=0), "0 query heads"), (dict(heads=-1), "-1 query"),
    (dict(ldq=508), "closer together"), (dict(ldk=252), "closer together"), (dict(ldv=0), "closer together"), (dict(ldq_out=511), "closer together"),
    (dict(ldq=1026), "multiples of 4"), (dict(ldk=1025), "multiples of 4"), (dict(ldv=1027), "multiples of 4"), (dict(ldq_out=1001), "multiples of 4"),
    (dict(ldq_out=512), "in place"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(q_out=None), "null"), (dict(positions=None), "null"),
    (dict(slots=None), "null"), (dict(q="odd"), "aligned"), (dict(k="odd"), "aligned"), (dict(v="odd"), "aligned"), (dict(q_out="odd"), "aligned"),
    (dict(q_norm="odd"), "unaligned"), (dict(k_norm="odd"), "unaligned"), (dict(frequencies="word"), "unaligned")])
def test_append_refusals(L, lib, ctx, memory, cache, change, words):
    at = {"m": memory, "odd": memory + 8, "word": memory + 4}
    args = [at.get(v, v) if isinstance(v, str) else v for v in {**APPEND, **change}.values()]
    assert lib.jl_kv_append(ctx, cache, *args) == L.JL_ERR_INVALID and words in said(lib), said(lib)


def test_append_of_nothing(L, lib, ctx, memory, cache):
    args = [memory if v == "m" else v for v in APPEND.values()]
    assert lib.jl_kv_append(ctx, cache, *args) == L.JL_OK
    assert lib.jl_kv_append(None, cache, *args) == lib.jl_kv_append(ctx, None, *args) == L.JL_ERR_INVALID
    without_q = dict(APPEND, q=None, q_out=None, heads=0, ldq=0, ldq_out=0, rotated=0, frequencies=None)
    assert lib.jl_kv_append(ctx, cache, *[memory if v == "m" else v for v in without_q.values()]) == L.JL_OK


def test_read_refusals(L, lib, ctx, memory, cache):
    m = memory
    assert lib.jl_kv_read(ctx, cache, m, 0, m, m, 1) == L.JL_OK
    assert lib.jl_kv_read(ctx, cache, m, 5, None, None, 1) == L.JL_OK
    for args, words in (((None, cache, m, 1, m, m, 1), "null"), ((ctx, None, m, 1, m, m, 1), "null"), ((ctx, cache, None, 1, m, m, 1), "null"),
                        ((ctx, cache, m, -1, m, m, 1), "-1 rows"), ((ctx, cache, m, 1, m + 8, m, 1), "aligned"), ((ctx, cache, m, 1, m, m + 4, 0), "aligned")):
        assert lib.jl_kv_read(*args) == L.JL_ERR_INVALID and words in said(lib)


ATTEND = dict(q="m", heads=4, ldq=512, rows=0, positions="m", row_requests=None, block_table="m", requests=4, table_stride=2, scale=0.1, window=0, out="m",
              out_f16=0, ldo=512, workspace="m", workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,words", [
    (dict(heads=0), "0 query heads"), (dict(heads=5), "5 query heads"), (dict(rows=-1), "-1 rows"), (dict(rows=65536), "65536 rows"),
    (dict(rows=5), "5 rows of 4"), (dict(requests=-1), "requests"), (dict(table_stride=0), "0 entries"), (dict(scale=float("nan")), "scale nan"),
    (dict(scale=float("inf")), "scale inf"), (dict(window=-1), "window -1"), (dict(ldq=508), "closer together"), (dict(ldo=511), "closer together"),
    (dict(ldq=514), "multiple of 4"), (dict(ldo=514), "multiple of 4"), (dict(ldo=516, out_f16=1), "ldo of 8"), (dict(q=None), "null"),
    (dict(positions=None), "null"), (dict(block_table=None), "null"), (dict(out=None), "null"), (dict(workspace=None), "null"), (dict(q="odd"), "aligned"),
    (dict(out="odd"), "aligned"), (dict(workspace="odd"), "aligned")])
def test_attention_refusals(L, lib, ctx, memory, cache, change, words):
    at = {"m": memory, "odd": memory + 8}
    args = [at.get(v, v) if isinstance(v, str) else v for v in {**ATTEND, **change}.values()]
    assert lib.jl_kv_attention(ctx, cache, *args) == L.JL_ERR_INVALID and words in said(lib), said(lib)


def test_attention_workspace(L, lib, ctx, memory, cache):
    args = dict(ATTEND)
    need = lib.jl_kv_attention_workspace_bytes(4, 2, 128)
    assert 0 < need < 1 << 28
    for bad in ((4, 0, 128), (0, 2, 128), (5, 2, 128), (4, 2, 0), (-4, -2, 128)):
        assert lib.jl_kv_attention_workspace_bytes(*bad) == 0
    args["workspace_bytes"] = need - 1
    assert lib.jl_kv_attention(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_ERR_WORKSPACE
    args["workspace_bytes"] = need
    assert lib.jl_kv_attention(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_OK   # no rows: nothing to do


def test_attention_workspace_init_refusals(L, lib, ctx, memory):
    assert lib.jl_kv_attention_workspace_init(None, memory, 1 << 20) == L.JL_ERR_INVALID
    assert lib.jl_kv_attention_workspace_init(ctx, None, 1 << 20) == L.JL_ERR_INVALID
    assert lib.jl_kv_attention_workspace_init(ctx, memory + 4, 1 << 20) == L.JL_ERR_INVALID and "aligned" in said(lib)
    assert lib.jl_kv_attention_workspace_init(ctx, memory, 16) == L.JL_ERR_WORKSPACE


def test_attention_of_more_work_than_a_call_lists(L, lib, ctx, memory, cache):
    args = dict(ATTEND, rows=65535, requests=65535, table_stride=2**27)
    assert lib.jl_kv_attention(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_ERR_INVALID and "in one call" in said(lib)


def test_calls_past_a_launch(L, lib, ctx, memory, cache):
    """More threads than a launch has along a side, an output over the queries, a scale that the powers of two lose."""
    args = dict(APPEND, rows=2**24)
    assert lib.jl_kv_append(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_ERR_INVALID and "2^24" in said(lib)
    assert lib.jl_kv_read(ctx, cache, memory, 2**27, memory, memory, 1) == L.JL_ERR_INVALID and "2^35" in said(lib)
    args = dict(ATTEND, rows=1)
    assert lib.jl_kv_attention(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_ERR_INVALID and "in place" in said(lib)
    args = dict(ATTEND, scale=3e38)
    assert lib.jl_kv_attention(ctx, cache, *[memory if v == "m" else v for v in args.values()]) == L.JL_ERR_INVALID and "scale" in said(lib)


def test_cache_of_another_device(L, lib, memory, cache):
    other = C.create_string_buffer(4096)
    other[0] = 1
    at = C.addressof(other)
    assert lib.jl_kv_append(at, cache, *[memory if v == "m" else v for v in APPEND.values()]) == L.JL_ERR_INVALID and "device 0" in said(lib)
    assert lib.jl_kv_attention(at, cache, *[memory if v == "m" else v for v in ATTEND.values()]) == L.JL_ERR_INVALID and "device 0" in said(lib)
    assert lib.jl_kv_read(at, cache, memory, 0, memory, memory, 1) == L.JL_ERR_INVALID and "device 0" in said(lib)


def test_binding_checks_what_the_library_cannot():
    """Rows that leave their array, arrays too short for the rows, norms of another length."""
    from jitllm_amd.attention import BlockTables, Rows, _place

    class Array:
        def __init__(self, size, itemsize=4):
            self.size, self.nbytes, self.ptr = size, size * itemsize, C.c_void_p(4096)

    assert _place("x", Rows(Array(100), 10, 4), 10, 6) == (4096 + 16, 10)
    assert _place("x", Rows(Array(100, 2), 10, 4), 10, 6) == (4096 + 8, 10)
    assert _place("x", Array(60), 10, 6) == (4096, 6) and _place("x", Rows(Array(0), 6), 0, 6) == (4096, 6)
    for rows, width, stride, offset in ((11, 6, 10, 4), (10, 7, 10, 4), (1, 11, 10, 0), (1, 4, 10, -1)):
        with pytest.raises(ValueError):
            _place("x", Rows(Array(100), stride, offset), rows, width)
    with pytest.raises(ValueError, match="no such arrays"):
        class Ctx:
            _lib = None
        sizes = dict(table=8, lengths=4, rowStarts=5, slots=3, positions=3, rowRequests=3, pageRing=6, freePages=2)
        BlockTables(Ctx(), 4, 2, 6, 16, 3, arrays={**{k: Array(n) for k, n in sizes.items()}, "tabel": Array(8)})
    with pytest.raises(ValueError, match="slots"):
        BlockTables(Ctx(), 4, 2, 6, 16, 3, arrays={**{k: Array(n) for k, n in sizes.items()}, "slots": Array(2)})


def test_binding_checks_of_elements_and_tables():
    """binary16 where fp32 is taken, norms of it, a table whose rows' length the number of requests does not say."""
    from jitllm_amd.attention import PagedAttention, PagedKvCache, Rows, _place

    class Array:
        def __init__(self, size, itemsize=4):
            self.size, self.nbytes, self.ptr = size, size * itemsize, C.c_void_p(4096)

    calls = []

    class Lib:
        def jl_kv_attention(self, *args):
            calls.append(args)
            return 0

    class Ctx:
        handle, _lib = None, Lib()

    with pytest.raises(ValueError, match="q: .* 2048 bytes"):
        _place("q", Rows(Array(1024, 2), 128), 8, 128, 4)
    assert _place("out", Rows(Array(1024, 2), 128, 64), 7, 128, 2) == (4096 + 128, 128)
    cache, attention = object.__new__(PagedKvCache), object.__new__(PagedAttention)
    cache.ctx, cache._lib, cache.kvHeads, cache.headDim, cache.handle = Ctx(), Lib(), 2, 64, None
    with pytest.raises(ValueError, match="kNorm"):
        cache.append(Array(128), Array(128), Array(1), Array(1), 1, kNorm=Array(64, 2))
    attention.ctx, attention._lib, attention.kvHeads, attention.headDim, attention.heads = Ctx(), Lib(), 2, 64, 4
    attention.width, attention.scale, attention.workspace = 256, 0.125, Array(10)
    for more, stride in ((dict(requests=8), 16), (dict(requests=3, blocksPerRequest=16), 16), (dict(requests=0), 1)):
        attention.attend(cache, Array(512), 2, Array(2), Array(128), Array(512), **more)
        assert calls[-1][9:11] == (more["requests"], stride)
    for more in (dict(requests=3), dict(requests=9, blocksPerRequest=16)):
        with pytest.raises(ValueError, match="block table"):
            attention.attend(cache, Array(512), 2, Array(2), Array(128), Array(512), **more)


def test_models_agree_with_each_other():
    """The oracle's own pieces: blocks decode to what they were made from, the rotation keeps lengths and composes."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 96))
    kept, d, _ = M.encode_blocks(x)
    assert np.abs(kept * np.repeat(d, 32, -1) - x).max() <= np.abs(d).max() / 2 * 1.001
    f = 1e4 ** (-np.arange(0, 32, 2) / 32)
    y = rng.standard_normal((7, 2, 64))
    for halves in (False, True):
        a = M.rotate(M.rotate(y, np.arange(7), f, halves), np.full(7, 11), f, halves)
        assert np.allclose(a, M.rotate(y, np.arange(7) + 11, f, halves))
        assert np.allclose((a * a).sum(-1), (y * y).sum(-1)) and np.array_equal(a[..., 32:], y[..., 32:])
    pool = rng.standard_normal((2, 3, 1, 16, 64))
    out, weight, _ = M.attend(pool, np.zeros((1, 2, 64)), [19], None, np.array([[2, 0]]), 1.0)
    assert np.allclose(out[0, 1], np.concatenate([pool[1, 2, 0], pool[1, 0, 0, :4]]).mean(0)) and (weight >= np.abs(out) - 1e-12).all()


def test_limits_that_the_header_states(L, lib, ctx, memory, cache):
    """One past each: heads of q, and the list of tiles, which goes by the table's room (2 heads of k and v, pages of 16)."""
    at = lambda form, **change: [memory if v == "m" else v for v in dict(form, **change).values()]                # noqa: E731
    wide = dict(heads=65538, ldq=65538 * 128)
    assert lib.jl_kv_attention(ctx, cache, *at(ATTEND, **wide, ldo=65538 * 128)) == L.JL_ERR_INVALID and "65538 query heads" in said(lib)
    assert lib.jl_kv_append(ctx, cache, *at(APPEND, **wide, ldq_out=65538 * 128)) == L.JL_ERR_INVALID and "65538 query heads" in said(lib)
    rows = 65535
    most = ((2 ** 32 - 1025) // (2 * rows) - 6) * 32 + 31       # tokens that are still listed
    args = dict(rows=rows, requests=rows, table_stride=most // 16 + 1)
    assert lib.jl_kv_attention(ctx, cache, *at(ATTEND, **args)) == L.JL_ERR_INVALID and "in one call" in said(lib)
    # ... a list that fits comes to the next check
    args["table_stride"] -= 1
    assert lib.jl_kv_attention(ctx, cache, *at(ATTEND, **args, window=-1)) == L.JL_ERR_INVALID and "window" in said(lib)

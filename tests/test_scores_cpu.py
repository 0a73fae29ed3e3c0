"""The 4-bit cache, attention with shaped scores and log probabilities without a GPU: what the calls refuse, and what the
binding checks.  Every check of an argument comes before the first call of the HIP runtime."""
import ctypes as C

import numpy as np
import pytest

import score_models as S
from test_kv_cpu import L, ctx, lib, memory, said  # noqa: F401


@pytest.fixture(scope="module")
def cache(L, lib, ctx, memory):  # noqa: F811
    h = C.c_void_p()
    assert lib.jl_kv_cache_wrap(ctx, memory, L.JL_KV_Q4_0, 4, 2, 128, 16, C.byref(h)) == L.JL_OK
    yield h
    assert lib.jl_kv_cache_free(h) == L.JL_OK


@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_cache_bytes_of_fours(L, lib, dim, page):  # noqa: F811
    assert lib.jl_kv_cache_bytes(L.JL_KV_Q4_0, 7, 3, dim, page) == 2 * 7 * 3 * S.part_bytes("q4", dim, page)
    assert S.part_bytes("q4", dim, page) % 16 == 0
    for which in (0, 1):                                       # the layout's places: each once, none left
        at, shift = S.fours_at(which, dim, page)
        assert sorted((2 * at + shift // 4).reshape(-1)) == list(range(page * dim))


def test_cache_of_fours_refusals(L, lib, ctx, memory):  # noqa: F811
    for args, words in (((L.JL_KV_Q4_0, 4, 2, 80, 16), "80 values"), ((L.JL_KV_Q4_0, 4, 2, 128, 8), "pages of 8"), ((3, 4, 2, 128, 16), "type 3"),
                        ((5, 4, 2, 128, 16), "type 5")):
        h = C.c_void_p(5)
        assert lib.jl_kv_cache_wrap(ctx, memory, *args, C.byref(h)) != L.JL_OK and words in said(lib) and not h.value


SCORED = dict(q="m", heads=4, ldq=512, rows=0, positions="m", row_requests=None, block_table="m", requests=4, table_stride=2, scale=0.1, window=0, cap=30.0,
              slopes="m", first_tokens="m", end_tokens="m", out="m", out_f16=0, ldo=512, workspace="m", workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,words", [
    (dict(cap=-1.0), "cap -1"), (dict(cap=float("nan")), "cap nan"), (dict(cap=float("inf")), "cap inf"), (dict(cap=1e-31), "cap 1e-31"), (dict(cap=2e30), "cap 2e+30"),
    (dict(slopes="odd"), "aligned"), (dict(first_tokens="odd"), "aligned"), (dict(end_tokens="odd"), "aligned"),
    (dict(heads=5), "5 query heads"), (dict(rows=-1), "-1 rows"), (dict(rows=65536), "65536 rows"), (dict(rows=5), "5 rows of 4"), (dict(requests=-1), "requests"),
    (dict(table_stride=0), "0 entries"), (dict(scale=float("nan")), "scale nan"), (dict(window=-1), "window -1"), (dict(ldq=508), "closer together"),
    (dict(ldo=514), "multiple of 4"), (dict(q=None), "null"), (dict(positions=None), "null"), (dict(block_table=None), "null"), (dict(out=None), "null"),
    (dict(workspace=None), "null"), (dict(rows=1), "in place"), (dict(rows=65535, requests=65535, table_stride=2**27), "in one call")])
def test_scored_refusals(L, lib, ctx, memory, cache, change, words):  # noqa: F811
    at = {"m": memory, "odd": memory + 2}
    args = [at.get(v, v) if isinstance(v, str) else v for v in {**SCORED, **change}.values()]
    assert lib.jl_kv_attention_scored(ctx, cache, *args) == L.JL_ERR_INVALID and words in said(lib) and "scored" in said(lib), said(lib)


def test_scored_of_nothing(L, lib, ctx, memory, cache):  # noqa: F811
    for change in ({}, dict(cap=0.0), dict(cap=1e-30), dict(cap=1e30), dict(slopes=None, first_tokens=None, end_tokens=None, cap=0.0)):
        args = [memory if v == "m" else v for v in {**SCORED, **change}.values()]
        assert lib.jl_kv_attention_scored(ctx, cache, *args) == L.JL_OK
    args = [memory if v == "m" else v for v in {**SCORED, "workspace_bytes": 100}.values()]
    assert lib.jl_kv_attention_scored(ctx, cache, *args) == L.JL_ERR_WORKSPACE
    assert lib.jl_kv_attention_scored(None, cache, *args) == lib.jl_kv_attention_scored(ctx, None, *args) == L.JL_ERR_INVALID


LOGPROBS = dict(logits="m", rows=0, n=100, row_stride=100, scale=1.0, cap=0.0, tokens="m", tokens_per_row=1, logprobs="m", entropy="m", top=5, top_tokens="m",
                top_logprobs="m", workspace="m", workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,words", [
    (dict(logits=None), "null"), (dict(workspace=None), "null"), (dict(rows=-1), "-1 rows"), (dict(rows=2**31), "rows"), (dict(n=0), "0 logits"),
    (dict(n=2**31, row_stride=2**31), "2147483648 logits"), (dict(row_stride=99), "closer together"), (dict(scale=0.0), "scale 0"), (dict(scale=-1.0), "scale -1"),
    (dict(scale=float("nan")), "scale nan"), (dict(scale=float("inf")), "scale inf"), (dict(scale=3e38), "scale"), (dict(scale=1e-40), "scale"),
    (dict(cap=-2.0), "cap -2"), (dict(cap=float("nan")), "cap nan"), (dict(cap=1e31), "cap 1e+31"), (dict(tokens_per_row=-1), "-1 tokens"),
    (dict(tokens_per_row=65537), "65537 tokens"), (dict(tokens=None), "null tokens"), (dict(logprobs=None), "null tokens"), (dict(top=-1), "-1 most"),
    (dict(top=65), "65 most"), (dict(n=4, top=5), "5 most probable of 4"), (dict(top_tokens=None), "null top"), (dict(top_logprobs=None), "null top"),
    (dict(logits="odd"), "aligned"), (dict(workspace="odd"), "aligned"), (dict(tokens="odd"), "aligned"), (dict(top_logprobs="odd"), "aligned")])
def test_logprobs_refusals(L, lib, ctx, memory, change, words):  # noqa: F811
    at = {"m": memory, "odd": memory + 2}
    args = [at.get(v, v) if isinstance(v, str) else v for v in {**LOGPROBS, **change}.values()]
    assert lib.jl_logprobs(ctx, *args) == L.JL_ERR_INVALID and words in said(lib), said(lib)


def test_logprobs_workspace(L, lib, ctx, memory):  # noqa: F811
    need = lib.jl_logprobs_workspace_bytes(100, 5)
    assert 0 < need < 1 << 26
    assert lib.jl_logprobs_workspace_bytes(0, 0) == lib.jl_logprobs_workspace_bytes(2**31, 0) == lib.jl_logprobs_workspace_bytes(9, -1) == 0
    assert lib.jl_logprobs_workspace_bytes(100, 65) == 0
    args = lambda **more: [memory if v == "m" else v for v in {**LOGPROBS, **more}.values()]      # noqa: E731
    assert lib.jl_logprobs(ctx, *args(workspace_bytes=need - 1)) == L.JL_ERR_WORKSPACE
    assert lib.jl_logprobs(ctx, *args(workspace_bytes=need)) == L.JL_OK                           # no rows: nothing to do
    assert lib.jl_logprobs(ctx, *args(tokens_per_row=0, tokens=None, logprobs=None, entropy=None, top=0, top_tokens=None, top_logprobs=None)) == L.JL_OK
    assert lib.jl_logprobs(None, *args()) == L.JL_ERR_INVALID
    assert lib.jl_logprobs_workspace_init(None, memory, 1 << 20) == lib.jl_logprobs_workspace_init(ctx, None, 1 << 20) == L.JL_ERR_INVALID
    assert lib.jl_logprobs_workspace_init(ctx, memory + 4, 1 << 20) == L.JL_ERR_INVALID
    assert lib.jl_logprobs_workspace_init(ctx, memory, 8) == L.JL_ERR_WORKSPACE


class Array:
    def __init__(self, size, itemsize=4):
        self.size, self.nbytes, self.ptr = size, size * itemsize, C.c_void_p(4096)


def test_binding_of_scored_attention(monkeypatch):
    """The plain call where nothing is asked for; arrays that are too short, slopes of another number."""
    from jitllm_amd.attention import PagedAttention, PagedKvCache
    calls = []

    class Lib:
        def jl_kv_attention(self, *args):
            calls.append(("plain",) + args)
            return 0

        def jl_kv_attention_scored(self, *args):
            calls.append(("scored",) + args)
            return 0

    class Ctx:
        handle, _lib = None, Lib()

    cache, attention = object.__new__(PagedKvCache), object.__new__(PagedAttention)
    cache.ctx, cache._lib, cache.kvHeads, cache.headDim, cache.handle = Ctx(), Lib(), 2, 64, None
    attention.ctx, attention._lib, attention.kvHeads, attention.headDim, attention.heads = Ctx(), Lib(), 2, 64, 4
    attention.width, attention.scale, attention.workspace = 256, 0.125, Array(10)
    attend = lambda **more: attention.attend(cache, Array(512), 2, Array(2), Array(128), Array(512), requests=8, **more)      # noqa: E731
    attend()
    assert calls[-1][0] == "plain"
    for more in (dict(cap=3.0), dict(slopes=Array(4)), dict(firstTokens=Array(2)), dict(endTokens=Array(3))):
        attend(**more)
        assert calls[-1][0] == "scored" and len(calls[-1]) == 23
    for more in (dict(slopes=Array(5)), dict(slopes=Array(4, 2)), dict(firstTokens=Array(1)), dict(endTokens=Array(1))):
        with pytest.raises(ValueError):
            attend(**more)


def test_binding_of_logprobs():
    from jitllm_amd.logits import LogProbabilities
    calls = []

    class Lib:
        def jl_logprobs(self, *args):
            calls.append(args)
            return 0

    class Ctx:
        handle, _lib = None, Lib()

    p = object.__new__(LogProbabilities)
    p.ctx, p._lib, p.vocab, p.top, p.workspace = Ctx(), Lib(), 100, 3, Array(10)
    p.compute(Array(400), 4, tokens=Array(4), logprobs=Array(4), entropy=Array(4), topTokens=Array(12), topLogprobs=Array(12))
    assert calls[-1][8] == 1 and calls[-1][11] == 3
    p.compute(Array(400), 4)
    assert calls[-1][8] == 0 and calls[-1][11] == 0
    p.compute(Array(1), 0)
    for more in (dict(tokens=Array(4)), dict(logprobs=Array(4)), dict(topTokens=Array(12)), dict(tokens=Array(3), logprobs=Array(4)), dict(entropy=Array(3)),
                 dict(tokens=Array(4), logprobs=Array(4), tokensPerRow=2), dict(topTokens=Array(12), topLogprobs=Array(11)), dict(rowStride=99), dict(rowStride=101)):
        with pytest.raises(ValueError):
            p.compute(Array(400), 4, **more)


def test_models_of_scores_agree_with_each_other():
    """The oracle's own pieces: fours decode to what they were made from; a probability is one that adds up; a cap that is far
    away and slopes of zero change nothing; ranges and windows that say the same are the same."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 96))
    n, d, _ = S.encode_fours(x)
    assert np.abs((n - 8) * np.repeat(d, 32, -1) - x).max() <= np.abs(d).max() * 1.001
    raw = S.random_pool(rng, "q4", 3, 2, 64, 16)
    pool = S.decode_pool(raw, "q4", 3, 2, 64, 16)
    part = raw.reshape(2, 3, 2, -1)[1, 2, 1]
    assert pool[1, 2, 1, 7, 9] == np.float16(((part[(1 * 16 + 2) * 8 + 3 * 2] >> 4) - 8.0) * float(part[512:].view(np.float16).reshape(2, 16)[0, 7]))
    logits = rng.standard_normal((3, 50)).astype(np.float32)
    logp, entropy = S.logprobs(logits, 1.3, 4.0)
    assert np.allclose(np.exp(logp).sum(-1), 1) and np.allclose(entropy, -(np.exp(logp) * logp).sum(-1))
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    table, positions = np.array([[0, 1, 2]]), np.array([3, 20, 40, 47])
    args = (pool, q, positions, np.zeros(4, int), table, 0.125)
    plain = S.attend(*args)[0]
    assert np.allclose(S.attend(*args, cap=1e6, slopes=np.zeros(4))[0], plain, atol=1e-9)
    assert np.allclose(S.attend(*args, first=np.maximum(positions - 9, 0))[0], S.attend(*args, window=10)[0])
    assert np.allclose(S.attend(*args, end=positions + 1)[0], plain)

"""Steps of a 4-bit cache, scored attention and log probabilities together: through a layer to the answer, in graphs, on two
streams, through shared workspaces."""
import numpy as np
import pytest

import kv_models as M
import score_models as S
import test_gpu_kv as K
import test_gpu_logprobs as P
import test_gpu_scores as T
from gpu_util import say

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -11


@pytest.fixture(scope="module")
def ctx():
    from jitllm_amd.runtime import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", S.KINDS)
def test_steps_through_a_layer_to_the_answer(ctx, kind):
    """plan -> q|k|v -> append -> scored attention -> output projection -> vocabulary -> token, its probability, the others:
    each held to 64 bits over what the call before it left, prompts and decoding, one request that ends."""
    from jitllm_amd import synthetic
    from jitllm_amd.attention import BlockTables, PagedAttention, PagedKvCache, Rope, RopeStyle, Rows
    from jitllm_amd.ggml import GGMLType
    from jitllm_amd.logits import LogProbabilities
    from jitllm_amd.projections import QuantizedBatchProjections
    rng = np.random.default_rng(71)
    y = K.Layer(ctx, rng, False, True)
    vocab, top, cap, final_cap, window = 1056, 6, 20.0, 15.0, 24
    wcls = ctx.load_weight(GGMLType.Q8_0, synthetic.weight(GGMLType.Q8_0, vocab, y.dim, seed=7), vocab, y.dim)
    requests, stride, page, pages, max_rows = 4, 6, 16, 14, 64
    w, hd = (y.heads + 2 * y.kv) * y.head_dim, y.heads * y.head_dim
    freq = 1e4 ** (-np.arange(0, y.head_dim, 2) / y.head_dim)
    rope = Rope.of_base(ctx, y.head_dim, 1e4, RopeStyle.HALVES)
    tables = BlockTables(ctx, requests, stride, pages, page, max_rows)
    cache = PagedKvCache(ctx, T.kv_type(kind), pages, y.kv, y.head_dim, page, memory=ctx.raw_buffer(
        PagedKvCache.bytes_for(T.kv_type(kind), pages, y.kv, y.head_dim, page)))
    cache.memory.upload(np.zeros(cache.nbytes, np.uint8))
    attention = PagedAttention(ctx, max_rows, y.heads, y.kv, y.head_dim)
    proj = QuantizedBatchProjections(ctx, max_rows, max(y.dim, hd, vocab), max(w, vocab))
    answers = LogProbabilities(ctx, max_rows, vocab, top)
    slopes = (2.0 ** (-2.0 * np.arange(1, y.heads + 1))).astype(np.float32)
    on_device = ctx.from_numpy(slopes)
    qkv, att, x_out = (ctx.float_array(max_rows * n, fill=0.0) for n in (w, hd, y.dim))
    logits = ctx.float_array(max_rows * vocab, fill=0.0)
    tokens, listed = K.ints(ctx, np.full(max_rows, -5)), K.ints(ctx, np.full(max_rows * top, -5))
    lp, entropy, lp_top = (ctx.float_array(max_rows * n, fill=9.0) for n in (1, 1, top))
    lengths = np.zeros(requests, int)
    for step, fresh in enumerate([[20, 7, 33, 0], [1, 1, 1, 0], [1, -1, 1, 0], [1, 0, 1, 29], [1, 0, 0, 1], [1, 16, 1, 1]]):
        rows = sum(max(f, 0) for f in fresh)
        X = ctx.from_numpy(2 * rng.standard_normal((max_rows, y.dim)).astype(np.float32))
        say("answer step", kind, step, fresh)
        tables.plan(K.ints(ctx, fresh))
        proj.fusedQKV(X, qkv, y.w[0], y.w[1], y.w[2], rows)
        ctx.sync()
        plain = qkv.get().reshape(max_rows, y.heads + 2 * y.kv, y.head_dim).astype(np.float64)
        cache.append(Rows(qkv, w, hd), Rows(qkv, w, hd + y.kv * y.head_dim), tables.positions, tables.slots, rows, rope=rope,
                     q=Rows(qkv, w), heads=y.heads)
        attention.attend(cache, Rows(qkv, w), rows, tables.positions, tables.table, att, requests=requests, rowRequests=tables.rowRequests,
                         window=window, cap=cap, slopes=on_device)
        proj.projection(att, x_out, y.w[3], hd, y.dim, False, rows)
        proj.projection(x_out, logits, wcls, y.dim, vocab, False, rows)
        proj.argmaxLogits(logits, vocab, tokens, rows)
        answers.compute(logits, rows, tokens=tokens, logprobs=lp, entropy=entropy, topTokens=listed, topLogprobs=lp_top, cap=final_cap)
        ctx.sync()
        for r, f in enumerate(fresh):
            lengths[r] = 0 if f < 0 else lengths[r] + f
        assert tables.lengths.get().tolist() == lengths.tolist()
        positions, of, table = tables.positions.get()[:rows], tables.rowRequests.get()[:rows], tables.table.get().reshape(requests, stride)
        turned = qkv.get().reshape(max_rows, -1, y.head_dim)[:rows]
        pool = T.pool_of(cache, kind)
        at = table[of, positions // page]
        k = M.rotate(plain[:rows, y.heads:y.heads + y.kv], positions, freq, True)
        share = {"f16": HALF, "q8": 1 / 127 / 2 + 2 * HALF, "q4": 1 / 8 + 2 * HALF}[kind]   # of the block's largest: half a step; one at the end of four bits
        for which, want in enumerate((k, plain[:rows, y.heads + y.kv:])):
            largest = np.repeat(np.abs(want).reshape(rows, y.kv, -1, 32).max(-1), 32, -1)
            assert (np.abs(pool[which, at, :, positions % page] - want) <= 1.01 * share * largest + 2.0 ** -24).all()
        got = att.get().reshape(max_rows, y.heads, y.head_dim)[:rows].astype(np.float64)
        T.check(got, *S.attend(pool, turned[:, :y.heads], positions, of, table, y.head_dim ** -0.5, window, cap, slopes))
        z = logits.get().reshape(max_rows, vocab)[:rows]
        best = tokens.get()
        assert np.array_equal(best[:rows], z.argmax(-1)) and (step > 0 or (best[rows:] == -5).all())
        P.check(z, best[:rows, None], (lp.get()[:rows, None], entropy.get()[:rows], listed.get().reshape(max_rows, top)[:rows],
                                       lp_top.get().reshape(max_rows, top)[:rows]), top, 1.0, final_cap)
        assert np.array_equal(listed.get().reshape(max_rows, top)[:rows, 0], best[:rows])


# ---- graphs, streams, workspaces -----------------------------------------------------------------

class Step:
    """A step's plan, append, scored attention and log probabilities of its rows (a row's outputs are its logits)."""

    def __init__(self, ctx, kind, pages, max_rows, attention, answers, requests=5, stride=80, page=16, heads=32, kv=8, dim=64):
        from jitllm_amd.attention import BlockTables, PagedKvCache, Rope
        self.ctx, self.max_rows, self.heads, self.kv, self.dim, self.requests = ctx, max_rows, heads, kv, dim, requests
        self.attention, self.answers, self.rope = attention, answers, Rope.of_base(ctx, dim, 1e4)
        self.tables = BlockTables(ctx, requests, stride, pages, page, max_rows)
        memory = ctx.raw_buffer(PagedKvCache.bytes_for(T.kv_type(kind), pages, kv, dim, page))
        self.cache = PagedKvCache(ctx, T.kv_type(kind), pages, kv, dim, page, memory=memory)
        self.w = (heads + 2 * kv) * dim
        self.fresh, self.qkv = K.ints(ctx, np.zeros(requests)), ctx.float_array(max_rows * self.w, fill=0.0)
        self.first = K.ints(ctx, np.zeros(max_rows))
        self.tokens, self.listed = K.ints(ctx, np.arange(max_rows) % (heads * dim)), K.ints(ctx, np.full(max_rows * 5, -9))
        self.out, self.lp, self.entropy, self.lp_top = (ctx.float_array(max_rows * n, fill=7.0) for n in (heads * dim, 1, 1, 5))
        self.slopes = ctx.from_numpy((2.0 ** (-8 * np.arange(1, heads + 1) / heads)).astype(np.float32))

    def start(self, lengths, table, order, raw):
        self.tables.table.set(table), self.tables.lengths.set(lengths)
        used = int((table >= 0).sum())
        ring = np.full(len(order), -1)
        ring[:len(order) - used] = order[used:]
        self.tables.pageRing.set(ring), self.tables.freePages.set([0, len(order) - used])
        self.cache.memory.upload(raw)

    def feed(self, fresh, x):
        self.fresh.set(fresh), self.qkv.set(x), self.out.init(7.0)

    def step(self):
        from jitllm_amd.attention import Rows
        t, n = self.tables, self.heads * self.dim
        t.plan(self.fresh)
        self.cache.append(Rows(self.qkv, self.w, n), Rows(self.qkv, self.w, n + self.kv * self.dim), t.positions, t.slots, self.max_rows,
                          rope=self.rope, q=Rows(self.qkv, self.w), heads=self.heads)
        self.attention.attend(self.cache, Rows(self.qkv, self.w), self.max_rows, t.positions, t.table, self.out, requests=self.requests,
                              rowRequests=t.rowRequests, cap=30.0, slopes=self.slopes, firstTokens=self.first)
        self.answers.compute(self.out, self.max_rows, tokens=self.tokens, logprobs=self.lp, entropy=self.entropy, topTokens=self.listed,
                             topLogprobs=self.lp_top, cap=5.0)

    def left(self):
        arrays = [self.out, self.lp, self.entropy, self.listed, self.lp_top, self.tables.lengths, self.tables.table, self.tables.positions]
        return [a.get().view(np.uint32) for a in arrays]


def state(rng, kind, pages=380, stride=80, page=16, kv=8, dim=64):
    lengths = np.array([1100, 3, 0, 700, 16])
    order = rng.permutation(pages)
    need = -(-lengths // page)
    table = np.full((len(lengths), stride), -1)
    table[np.arange(stride) < need[:, None]] = order[:need.sum()]
    return lengths, table, order, S.random_pool(rng, kind, pages, kv, dim, page)


FRESH = {8: [[1, 1, 0, 1, 1], [1, 1, 2, 1, 1], [1, -1, 1, 1, 0], [1, 0, 1, 1, 5], [1, 3, 1, -1, 1], [1, 1, 1, 0, 1]],
         512: [[1, 150, 61, 1, 290], [130, 1, 1, 66, 1], [1, -1, 400, 1, 0], [0, 0, 0, 0, 0], [1, 1, 1, 1, 1], [30, 200, 1, -1, 64]]}


@pytest.mark.parametrize("max_rows", [8, 512])
@pytest.mark.parametrize("kind", S.KINDS)
def test_captured_steps_replayed_while_lengths_grow(ctx, kind, max_rows):
    """Two graphs over the same workspaces, in turn, each replay after the program's own eager work, held bit for bit to the
    same steps made eagerly over a copy of the state; rows that decode, and rows enough that prompts go in blocks."""
    import bench
    from jitllm_amd.attention import PagedAttention
    from jitllm_amd.logits import LogProbabilities
    hip = bench.Hip()
    rng = np.random.default_rng(31)
    attention, answers = PagedAttention(ctx, max_rows, 32, 8, 64), LogProbabilities(ctx, max_rows, 32 * 64, 5)
    begin = state(rng, kind)
    sides = [Step(ctx, kind, 380, max_rows, attention, answers) for _ in range(3)]
    for side in sides:
        side.start(*begin)
    a, again, b = sides
    say("captured answers", kind, max_rows)
    for side in (a, again):
        side.fresh.set([0] * 5)
        side.step()                                            # warmed up: nothing new
    ctx.sync()
    graphs = [hip.capture(ctx.stream, side.step) for side in (a, again)]
    try:
        for n, fresh in enumerate(FRESH[max_rows]):
            x = rng.standard_normal((max_rows, b.w)).astype(np.float32)
            for side in sides:
                side.feed(fresh, x)
            b.step()
            q = ctx.float_array(32 * 64, fill=0.5)
            attention.attend(b.cache, q, 1, K.ints(ctx, [600]), K.ints(ctx, np.arange(80)), ctx.float_array(32 * 64), requests=1, cap=3.0)
            ctx.sync()
            hip.launch(graphs[0], ctx.stream)
            hip.launch(graphs[1], ctx.stream)                  # behind the first, through the same workspaces
            ctx.sync()
            want = b.left()
            for side in (a, again):
                for i, (got, right) in enumerate(zip(side.left(), want)):
                    assert np.array_equal(got, right), (n, i)
            rows = sum(max(f, 0) for f in fresh)
            out = a.out.get().reshape(max_rows, -1)
            assert (out[rows:] == 0).all() and (rows == 0 or (out[:rows] != 0).any(-1).all())   # padding: nothing to read
    finally:
        for exe in graphs:
            hip.destroy_graph(exe)


@pytest.mark.parametrize("max_rows", [8, 512])
def test_two_contexts_at_once(ctx, max_rows):
    """Two streams, a workspace each, steps in flight side by side: each is what it is alone."""
    from jitllm_amd.attention import PagedAttention
    from jitllm_amd.logits import LogProbabilities
    from jitllm_amd.runtime import Context
    rng = np.random.default_rng(33)
    begin = state(rng, "q4")
    steps = FRESH[max_rows][:3]
    say("two contexts", max_rows)
    with Context(0) as second:
        inputs = [[rng.standard_normal((max_rows, (32 + 16) * 64)).astype(np.float32) for _ in steps] for _ in range(2)]

        def side_of(c):
            return Step(c, "q4", 380, max_rows, PagedAttention(c, max_rows, 32, 8, 64), LogProbabilities(c, max_rows, 32 * 64, 5))

        sides = [side_of(c) for c in (ctx, second)]
        alone = []
        for side, xs in zip(sides, inputs):
            side.start(*begin)
            alone.append([])
            for fresh, x in zip(steps, xs):
                side.feed(fresh, x)
                side.step()
                side.ctx.sync()
                alone[-1].append(side.left())
        for _ in range(4):
            for side in sides:
                side.start(*begin)
            for n, fresh in enumerate(steps):
                for side, xs in zip(sides, inputs):
                    side.feed(fresh, xs[n])
                for side in sides:
                    side.step()
                for side, want in zip(sides, alone):
                    side.ctx.sync()
                    for got, right in zip(side.left(), want[n]):
                        assert np.array_equal(got, right)
        for side in sides:
            side.cache.free()
        del sides, side, alone


def test_one_workspace_for_calls_of_several_shapes(ctx):
    """Layers of different heads, with scores of their own and without, prompts and rows that decode: one workspace."""
    from jitllm_amd.attention import PagedAttention
    rng = np.random.default_rng(43)
    wide = PagedAttention(ctx, 8, 64, 2, 256)
    calls = [([(0, 2999, 1), (1, 39, 1)], 64, 2, 256, "q4", 0.0), ([(0, 0, 600)], 16, 8, 64, "f16", 20.0), ([(0, 1999, 1)], 8, 1, 64, "f16", 5.0),
             ([(0, 100, 400)], 12, 4, 128, "q4", 0.0), ([(0, 3999, 1), (1, 0, 3)], 6, 6, 96, "q8", 10.0), ([(0, 0, 700)], 4, 4, 64, "q8", 8.0)]
    for runs, heads, kv, dim, kind, cap in calls * 2:
        of = np.concatenate([np.full(n, r) for r, _, n in runs])
        positions = np.concatenate([np.arange(first, first + n) for _, first, n in runs])
        most = [first + n for _, first, n in runs]
        table, pages = K.make_tables(rng, most, 32)
        raw = S.random_pool(rng, kind, pages, kv, dim, 32)
        cache = T.cache_of(ctx, kind, pages, kv, dim, 32, raw)
        attention = PagedAttention(ctx, 8, heads, kv, dim)
        assert attention.workspace.nbytes <= wide.workspace.nbytes
        attention.workspace = wide.workspace
        q = rng.standard_normal((len(of), heads, dim)).astype(np.float32)
        say("shared workspace", runs, heads, kv, dim, kind, cap)
        got = T.run(ctx, cache, q, positions, of, table, cap=cap, attention=attention)
        T.check(got, *S.attend(S.decode_pool(raw, kind, pages, kv, dim, 32), q, positions, of, table, dim ** -0.5, 0, cap))


def test_one_workspace_for_vocabularies_of_several_sizes(ctx):
    from jitllm_amd.logits import LogProbabilities
    rng = np.random.default_rng(44)
    wide = LogProbabilities(ctx, 100, 151936, 64)
    for rows, n, top in [(1, 151936, 64), (70, 1000, 5), (3, 50001, 20), (1, 64, 64), (300, 33, 1), (2, 128256, 0)] * 2:
        probabilities = LogProbabilities(ctx, rows, n, top)
        assert probabilities.workspace.nbytes <= wide.workspace.nbytes
        probabilities.workspace = wide.workspace
        logits = (4 * rng.standard_normal((rows, n))).astype(np.float32)
        tokens = rng.integers(0, n, (rows, 2))
        say("shared workspace", rows, n, top)
        P.check(logits, tokens, P.run(ctx, logits, tokens, top, probabilities=probabilities), top)

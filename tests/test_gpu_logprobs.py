"""Log probabilities, entropy and the most probable tokens on the GPU, against numpy in 64 bits."""
import numpy as np
import pytest

import score_models as S
from gpu_util import say

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24


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
    return a


def run(ctx, logits, tokens=None, top=0, scale=1.0, cap=0.0, pad=0, shift=0, entropy=True, probabilities=None):
    """(logprobs, entropy, top tokens, top logprobs) as the call leaves them; rows ``pad`` further apart than they are long,
    beginning ``shift`` floats off the allocation's boundary."""
    from jitllm_amd.logits import LogProbabilities
    rows, n = logits.shape
    flat = np.full(shift + rows * (n + pad), np.nan, np.float32)
    flat[shift:].reshape(rows, n + pad)[:, :n] = logits
    memory = ctx.from_numpy(flat)

    class Shifted:
        ptr, nbytes = type(memory.ptr)(memory.ptr.value + 4 * shift), memory.nbytes - 4 * shift

    per = 0 if tokens is None else tokens.shape[1]
    probabilities = probabilities or LogProbabilities(ctx, rows, n, top)
    out = [ctx.float_array(rows * max(k, 1) + 4, fill=-77.0) for k in (per, 1, top)]
    listed = ints(ctx, np.full(rows * max(top, 1) + 4, -77))
    probabilities.compute(Shifted, rows, tokens=ints(ctx, tokens) if per else None, logprobs=out[0] if per else None, entropy=out[1] if entropy else None,
                          topTokens=listed if top else None, topLogprobs=out[2] if top else None, tokensPerRow=per, scale=scale, cap=cap, rowStride=n + pad)
    ctx.sync()
    got = [a.get() for a in out] + [listed.get()]
    for a, k in zip(got, (per, int(entropy), top, top)):
        assert (a[rows * k:] == -77).all()                     # nothing behind what was asked for
    return got[0][:rows * per].reshape(rows, per), got[1][:rows], got[3][:rows * top].reshape(rows, top), got[2][:rows * top].reshape(rows, top)


def bounds(logits, logp, entropy, scale, cap):
    """How far fp32 arithmetic may be off a log p, and the entropy.  A value x below the largest by u: the cap's tanh and
    products are 2^-21 of it and 4 half steps, the difference, its scaling and the rounding of the power's argument 3 of u,
    so its weight is off by that and the power's own 2; the sum of n by its log2 n levels and what a thread adds one after
    the other, n / 64 at most; the logarithm by 2 of itself."""
    x = logits.astype(np.float64)
    n = x.shape[1]
    with np.errstate(invalid="ignore", over="ignore"):
        c = cap * np.tanh(x / cap) if cap else x
        c = np.where(np.isneginf(x), -np.inf, c)
        m = c.max(-1, keepdims=True)
        u = np.where(np.isfinite(c - m), scale * (m - c), 0)
        size = scale * (np.where(np.isfinite(c), np.abs(c), 0) + np.abs(np.where(np.isfinite(m), m, 0))) if cap else 0
        p = np.exp(np.where(np.isfinite(logp), logp, -np.inf))
        each = 3 * u + (12 * size if cap else 0)
        total = (p * (each + 2)).sum(-1, keepdims=True) + n / 64 + 20
        logs = 2 * np.abs(u + np.where(np.isfinite(logp), logp, 0)) + 2
        spread = (p * (each + 2) * (1 + u)).sum(-1) + (n / 64 + 20) * (1 + (p * u).sum(-1))
    return ULP * (each + total + logs + 2 * np.where(np.isfinite(logp), np.abs(logp), 0)), ULP * (spread + total[:, 0] + logs[:, 0] + 4 * np.abs(entropy))


def near_to(got, want, off):
    with np.errstate(invalid="ignore"):                        # (-inf, both)
        return ((got == want) | (np.abs(got - want) <= off)).all()


def check(logits, tokens, got, top, scale=1.0, cap=0.0):
    logprobs, entropy, listed, of_listed = got
    logp, want = S.logprobs(logits, scale, cap)
    near, near_entropy = bounds(logits, logp, want, scale, cap)
    assert (np.abs(entropy - want) <= near_entropy).all(), np.max(np.abs(entropy - want) / near_entropy)
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < logits.shape[1])
        at = np.where(inside, tokens, 0)
        right, off = (np.take_along_axis(a, at, 1) for a in (logp, near))
        right = np.where(inside, right, 0)
        assert near_to(logprobs, right, off)
    if top:
        order = S.ranked(logits, top)
        assert np.array_equal(listed, order)
        right, off = (np.take_along_axis(a, order, 1) for a in (logp, near))
        assert near_to(of_listed, right, off)


CASES = [
    # rows, n, tokens a row, top, scale, cap, pad, shift
    (1, 128256, 1, 5, 1.0, 0.0, 0, 0), (1, 151936, 0, 64, 1.0, 30.0, 0, 0), (3, 32000, 2, 20, 1.25, 0.0, 0, 0), (64, 5000, 1, 1, 0.5, 0.0, 24, 0),
    (1, 1, 1, 1, 1.0, 0.0, 0, 0), (2, 2, 3, 2, 1.0, 5.0, 0, 0), (5, 63, 1, 20, 1.0, 0.0, 0, 1), (7, 64, 1, 64, 2.0, 0.0, 1, 0), (9, 65, 1, 64, 1.0, 0.0, 0, 3),
    (300, 255, 1, 7, 1.0, 0.0, 0, 0), (513, 257, 1, 0, 1.0, 20.0, 2, 1), (2, 1023, 9, 33, 1.0, 0.0, 1, 2), (4, 1025, 1, 64, 0.1, 0.0, 0, 0), (1, 4095, 1, 10, 1.0, 0.0, 0, 1),
    (6, 4097, 1, 10, 1.0, 50.0, 3, 0), (33, 16384, 1, 3, 1.0, 0.0, 0, 0), (1100, 3001, 1, 4, 3.0, 0.0, 0, 0), (2, 300001, 1, 50, 1.0, 0.0, 0, 0), (17, 40000, 5, 64, 1.0, 0.0, 0, 0)]


@pytest.mark.parametrize("rows,n,per,top,scale,cap,pad,shift", CASES)
def test_logprobs(ctx, rows, n, per, top, scale, cap, pad, shift):
    say("logprobs", rows, n, per, top, scale, cap, pad, shift)
    rng = np.random.default_rng(rows + n)
    logits = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    logits[np.arange(rows), rng.integers(0, n, rows)] += 12
    tokens = rng.integers(0, n, (rows, per)) if per else None
    if per and rows > 2:
        tokens[1, 0], tokens[2, 0] = -1, n
    check(logits, tokens, run(ctx, logits, tokens, top, scale, cap, pad, shift), top, scale, cap)


ORDERS = {
    "ascending": lambda rng, n: np.sort(rng.standard_normal(n)),
    "descending": lambda rng, n: np.sort(rng.standard_normal(n))[::-1],
    "all equal": lambda rng, n: np.full(n, 1.5),
    "few values": lambda rng, n: rng.integers(0, 4, n),
    "signs of zero": lambda rng, n: np.where(rng.random(n) < 0.5, -0.0, 0.0),
    "all left out but some": lambda rng, n: np.where(rng.random(n) < 10 / n, rng.standard_normal(n), -np.inf),
    "all left out": lambda rng, n: np.full(n, -np.inf),
    "the lowest number in place of them": lambda rng, n: np.where(rng.random(n) < 10 / n, rng.standard_normal(n), np.finfo(np.float32).min),
    "nothing but the lowest number": lambda rng, n: np.full(n, np.finfo(np.float32).min),
    "one far above": lambda rng, n: np.where(np.arange(n) == n // 3, 1e4, rng.standard_normal(n)),
    "huge": lambda rng, n: 1e38 * rng.uniform(-1.5, 1.5, n),
    "tiny": lambda rng, n: 1e-42 * rng.integers(-3, 3, n),
    "far from zero": lambda rng, n: -3e4 + rng.standard_normal(n),
    "the largest all in one place": lambda rng, n: np.where(np.arange(n) // 97 == n // 194, 5, 0) + rng.random(n),
    "the largest a stride apart": lambda rng, n: np.where(np.arange(n) % 256 == 17, 5, 0) + rng.random(n),
}


@pytest.mark.parametrize("n", [70, 1000, 20000, 130000])
@pytest.mark.parametrize("name", ORDERS)
def test_logprobs_orders(ctx, name, n):
    """Values in orders and of sizes that a threshold, a list or a running maximum may stumble over."""
    say("logprobs order", name, n)
    rng = np.random.default_rng(n)
    with np.errstate(over="ignore"):
        logits = np.stack([ORDERS[name](rng, n) for _ in range(3)]).astype(np.float32)
    tokens = rng.integers(0, n, (3, 4))
    tokens[:, 0] = logits.argmax(-1)
    for top in (1, 20, 64):
        check(logits, tokens, run(ctx, logits, tokens, top), top)


@pytest.mark.parametrize("n", [64, 4000, 100000])
def test_logprobs_of_nan_and_infinity(ctx, n):
    """A row with NaN is NaN but for its list, which the others make; the rows beside it are not touched."""
    rng = np.random.default_rng(n)
    logits = rng.standard_normal((5, n)).astype(np.float32)
    logits[0, n // 2] = np.nan
    logits[1, :] = np.nan
    logits[2, 5] = np.inf
    logits[3, 10:] = np.nan
    tokens = np.array([[0, n // 2], [0, 1], [5, 6], [0, 11], [0, 1]])
    say("logprobs nan", n)
    logprobs, entropy, listed, of_listed = run(ctx, logits, tokens, 20)
    assert np.isnan(logprobs[:4]).all() and np.isnan(entropy[:4]).all()
    assert np.array_equal(listed, S.ranked(logits, 20))
    assert (listed[1] == -1).all() and (of_listed[1] == -np.inf).all() and (of_listed[3, 10:] == -np.inf).all()
    check(logits[4:], tokens[4:], tuple(a[4:] for a in (logprobs, entropy, listed, of_listed)), 20)
    # a cap makes an infinity a logit like others, and leaves out what is left out
    logits = rng.standard_normal((1, n)).astype(np.float32)
    logits[0, 3], logits[0, 4] = np.inf, -np.inf
    check(logits, np.array([[3, 4]]), run(ctx, logits, np.array([[3, 4]]), 20, cap=30.0), 20, cap=30.0)


def test_logprobs_parts_that_are_not_asked_for(ctx):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((9, 30000)).astype(np.float32)
    tokens = rng.integers(0, 30000, (9, 1))
    say("logprobs parts")
    whole = run(ctx, logits, tokens, 6)
    assert np.array_equal(run(ctx, logits, tokens)[0], whole[0]) and np.array_equal(run(ctx, logits)[1], whole[1])
    a = run(ctx, logits, None, 6, entropy=False)
    assert np.array_equal(a[2], whole[2]) and np.array_equal(a[3], whole[3])
    run(ctx, logits, entropy=False)


def test_logprobs_are_the_same_every_time(ctx):
    """With the same object, another one, and rows of other batches between."""
    from jitllm_amd.logits import LogProbabilities
    rng = np.random.default_rng(6)
    one = LogProbabilities(ctx, 64, 128256, 20)
    logits, more = rng.standard_normal((2, 128256)).astype(np.float32), rng.standard_normal((40, 128256)).astype(np.float32)
    tokens = rng.integers(0, 128256, (2, 1))
    say("logprobs repeats")
    first = run(ctx, logits, tokens, 20, probabilities=one)
    for turn in range(3):
        run(ctx, more, None, 20, probabilities=one)
        for a, b in zip(first, run(ctx, logits, tokens, 20, probabilities=one if turn else None)):
            assert np.array_equal(a, b)


def test_logprobs_of_no_rows(ctx):
    from jitllm_amd.logits import LogProbabilities
    one = LogProbabilities(ctx, 4, 100, 3)
    one.compute(ctx.float_array(100), 0, topTokens=ints(ctx, []), topLogprobs=ctx.float_array(1))
    ctx.sync()


@pytest.mark.parametrize("rows", [3, 1030])
@pytest.mark.parametrize("cap", [1e-30, 1e-6, 1e-4, 0.7, 30.0, 5e4, 1e6, 1e30])
def test_logprobs_of_logits_around_a_cap(ctx, rows, cap):
    """Logits of rows that are cut and that are not, within the cap, a few times as large, beyond; caps whose powers are no numbers."""
    rng = np.random.default_rng(8)
    n = 6000
    reach = np.array([0.02, 0.99, 2.4, 7, 1000])[np.arange(rows) % 5, None]
    top = min(cap, 1e30)
    logits = (np.clip(rng.standard_normal((rows, n)) / 3, -1, 1) * reach * top).astype(np.float32)
    logits[1::5, 100] = np.float32(top)
    scale = float(np.float32(8 / cap)) if 1e-8 < cap < 1e8 else 1.0
    say("logprobs around a cap", rows, cap)
    tokens = rng.integers(0, n, (rows, 1))
    check(logits, tokens, run(ctx, logits, tokens, 5, scale, cap), 5, scale, cap)

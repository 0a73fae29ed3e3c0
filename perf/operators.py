"""The steps between a layer's q|k|v projection and its output projection, as cases that can be timed and compared.

Three operators, each through the Python binding (``jitllm_amd.attention``) on a torch stream:

``plan``     pages of a key-value cache given to the requests of a step: block tables, lengths, and for
             every new token its request, position and slot, from request lengths that lie on the GPU
``append``   the rotation of q and k (each normalised first where a model does that) and the write of k and v
             into the pages, as binary16 or as blocks of 32 signed bytes with a binary16 scale
``attend``   attention of one new token of each request over its pages

``own`` false: the same in elementary torch operations.  Sizes are those of the models that bench.py, the tests
and ``perf/cases.py`` name (64 or 128 values a head; 32/8, 28/4 and 32/32 heads), and generic ones.

A cache is ``[2][pages][heads of k and v][one head's part of a page]``: of binary16, ``page_tokens`` rows of
``head_dim`` values; of 8-bit blocks, the rows' signed bytes and behind them the scales, ``[head_dim / 32][page_tokens]``.
An element of a block stands for the binary16 nearest to scale * byte.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
BLOCK = 32


def _plan(name, requests, page, context, rows, scarce=False):
    return {"name": name, "op": "plan", "requests": requests, "page": page, "context": context, "rows": rows, "scarce": scarce}


def _append(name, rows, heads, kv, dim, page, cache, context, halves, norm, rotated=None):
    return {"name": name, "op": "append", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "page": page, "cache": cache,
            "context": context, "halves": halves, "norm": norm, "rotated": rotated or dim}


def _attend(name, rows, heads, kv, dim, page, cache, context, ragged=False, window=0, half=False, mapped=False):
    return {"name": name, "op": "attend", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "page": page, "cache": cache,
            "context": context, "ragged": ragged, "window": window, "half": half, "mapped": mapped}


def listed():
    return [
        # one step of a batch of 64 that decodes: nearly every request has one new token, a few begin or end
        _plan("plan_64", 64, 16, 4096, 512),
        # a step that takes prompts in beside what it decodes, with fewer free pages than are asked for
        _plan("plan_512_scarce", 512, 64, 8192, 8192, scarce=True),
        # as many requests as a large server has in flight
        _plan("plan_4096", 4096, 64, 8192, 65536),
        # one token of Llama-3.2-1B: the smallest call
        _append("append_1_1b", 1, 32, 8, 64, 16, "f16", 1000, False, False),
        # one token of each of 64 requests, heads normalised (Qwen3-8B-like), into 8-bit blocks
        _append("append_64_8b_q8", 64, 32, 8, 128, 32, "q8", 8192, True, True),
        # the chunk of a prompt
        _append("append_2048_8b", 2048, 32, 8, 128, 64, "f16", 131072, False, False),
        # a short conversation with Llama-3.2-1B: latency
        _attend("attend_1x201_1b", 1, 32, 8, 64, 16, "f16", 201),
        # one very long one with an 8B model: the cache's length is all there is to split
        _attend("attend_1x131072_8b", 1, 32, 8, 128, 64, "f16", 131072),
        # a few long ones of different lengths over an 8-bit cache
        _attend("attend_8x32768_8b_q8", 8, 32, 8, 128, 32, "q8", 32768, ragged=True, mapped=True),
        # a full batch of Qwen2.5-7B (seven heads share one of k and v), binary16 out
        _attend("attend_64x8192_7b", 64, 28, 4, 128, 16, "f16", 8192, ragged=True, half=True),
        # Llama-2-7B: every head has its own k and v
        _attend("attend_29x950_7b", 29, 32, 32, 128, 16, "f16", 950, ragged=True, half=True),
        # wide heads that look back over a window
        _attend("attend_16x4096_window", 16, 16, 4, 256, 16, "q8", 4096, window=1024),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    op = rng.choice(("plan", "append", "attend", "attend"))
    if op == "plan":
        requests = int(_log(rng, 1, 4097))
        page = rng.choice((16, 32, 64, 128))
        most = min(32768, (page << 19) // requests)             # tokens a request may have: no larger tables than the listed ones
        case = _plan("", requests, page, int(_log(rng, 64, most)), int(_log(rng, max(64, 2 * requests), 65537)), rng.random() < 0.3)
    else:
        kv = rng.choice((1, 2, 4, 8))
        group = rng.choice((1, 2, 3, 4, 6, 7, 8, 12, 16))
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        cache = rng.choice(("f16", "q8"))
        page = rng.choice((16, 32, 64, 128))
        if op == "append":
            case = _append("", int(_log(rng, 1, 2049)), kv * group, kv, dim, page, cache, int(_log(rng, 64, 131072)), rng.random() < 0.5,
                           rng.random() < 0.4, dim if rng.random() < 0.7 else dim // 2)
            while work(case)["bytes"] > work(listed()[5])["bytes"]:
                case["rows"] = case["rows"] * 3 // 4
        else:
            context = int(_log(rng, 1, 65537))
            window = int(_log(rng, 16, 4097)) if rng.random() < 0.25 else 0
            case = _attend("", int(_log(rng, 1, 129)), kv * group, kv, dim, page, cache, context, rng.random() < 0.6, window, rng.random() < 0.5,
                           rng.random() < 0.3)
            whole, most = dict(case, window=0), work(listed()[9])
            while whole["rows"] > 1 and (_cached(whole) > most["bytes"] or work(whole)["flops"] > most["flops"]):
                whole["rows"] = max(1, whole["rows"] * 3 // 4)
            while _cached(whole) > most["bytes"] or work(whole)["flops"] > most["flops"]:
                whole["context"] = whole["context"] * 3 // 4
            case = dict(whole, window=window)
    del case["name"]
    return case


# ---- what a program has in hand ------------------------------------------------------------------

class State:
    pass


_context = None


def context():
    """The program's one context, on a torch stream that is made the current one."""
    global _context
    if _context is None:
        from jitllm_amd.runtime import Context
        stream = torch.cuda.Stream()
        torch.cuda.set_stream(stream)
        _context = Context(torch.cuda.current_device(), stream=stream.cuda_stream)
        _context.torch_stream = stream
    return _context


def _head_page_bytes(case):
    values = case["page"] * case["dim"]
    return 2 * values if case["cache"] == "f16" else values + values // BLOCK * 2


def _lengths(case):
    """Tokens each row sees, its own included: all the context, or lengths spread evenly over it."""
    n = case["rows"]
    if not case["ragged"]:
        return [case["context"]] * n
    return [max(1, math.ceil(case["context"] * (i + 1) / n)) for i in range(n)]


def _random_pool(case, pages, gen):
    per = _head_page_bytes(case)
    if case["cache"] == "f16":
        return torch.randn(2 * pages * case["kv"] * per // 2, device="cuda", generator=gen, dtype=torch.float16).view(torch.uint8)
    values = case["page"] * case["dim"]
    pool = torch.randint(0, 255, (2 * pages * case["kv"], per), device="cuda", generator=gen, dtype=torch.uint8).sub_(127)
    d = torch.empty((2 * pages * case["kv"], values // BLOCK), device="cuda").uniform_(0.004, 0.03, generator=gen)
    pool[:, values:] = d.to(torch.float16).view(torch.uint8)
    return pool.view(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    s = State()
    s.case = case
    ctx = context() if own else None

    def ints(values):
        return torch.as_tensor(np.ascontiguousarray(values, dtype=np.int32)).cuda()

    if case["op"] == "plan":
        _prepare_plan(s, case, host, ints)
    elif case["op"] == "append":
        rows, heads, kv, dim, page = (case[k] for k in ("rows", "heads", "kv", "dim", "page"))
        pages = -(-rows // page) * 2 + 3
        s.pool = _random_pool(case, pages, gen)
        s.qkv = torch.randn((rows, (heads + 2 * kv) * dim), device="cuda", generator=gen)
        s.q_out = torch.zeros((rows, heads * dim), device="cuda")
        s.slots = ints(host.permutation(pages * page)[:rows] if rows < 128 else host.permutation(pages)[np.arange(rows) // page] * page + np.arange(rows) % page)
        s.positions = ints(host.integers(0, case["context"], rows) if rows < 128 else case["context"] - rows + np.arange(rows) if case["context"] >= rows else np.arange(rows))
        r = case["rotated"]
        s.frequencies = 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
        s.q_norm, s.k_norm = (1 + 0.1 * torch.randn(dim, device="cuda", generator=gen) if case["norm"] else None for _ in range(2))
        s.k_read, s.v_read = (torch.zeros((rows, kv, dim), device="cuda", dtype=torch.float16) for _ in range(2))
        s.pages = pages
    else:
        rows, heads, kv, dim, page = (case[k] for k in ("rows", "heads", "kv", "dim", "page"))
        lengths = host.permutation(np.array(_lengths(case)))
        requests = rows + (rows // 4 + 1 if case["mapped"] else 0)
        blocks = -(-case["context"] // page)
        first = np.maximum(0, lengths - case["window"]) // page if case["window"] else np.zeros(rows, np.int64)
        held = -(-lengths // page) - first                     # pages that left the window are no longer held
        pages = int(held.sum()) + 2
        order = host.permutation(pages)[:int(held.sum())]
        table = np.zeros((requests, blocks), np.int64)
        requests_of = host.permutation(requests)[:rows]
        ends = np.cumsum(held)
        for i in range(rows):
            table[requests_of[i], first[i]:first[i] + held[i]] = order[ends[i] - held[i]:ends[i]]
        if not case["mapped"]:
            table = table[requests_of]
        s.pool = _random_pool(case, pages, gen)
        s.table, s.positions = ints(table), ints(lengths - 1)
        s.requests_of = ints(requests_of) if case["mapped"] else None
        s.q = 1.5 * torch.randn((rows, heads * dim), device="cuda", generator=gen)
        s.out = torch.zeros((rows, heads * dim), device="cuda", dtype=torch.float16 if case["half"] else torch.float32)
        s.pages = pages
    if own:
        _bind(s, case, ctx)
    torch.cuda.synchronize()
    return s


def _prepare_plan(s, case, host, ints):
    n, page, blocks = case["requests"], case["page"], -(-case["context"] // case["page"])
    past = host.integers(1, case["context"], n)
    kind = host.random(n)
    fresh = np.where(kind < 0.86, 1, np.where(kind < 0.9, 0, np.where(kind < 0.94, -1, 2)))
    starting = np.flatnonzero(fresh == 2)
    past[starting] = 0
    room = max(1, (case["rows"] - n) // max(1, len(starting)))   # the step's prompts share what its rows leave
    fresh[starting] = np.minimum(host.integers(1, 2 * room + 1, len(starting)), case["context"])
    had = -(-past // page)
    need = np.maximum(0, -(-(past + np.maximum(fresh, 0)) // page) - had)
    pages = n * blocks + 8                                      # room for every request's whole context
    free = min(int(need.sum() * 0.6) if case["scarce"] else int(need.sum() * 1.5) + 8, pages - int(had.sum()))
    order = host.permutation(pages)
    table = np.full((n, blocks), -1, np.int64)
    table[np.arange(blocks) < had[:, None]] = order[:int(had.sum())]
    head = int(host.integers(0, pages))
    ring = np.full(pages, -1, np.int64)
    ring[(head + np.arange(free)) % pages] = order[int(had.sum()):int(had.sum()) + free]
    s.pages, s.blocks = pages, blocks
    s.past, s.fresh, s.table, s.ring = ints(past), ints(fresh), ints(table), ints(ring)
    s.free = ints([head, free])
    s.free_out, s.lengths, s.row_starts = ints([0, 0]), ints(np.zeros(n)), ints(np.zeros(n + 1))
    s.slots, s.positions, s.requests_of = (ints(np.zeros(case["rows"])) for _ in range(3))


def _bind(s, case, ctx):
    """The framework's objects over the tensors."""
    from jitllm_amd.attention import BlockTables, KvType, PagedAttention, PagedKvCache, Rope, RopeStyle

    def memory(t):
        return _Memory(ctx, t)

    if case["op"] == "plan":
        s.tables = BlockTables(ctx, case["requests"], s.blocks, s.pages, case["page"], case["rows"],
                               arrays={"table": memory(s.table), "pageRing": memory(s.ring), "freePages": memory(s.free_out),
                                       "lengths": memory(s.lengths), "rowStarts": memory(s.row_starts), "slots": memory(s.slots),
                                       "positions": memory(s.positions), "rowRequests": memory(s.requests_of)})
        s.m_past, s.m_fresh, s.m_free = memory(s.past), memory(s.fresh), memory(s.free)
        return
    kind = KvType.F16 if case["cache"] == "f16" else KvType.Q8_0
    s.cache = PagedKvCache(ctx, kind, s.pages, case["kv"], case["dim"], case["page"], memory=memory(s.pool))
    s.m_positions = memory(s.positions)
    if case["op"] == "append":
        s.m_qkv, s.m_q_out, s.m_slots = memory(s.qkv), memory(s.q_out), memory(s.slots)
        s.rope = Rope(ctx, memory(s.frequencies), case["rotated"], RopeStyle.HALVES if case["halves"] else RopeStyle.PAIRS)
        s.m_q_norm, s.m_k_norm = (memory(t) if t is not None else None for t in (s.q_norm, s.k_norm))
        s.m_k_read, s.m_v_read = memory(s.k_read), memory(s.v_read)
    else:
        s.m_q, s.m_out, s.m_table = memory(s.q), memory(s.out), memory(s.table)
        s.m_requests = memory(s.requests_of) if s.requests_of is not None else None
        s.attention = PagedAttention(ctx, case["rows"], case["heads"], case["kv"], case["dim"])


class _Memory:
    """A tensor's memory as the binding takes arrays: a pointer, a count of elements, and the bytes of one."""

    def __init__(self, ctx, tensor):
        import ctypes
        assert tensor.is_contiguous()
        self.ctx, self.tensor, self.ptr = ctx, tensor, ctypes.c_void_p(tensor.data_ptr())
        self.size, self.nbytes = tensor.numel(), tensor.numel() * tensor.element_size()
        self.itemsize = tensor.element_size()


# ---- a pass --------------------------------------------------------------------------------------

def run(s):
    return {"plan": _run_plan, "append": _run_append, "attend": _run_attend}[s.case["op"]](s)


def _run_plan(s):
    if not own:
        return _plain_plan(s)
    s.tables.plan(s.m_fresh, past=s.m_past, freeIn=s.m_free)
    return {"lengths": s.lengths, "row_starts": s.row_starts, "table": s.table, "ring": s.ring, "free": s.free_out, "slots": s.slots,
            "positions": s.positions, "requests": s.requests_of}


def _run_append(s):
    if not own:
        return _plain_append(s)
    from jitllm_amd.attention import Rows
    c = s.case
    q, k = c["heads"] * c["dim"], c["kv"] * c["dim"]
    stride = q + 2 * k
    s.cache.append(Rows(s.m_qkv, stride, q), Rows(s.m_qkv, stride, q + k), s.m_positions, s.m_slots, c["rows"], rope=s.rope,
                   q=Rows(s.m_qkv, stride), qOut=Rows(s.m_q_out, q), heads=c["heads"], qNorm=s.m_q_norm, kNorm=s.m_k_norm, eps=EPS)
    if c["cache"] == "f16":
        return {"q": s.q_out, "cache": s.pool.view(torch.float16)}
    s.cache.read(s.m_slots, c["rows"], s.m_k_read, s.m_v_read)
    return {"q": s.q_out, "k": s.k_read, "v": s.v_read}


def _run_attend(s):
    if not own:
        return _plain_attend(s)
    s.attention.attend(s.cache, s.m_q, s.case["rows"], s.m_positions, s.m_table, s.m_out, requests=s.table.shape[0], rowRequests=s.m_requests,
                       window=s.case["window"])
    return s.out


# ---- the plain forms -----------------------------------------------------------------------------

def _plain_plan(s):
    page, rows, pages, blocks = s.case["page"], s.case["rows"], s.pages, s.blocks
    past, fresh = s.past.long(), s.fresh.long()
    wanted = fresh.clamp(min=0)
    ends = wanted.cumsum(0)
    had = (past + page - 1) // page
    fits = (ends <= rows) & (past + wanted <= blocks * page)
    need = torch.where(fits, (past + wanted + page - 1) // page - had, 0)
    through = need.cumsum(0)
    head, count = s.free.long().unbind()
    granted = fits & (wanted > 0) & ((need == 0) | (through <= count))
    need = torch.where(granted, need, 0)
    ended = fresh < 0
    lengths = torch.where(ended, 0, torch.where(granted, past + wanted, past))
    b = torch.arange(blocks, device=past.device)
    new = (b >= had[:, None]) & (b < (had + need)[:, None])
    table = torch.where(new, s.ring.long()[(head + (through - need)[:, None] + b - had[:, None]) % pages], s.table.long())
    back = torch.where(ended, had, 0)
    back_at = back.cumsum(0) - back
    given_back = ended[:, None] & (b < had[:, None])
    place = torch.where(given_back, (head + count + back_at[:, None] + b) % pages, pages)
    ring = torch.cat([s.ring.long(), s.ring.new_zeros(1).long()])
    ring = ring.scatter(0, place.view(-1), table.view(-1))[:pages]
    taken, returned = need.sum(), back.sum()
    i = torch.arange(rows, device=past.device)
    request = torch.searchsorted(ends, i, right=True)
    used = request < len(past)
    at = request.clamp(max=len(past) - 1)
    live = used & granted[at]
    position = past[at] + i - (ends - wanted)[at]
    paged = table[at, (position // page).clamp(0, blocks - 1)] * page + position % page
    minus = torch.full_like(i, -1)
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=rows)
    out = {"lengths": lengths, "row_starts": starts, "table": table, "ring": ring, "free": torch.stack([(head + taken) % pages, count - taken + returned]),
           "slots": torch.where(live, paged, minus), "positions": torch.where(live, position, minus), "requests": torch.where(used, request, minus)}
    return {k: v.int() for k, v in out.items()}


def _plain_rotate(s, x, norm):
    c = s.case
    if norm is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * norm
    r = c["rotated"]
    angle = s.positions.double()[:, None] * s.frequencies                       # far positions need 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if c["halves"]:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_append(s):
    c = s.case
    rows, heads, kv, dim, page = (c[k] for k in ("rows", "heads", "kv", "dim", "page"))
    x = s.qkv.view(rows, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    q, k = _plain_rotate(s, q, s.q_norm), _plain_rotate(s, k, s.k_norm)
    q = q.reshape(rows, heads * dim)
    if c["cache"] == "f16":
        pool = s.pool.view(torch.float16).view(2, s.pages, kv, page, dim).clone()
        slots = s.slots.long()
        pool[0, slots // page, :, slots % page] = k.half()
        pool[1, slots // page, :, slots % page] = v.half()
        return {"q": q, "cache": pool.view(-1)}
    return {"q": q, "k": _plain_blocks(k), "v": _plain_blocks(v)}


def _plain_blocks(x):
    """What blocks of 32 signed bytes and a binary16 scale keep of x."""
    blocks = x.reshape(-1, BLOCK)
    d = (blocks.abs().amax(-1, keepdim=True) / 127).half().float()
    kept = torch.where(d > 0, (blocks / d).round().clamp(-127, 127), torch.zeros_like(blocks))
    return (kept * d).half().view(x.shape)


def _values(case, pool):
    """[..., page_tokens, head_dim] in 32 bits of heads' parts of pages, [..., bytes]."""
    page, dim = case["page"], case["dim"]
    if case["cache"] == "f16":
        return pool.view(torch.float16).view(*pool.shape[:-1], page, dim).float()
    quants = pool[..., :page * dim].view(torch.int8).view(*pool.shape[:-1], page, dim // BLOCK, BLOCK).float()
    d = pool[..., page * dim:].contiguous().view(torch.float16).view(*pool.shape[:-1], dim // BLOCK, page).transpose(-1, -2).float()
    return (quants * d[..., None]).half().float().view(*pool.shape[:-1], page, dim)


def _plain_attend(s):
    c = s.case
    rows, heads, kv, dim, page = (c[k] for k in ("rows", "heads", "kv", "dim", "page"))
    table = s.table.long() if s.requests_of is None else s.table.long()[s.requests_of.long()]
    blocks = table.shape[1]
    pool = s.pool.view(2, s.pages, kv, -1)
    k, v = (_values(c, pool[i][table]).transpose(1, 2).reshape(rows, kv, blocks * page, dim) for i in (0, 1))
    j = torch.arange(blocks * page, device=table.device)
    seen = j <= s.positions[:, None]
    if c["window"]:
        seen &= j > s.positions[:, None] - c["window"]
    seen = seen[:, None, None]
    scores = torch.matmul(s.q.view(rows, kv, heads // kv, dim) * dim ** -0.5, k.transpose(-1, -2))
    scores = torch.where(seen, scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top.isfinite(), top, 0))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total > 0, total, 1)
    return out.reshape(rows, heads * dim).to(s.out.dtype)


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None                                            # whole numbers
    s = prepare(case, seed)
    return (_exact_append if case["op"] == "append" else _exact_attend)(s, case)


def _exact_append(s, case):
    rows, heads, kv, dim, page, r = (case[k] for k in ("rows", "heads", "kv", "dim", "page", "rotated"))
    qkv = s.qkv.double().view(rows, heads + 2 * kv, dim)
    q, k, v = qkv.split([heads, kv, kv], 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s.positions.double(), s.frequencies))[:, None]

    def rotate(x, norm):
        if norm is not None:
            x = x * norm.double() * torch.rsqrt((x * x).sum(-1, keepdim=True) / dim + EPS)
        pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["halves"] else x[..., :r].unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2).flatten(-2) if case["halves"] else z.flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    q, k = rotate(q, s.q_norm).reshape(rows, heads * dim), rotate(k, s.k_norm)
    if case["cache"] == "f16":
        cache = s.pool.view(torch.float16).double().view(2, s.pages, kv, page, dim)
        at = s.slots.long()
        cache[0].index_put_((at // page, torch.arange(kv, device="cuda")[:, None], at % page), k.transpose(0, 1).half().double())
        cache[1].index_put_((at // page, torch.arange(kv, device="cuda")[:, None], at % page), v.transpose(0, 1).half().double())
        return {"q": q, "cache": cache.reshape(-1)}

    def kept(x):
        y = x.unflatten(-1, (dim // BLOCK, BLOCK))
        d = (torch.linalg.vector_norm(y, ord=float("inf"), dim=-1, keepdim=True) / 127).half().double()
        return (torch.round(y / d).clamp(-127, 127) * d).half().double().flatten(-2)

    return {"q": q, "k": kept(k), "v": kept(v)}


def _exact_attend(s, case):
    heads, kv, dim, page = (case[k] for k in ("heads", "kv", "dim", "page"))
    parts = s.pool.view(2, s.pages, kv, -1)
    out = torch.zeros((case["rows"], heads, dim), dtype=torch.float64, device="cuda")
    for row, last in enumerate(s.positions.tolist()):
        request = row if s.requests_of is None else int(s.requests_of[row])
        begin = max(0, last + 1 - case["window"]) if case["window"] else 0
        held = s.table[request, begin // page:last // page + 1].long()
        token = torch.arange(begin, last + 1, device="cuda") - begin // page * page
        for h in range(kv):
            keys, values = (_exact_values(parts[i, held, h], case)[token] for i in (0, 1))
            q = s.q[row].double().view(kv, heads // kv, dim)[h]
            out[row].view(kv, heads // kv, dim)[h] = torch.softmax(q @ keys.T / math.sqrt(dim), -1) @ values
    return out.view(case["rows"], heads * dim)


def _exact_values(raw, case):
    page, dim = case["page"], case["dim"]
    if case["cache"] == "f16":
        return raw.contiguous().view(torch.float16).double().view(-1, dim)
    d = raw[:, page * dim:].contiguous().view(torch.float16).double().view(-1, dim // BLOCK, page)
    quants = raw[:, :page * dim].contiguous().view(torch.int8).double().view(-1, page, dim // BLOCK, BLOCK)
    return (quants * d.transpose(1, 2).unsqueeze(-1)).half().double().reshape(-1, dim)


# ---- what a pass cannot do without ---------------------------------------------------------------

def _cached(case):
    """Bytes of the cache that an attention pass reads."""
    seen = sum(min(n, case["window"] or n) for n in _lengths(case))
    return 2 * case["kv"] * seen * _head_page_bytes(case) // case["page"]


def work(case):
    if case["op"] == "plan":
        n, rows = case["requests"], case["rows"]
        # past and fresh, lengths and row starts, three numbers a row; pages taken, once read and once written
        return {"bytes": 16 * n + 12 * rows + 8 * (rows // case["page"]), "flops": 4 * (n + rows)}
    heads, kv, dim, rows = (case[k] for k in ("heads", "kv", "dim", "rows"))
    if case["op"] == "append":
        written = 2 * kv * _head_page_bytes(case) // case["page"]
        back = 0 if case["cache"] == "f16" else written + 4 * kv * dim
        return {"bytes": rows * (4 * (heads + 2 * kv) * dim + 4 * heads * dim + written + back + 8),
                "flops": rows * (heads + kv) * (3 * case["rotated"] + (4 * dim if case["norm"] else 0))}
    seen = sum(min(n, case["window"] or n) for n in _lengths(case))
    return {"bytes": _cached(case) + rows * heads * dim * (4 + (2 if case["half"] else 4)) + 4 * (seen // case["page"] + rows),
            "flops": 4 * heads * dim * seen}

"""A step's attention over a cache of 4 bits, with scores that are capped, biased or masked, and its log probabilities,
as cases that can be timed and compared.

Three operators, each through the Python binding on a torch stream:

``append``    the rotation of q and k and the write of k and v into pages of 4-bit blocks (``jitllm_amd.attention``)
``attend``    attention of the rows of a step over their requests' pages: over 4-bit blocks; or with scores that are
              capped, lowered by the distance of the token, or kept to a document or opened to a prefix, over any cache
``logprobs``  log probabilities of given tokens, the entropy and the most probable tokens, from rows of logits
              (``jitllm_amd.logits``)

``own`` false: the same in elementary torch operations.  Sizes are those of the models that bench.py, the tests and
``perf/cases.py`` name (64 or 128 values a head; 32/8, 28/4 and 32/32 heads; vocabularies of 32000, 128256 and 151936),
and generic ones.

A 4-bit block is 32 values and a binary16 d: d = the value of largest magnitude / -8, each value the nearest whole
multiple of d from -8 to 7; an element stands for the binary16 nearest to d * multiple.  A cache is
``[2][pages][heads of k and v][one head's part of a page]``, a part ``page_tokens * head_dim / 2`` bytes of multiples (plus
8, four bits each) and behind them the scales, ``[head_dim / 32][page_tokens]``.  Of a token's keys, byte b has the
elements 2 b (low) and 2 b + 1.  Of values, tokens stand in fours: for each four tokens and four elements, two bytes of each
of the tokens.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 32


def _append(name, rows, heads, kv, dim, page, context, halves, rotated=None):
    return {"name": name, "op": "append", "rows": rows, "heads": heads, "kv": kv, "dim": dim, "page": page, "cache": "q4",
            "context": context, "halves": halves, "rotated": rotated or dim}


def _attend(name, requests, past, fresh, heads, kv, dim, page, cache, ragged=False, window=0, half=False, cap=0.0, slopes=False,
            documents=0, prefix=False):
    return {"name": name, "op": "attend", "requests": requests, "past": past, "fresh": fresh, "heads": heads, "kv": kv, "dim": dim,
            "page": page, "cache": cache, "ragged": ragged, "window": window, "half": half, "cap": cap, "slopes": slopes,
            "documents": documents, "prefix": prefix}


def _logprobs(name, rows, vocab, top, tokens=1, cap=0.0, scale=1.0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "tokens": tokens, "cap": cap, "scale": scale}


def listed():
    return [
        # one token of each of 64 requests of an 8B model
        _append("append_64_8b_q4", 64, 32, 8, 128, 32, 8192, True),
        # the chunk of a prompt of Llama-3.2-1B
        _append("append_2048_1b_q4", 2048, 32, 8, 64, 16, 16384, False),
        # a short conversation with Llama-3.2-1B: the smallest call
        _attend("attend_1x201_1b_q4", 1, 200, 1, 32, 8, 64, 16, "q4"),
        # one very long one with an 8B model: what a 4-bit cache is for
        _attend("attend_1x131072_8b_q4", 1, 131071, 1, 32, 8, 128, 64, "q4"),
        # a batch of Qwen2.5-7B whose contexts are long and of all lengths
        _attend("attend_24x16384_7b_q4", 24, 16383, 1, 28, 4, 128, 32, "q4", ragged=True, half=True),
        # wide heads with capped scores, every second layer of such a model: the whole context ...
        _attend("attend_capped_16x4096", 16, 4095, 1, 16, 8, 256, 16, "f16", ragged=True, cap=50.0),
        # ... a bias by distance in place of a rotation, every head with its own k and v
        _attend("attend_slopes_29x2048", 29, 2047, 1, 32, 32, 128, 16, "f16", ragged=True, half=True, slopes=True),
        # a prompt chunk into which several short documents are packed
        _attend("attend_documents_4096", 1, 0, 4096, 32, 8, 128, 64, "f16", half=True, documents=9),
        # four prompts whose first part every row sees, of a model that caps its scores, into a 4-bit cache
        _attend("attend_prefix_4x700_q4", 4, 0, 700, 8, 4, 128, 32, "q4", ragged=True, cap=30.0, prefix=True),
        # the token that was drawn for one sequence of Llama-3.2-1B, with five alternatives
        _logprobs("logprobs_1x128256_top5", 1, 128256, 5),
        # a batch of Qwen2.5-7B, twenty alternatives each, drawn at a temperature of 0.8
        _logprobs("logprobs_64x151936_top20", 64, 151936, 20, scale=1.25),
        # scoring a prompt of Llama-2-7B's vocabulary, logits capped
        _logprobs("logprobs_2048x32000", 2048, 32000, 0, cap=30.0),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "logprobs", "logprobs"))
    most = {o: max(_cost(c) for c in listed() if c["op"] == o) for o in ("append", "attend", "logprobs")}[op]
    if op == "logprobs":
        case = _logprobs("", int(_log(rng, 1, 2049)), int(_log(rng, 64, 262145)), rng.choice((0, 1, 5, 20, 64)), rng.choice((0, 1, 1, 4)),
                         rng.choice((0.0, 0.0, 30.0)), rng.choice((1.0, 1.0, 1.25, 0.7)))
        while _cost(case) > most:
            case["rows"] = case["rows"] * 3 // 4
    else:
        kv = rng.choice((1, 2, 4, 8))
        group = rng.choice((1, 2, 3, 4, 6, 7, 8, 12, 16))
        dim = rng.choice((64, 96, 128, 128, 192, 256))
        page = rng.choice((16, 32, 64, 128))
        if op == "append":
            case = _append("", int(_log(rng, 1, 2049)), kv * group, kv, dim, page, int(_log(rng, 64, 131072)), rng.random() < 0.5,
                           dim if rng.random() < 0.7 else dim // 2)
            while _cost(case) > most:
                case["rows"] = case["rows"] * 3 // 4
        else:
            prompt = rng.random() < 0.4
            case = _attend("", int(_log(rng, 1, 9 if prompt else 65)), int(_log(rng, 1, 4097 if prompt else 65537)) - 1,
                           int(_log(rng, 2, 2049)) if prompt else 1, kv * group, kv, dim, page, rng.choice(("q4", "q4", "f16", "q8")), rng.random() < 0.6,
                           int(_log(rng, 16, 4097)) if rng.random() < 0.25 else 0, rng.random() < 0.5)
            if case["cache"] != "q4" or rng.random() < 0.5:
                case["cap"] = rng.choice((0.0, 30.0, 50.0))
                mask = rng.choice(("", "documents", "prefix"))
                case["slopes"] = rng.random() < 0.4 or not (case["cap"] or mask)
                case["documents"] = rng.randrange(2, 9) if mask == "documents" else 0
                case["prefix"] = mask == "prefix"
            while _cost(case) > most or _room(case) > 1 << 32:
                for k in ("requests", "past", "fresh"):
                    case[k] = max(1 if k != "past" else 0, case[k] * 7 // 8)
    del case["name"]
    return case


def _room(case):
    """Bytes of the scores and of the keys that the plain form makes."""
    tokens = case["past"] + case["fresh"]
    return 4 * case["requests"] * tokens * max(case["heads"] * case["fresh"], case["kv"] * case["dim"])


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
    return {"f16": 2 * values, "q8": values + values // BLOCK * 2, "q4": values // 2 + values // BLOCK * 2}[case["cache"]]


def _spread(most, n, ragged):
    return [most] * n if not ragged else [math.ceil(most * (i + 1) / n) for i in range(n)]


def _requests(case):
    """(tokens before the step, rows of the step) of each request."""
    n = case["requests"]
    return list(zip(_spread(case["past"], n, case["ragged"]), _spread(case["fresh"], n, case["ragged"] and case["fresh"] > 1)))


def _ranges(case, past, fresh):
    """The tokens [first, end) that each of a request's rows sees, as two arrays."""
    tokens = past + fresh
    at = np.arange(past, tokens)
    first, end = np.zeros(fresh, np.int64), at + 1
    if case["documents"]:
        n = case["documents"]
        starts = np.unique((tokens * (np.arange(n) / n) ** 1.3).astype(np.int64))     # documents grow longer
        first = starts[np.searchsorted(starts, at, side="right") - 1]
    if case["prefix"]:
        end = np.maximum(end, tokens * 5 // 8)
    if case["window"]:
        first = np.maximum(first, at - case["window"] + 1)
    return first, end


def _random_pool(case, pages, gen):
    per = _head_page_bytes(case)
    parts = 2 * pages * case["kv"]
    if case["cache"] == "f16":
        return torch.randn(parts * per // 2, device="cuda", generator=gen, dtype=torch.float16).view(torch.uint8)
    values = case["page"] * case["dim"]
    codes = values if case["cache"] == "q8" else values // 2
    pool = torch.randint(0, 256, (parts, per), device="cuda", generator=gen, dtype=torch.uint8)
    lo, hi = (0.004, 0.03) if case["cache"] == "q8" else (0.1, 0.4)
    d = torch.empty((parts, values // BLOCK), device="cuda").uniform_(lo, hi, generator=gen)
    if case["cache"] == "q4":
        d *= torch.randint(0, 2, d.shape, device="cuda", generator=gen) * 2 - 1      # the largest of a block has either sign
    pool[:, codes:] = d.to(torch.float16).view(torch.uint8)
    return pool.view(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = np.random.default_rng(seed)
    s = State()
    s.case = case
    ctx = context() if own else None

    def ints(values):
        return torch.as_tensor(np.ascontiguousarray(values, dtype=np.int32)).cuda()

    if case["op"] == "append":
        rows, heads, kv, dim, page, r = (case[k] for k in ("rows", "heads", "kv", "dim", "page", "rotated"))
        pages = -(-rows // page) * 2 + 3
        s.pool = _random_pool(case, pages, gen)
        s.qkv = torch.randn((rows, (heads + 2 * kv) * dim), device="cuda", generator=gen)
        s.q_out = torch.zeros((rows, heads * dim), device="cuda")
        decoding = rows < 128                                  # requests' next tokens, else one prompt's chunk
        s.slots = ints(host.permutation(pages * page)[:rows] if decoding else host.permutation(pages)[np.arange(rows) // page] * page + np.arange(rows) % page)
        s.positions = ints(host.integers(0, case["context"], rows) if decoding else max(case["context"] - rows, 0) + np.arange(rows))
        s.frequencies = 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
        s.k_read, s.v_read = (torch.zeros((rows, kv, dim), device="cuda", dtype=torch.float16) for _ in range(2))
        s.pages = pages
    elif case["op"] == "attend":
        _prepare_attend(s, case, gen, host, ints)
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        s.logits = 3 * torch.randn((rows, vocab), device="cuda", generator=gen)
        likely = torch.as_tensor(host.integers(0, vocab, (rows, 6))).cuda()          # what a model thinks comes next
        s.logits.scatter_add_(1, likely, 14 + 4 * torch.randn((rows, 6), device="cuda", generator=gen))
        tokens = np.where(host.random((rows, case["tokens"])) < 0.7, likely.cpu().numpy()[:, :1], host.integers(0, vocab, (rows, case["tokens"])))
        s.tokens = ints(tokens)
        s.logprobs, s.entropy = torch.zeros(tokens.shape, device="cuda"), torch.zeros(rows, device="cuda")
        top = min(top, vocab)
        s.top_tokens, s.top_logprobs = ints(np.zeros((rows, top))), torch.zeros((rows, top), device="cuda")
    if own:
        _bind(s, case, ctx)
    torch.cuda.synchronize()
    return s


def _prepare_attend(s, case, gen, host, ints):
    heads, kv, dim, page = (case[k] for k in ("heads", "kv", "dim", "page"))
    requests = [_requests(case)[i] for i in host.permutation(case["requests"])]
    ranges = [_ranges(case, *r) for r in requests]
    tokens = np.array([p + f for p, f in requests])
    fresh = np.array([f for _, f in requests])
    blocks = -(-(case["past"] + case["fresh"]) // page)
    begin = np.array([int(first.min()) // page for first, _ in ranges])   # pages that left the window are no longer held
    held = -(-tokens // page) - begin
    pages = int(held.sum()) + 2
    order, ends = host.permutation(pages), np.cumsum(held)
    table = np.zeros((len(requests), blocks), np.int64)
    for i in range(len(requests)):
        table[i, begin[i]:begin[i] + held[i]] = order[ends[i] - held[i]:ends[i]]
    rows = int(fresh.sum())
    s.rows, s.pages, s.most_rows, s.most_tokens = rows, pages, int(fresh.max()), int(tokens.max())
    s.row_starts = ints(np.concatenate([[0], np.cumsum(fresh)]))
    s.requests_of = ints(np.repeat(np.arange(len(requests)), fresh))
    s.positions = ints(np.concatenate([np.arange(p, p + f) for p, f in requests]))
    s.first = ints(np.concatenate([f for f, _ in ranges])) if case["documents"] else None
    s.end = ints(np.concatenate([e for _, e in ranges])) if case["prefix"] else None
    s.slopes = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["slopes"] else None
    s.pool, s.table = _random_pool(case, pages, gen), ints(table)
    s.q = (4.0 if case["cap"] else 1.5) * torch.randn((rows, heads * dim), device="cuda", generator=gen)
    s.out = torch.zeros((rows, heads * dim), device="cuda", dtype=torch.float16 if case["half"] else torch.float32)


def _bind(s, case, ctx):
    """The framework's objects over the tensors."""
    from jitllm_amd.attention import KvType, PagedAttention, PagedKvCache, Rope, RopeStyle

    def memory(t):
        return _Memory(ctx, t) if t is not None and t.numel() else None

    if case["op"] == "logprobs":
        from jitllm_amd.logits import LogProbabilities
        s.m_logits, s.m_tokens, s.m_logprobs, s.m_entropy = memory(s.logits), memory(s.tokens), memory(s.logprobs), memory(s.entropy)
        s.m_top_tokens, s.m_top_logprobs = memory(s.top_tokens), memory(s.top_logprobs)
        s.probabilities = LogProbabilities(ctx, case["rows"], case["vocab"], s.top_tokens.shape[1])
        return
    kind = {"f16": KvType.F16, "q8": KvType.Q8_0, "q4": KvType.Q4_0}[case["cache"]]
    s.cache = PagedKvCache(ctx, kind, s.pages, case["kv"], case["dim"], case["page"], memory=memory(s.pool))
    s.m_positions = memory(s.positions)
    if case["op"] == "append":
        s.m_qkv, s.m_q_out, s.m_slots = memory(s.qkv), memory(s.q_out), memory(s.slots)
        s.rope = Rope(ctx, memory(s.frequencies), case["rotated"], RopeStyle.HALVES if case["halves"] else RopeStyle.PAIRS)
        s.m_k_read, s.m_v_read = memory(s.k_read), memory(s.v_read)
    else:
        s.m_q, s.m_out, s.m_table, s.m_requests = memory(s.q), memory(s.out), memory(s.table), memory(s.requests_of)
        s.m_first, s.m_end, s.m_slopes = memory(s.first), memory(s.end), memory(s.slopes)
        s.attention = PagedAttention(ctx, s.rows, case["heads"], case["kv"], case["dim"])


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
    return {"append": _run_append, "attend": _run_attend, "logprobs": _run_logprobs}[s.case["op"]](s)


def _run_append(s):
    if not own:
        return _plain_append(s)
    from jitllm_amd.attention import Rows
    c = s.case
    q, k = c["heads"] * c["dim"], c["kv"] * c["dim"]
    stride = q + 2 * k
    s.cache.append(Rows(s.m_qkv, stride, q), Rows(s.m_qkv, stride, q + k), s.m_positions, s.m_slots, c["rows"], rope=s.rope,
                   q=Rows(s.m_qkv, stride), qOut=Rows(s.m_q_out, q), heads=c["heads"])
    s.cache.read(s.m_slots, c["rows"], s.m_k_read, s.m_v_read)
    return {"q": s.q_out, "k": s.k_read, "v": s.v_read}


def _run_attend(s):
    if not own:
        return _plain_attend(s)
    s.attention.attend(s.cache, s.m_q, s.rows, s.m_positions, s.m_table, s.m_out, requests=s.table.shape[0], rowRequests=s.m_requests,
                       window=s.case["window"], cap=s.case["cap"], slopes=s.m_slopes, firstTokens=s.m_first, endTokens=s.m_end)
    return s.out


def _run_logprobs(s):
    if not own:
        return _plain_logprobs(s)
    s.probabilities.compute(s.m_logits, s.case["rows"], tokens=s.m_tokens, logprobs=s.m_logprobs, entropy=s.m_entropy, topTokens=s.m_top_tokens,
                            topLogprobs=s.m_top_logprobs, tokensPerRow=s.case["tokens"], scale=s.case["scale"], cap=s.case["cap"])
    return {"logprobs": s.logprobs, "entropy": s.entropy, "top": s.top_tokens, "top_logprobs": s.top_logprobs}


# ---- the plain forms -----------------------------------------------------------------------------

def _plain_rotate(s, x):
    """In 64 bits: far positions need them, and so do values next to the border between two multiples of a block's scale."""
    r = s.case["rotated"]
    x = x.double()
    angle = s.positions.double()[:, None] * s.frequencies
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    if s.case["halves"]:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., r:]], -1).float()
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1).float()


def _plain_append(s):
    c = s.case
    rows, heads, kv, dim, page = (c[k] for k in ("rows", "heads", "kv", "dim", "page"))
    x = s.qkv.view(rows, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    turned = _plain_rotate(s, torch.cat([q, k], 1))
    q, k = turned[:, :heads].reshape(rows, heads * dim), turned[:, heads:]
    # written into the pages, and read from them
    pool = s.pool.view(2, s.pages, kv, -1).clone()
    slots = s.slots.long()
    at, offset = slots // page, slots % page
    codes = pool[..., :page * dim // 2]
    scales = pool[..., page * dim // 2:].view(torch.float16).view(2, s.pages, kv, dim // BLOCK, page)
    read = []
    for i, x in ((0, k), (1, v)):                              # (keys, and values, whose tokens stand in fours)
        blocks = x.reshape(rows, kv, dim // BLOCK, BLOCK)
        largest = blocks.gather(-1, blocks.abs().argmax(-1, keepdim=True))
        d = (largest / -8).half().float()
        n = torch.where(d != 0, (blocks / d).round().clamp(-8, 7), torch.zeros_like(blocks)) + 8
        n = n.to(torch.uint8).view(rows, kv, dim)
        held = n[..., 0::2] | n[..., 1::2] << 4
        d = d.half().view(rows, kv, dim // BLOCK)
        scales[i, at, :, :, offset] = d
        if i == 0:
            view = codes[0].view(s.pages, kv, page, dim // 2)
            view[at, :, offset] = held
            back = view[at, :, offset]
        else:
            view = codes[1].view(s.pages, kv, page // 4, dim // 4, 4, 2)
            view[at, :, offset // 4, :, offset % 4] = held.view(rows, kv, dim // 4, 2)
            back = view[at, :, offset // 4, :, offset % 4].reshape(rows, kv, dim // 2)
        back = torch.stack([back & 15, back >> 4], -1).float().view(rows, kv, dim // BLOCK, BLOCK) - 8
        read.append((back * scales[i, at, :, :, offset].float()[..., None]).half().view(rows, kv, dim))
    return {"q": q, "k": read[0], "v": read[1]}


def _values(case, pool, which):
    """[..., page_tokens, head_dim] in 32 bits of heads' parts of pages of keys (0) or values (1), [..., bytes]."""
    page, dim = case["page"], case["dim"]
    if case["cache"] == "f16":
        return pool.view(torch.float16).view(*pool.shape[:-1], page, dim).float()
    codes = page * dim if case["cache"] == "q8" else page * dim // 2
    d = pool[..., codes:].contiguous().view(torch.float16).view(*pool.shape[:-1], dim // BLOCK, page).transpose(-1, -2).float()
    if case["cache"] == "q8":
        n = pool[..., :codes].contiguous().view(torch.int8).float()
    else:
        n = pool[..., :codes]
        if which:
            n = n.reshape(*pool.shape[:-1], page // 4, dim // 4, 4, 2).transpose(-3, -2)
        n = n.reshape(*pool.shape[:-1], page, dim // 2)
        n = torch.stack([n & 15, n >> 4], -1).float() - 8
    n = n.reshape(*pool.shape[:-1], page, dim // BLOCK, BLOCK)
    return (n * d[..., None]).half().float().view(*pool.shape[:-1], page, dim)


def _plain_attend(s):
    c = s.case
    heads, kv, dim, page = (c[k] for k in ("heads", "kv", "dim", "page"))
    n, blocks = s.table.shape
    pool = s.pool.view(2, s.pages, kv, -1)
    k, v = (_values(c, pool[i][s.table.long()], i).transpose(1, 2).reshape(n, kv, blocks * page, dim)[:, :, :s.most_tokens] for i in (0, 1))
    # the rows of a request beside each other: [requests][rows of the longest]
    at = s.row_starts.long()[:-1, None] + torch.arange(s.most_rows, device="cuda")
    there = at < s.row_starts.long()[1:, None]
    at = at.clamp(max=s.rows - 1)
    position = s.positions.long()[at][..., None]
    j = torch.arange(s.most_tokens, device="cuda")
    seen = (j <= position if s.end is None else j < s.end.long()[at][..., None]) & there[..., None]
    if s.first is not None:
        seen &= j >= s.first.long()[at][..., None]
    if c["window"]:
        seen &= j > position - c["window"]
    q = s.q.view(s.rows, kv, heads // kv, dim)[at] * dim ** -0.5                     # [requests][rows][kv][group][dim]
    q = q.permute(0, 2, 3, 1, 4).reshape(n, kv, heads // kv * s.most_rows, dim)
    scores = torch.matmul(q, k.transpose(-1, -2)).view(n, kv, heads // kv, s.most_rows, s.most_tokens)
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    if s.slopes is not None:
        scores = scores - s.slopes.view(kv, heads // kv, 1, 1) * (position - j).abs().float()[:, None, None]
    scores = torch.where(seen[:, None, None], scores, -torch.inf)
    top = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top.isfinite(), top, 0))
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, 1)
    out = torch.matmul(weight.view(n, kv, heads // kv * s.most_rows, s.most_tokens), v).view(n, heads, s.most_rows, dim)
    return out.transpose(1, 2)[there].reshape(s.rows, heads * dim).to(s.out.dtype)


def _plain_logprobs(s):
    c = s.case
    x = s.logits
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    x = x * c["scale"]
    most = x.amax(-1, keepdim=True)
    below = x - most
    weight = torch.exp(below)
    total = weight.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - (weight * below).sum(-1, keepdim=True) / total)[:, 0]
    logprobs = below.gather(1, s.tokens.long()) - log_total
    ranked = torch.sort(s.logits, dim=-1, descending=True, stable=True).indices[:, :s.top_tokens.shape[1]]
    return {"logprobs": logprobs, "entropy": entropy, "top": ranked.int(), "top_logprobs": below.gather(1, ranked) - log_total}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](s, case)


def _exact_append(s, case):
    rows, heads, kv, dim, r = (case[k] for k in ("rows", "heads", "kv", "dim", "rotated"))
    q, k, v = s.qkv.double().view(rows, heads + 2 * kv, dim).split([heads, kv, kv], 1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s.positions.double(), s.frequencies))[:, None]

    def rotate(x):
        pairs = x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2) if case["halves"] else x[..., :r].unflatten(-1, (r // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z.transpose(-1, -2).flatten(-2) if case["halves"] else z.flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    def kept(x):
        y = x.unflatten(-1, (dim // BLOCK, BLOCK))
        low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
        d = (torch.where(-low >= high, low, high) * -0.125).half().double()
        return (torch.floor(y / d + 0.5).clamp(-8, 7) * d).half().double().flatten(-2)

    return {"q": rotate(q).reshape(rows, heads * dim), "k": kept(rotate(k)), "v": kept(v)}


def _exact_attend(s, case):
    heads, kv, dim, page = (case[k] for k in ("heads", "kv", "dim", "page"))
    parts = s.pool.view(2, s.pages, kv, -1)
    out = torch.zeros((s.rows, kv, heads // kv, dim), dtype=torch.float64, device="cuda")
    starts, group = s.row_starts.tolist(), heads // kv
    for request in range(len(starts) - 1):
        rows = slice(starts[request], starts[request + 1])
        positions = s.positions[rows].double()[:, None]
        tokens = int(s.positions[rows][-1]) + 1
        j = torch.arange(tokens, device="cuda", dtype=torch.float64)
        hidden = j > positions if s.end is None else j >= s.end[rows].double()[:, None]
        if s.first is not None:
            hidden |= j < s.first[rows].double()[:, None]
        if case["window"]:
            hidden |= positions - j >= case["window"]
        held = s.table[request, :-(-tokens // page)].long()
        for h in range(kv):
            keys, values = (_exact_values(parts[i, held, h], case, i)[:tokens] for i in (0, 1))
            for g in range(group):
                q = s.q[rows].double().view(-1, kv, group, dim)[:, h, g]
                score = q @ keys.T / math.sqrt(dim)
                if case["cap"]:
                    score = torch.tanh(score / case["cap"]) * case["cap"]
                if case["slopes"]:
                    score = score - s.slopes[h * group + g].double() * (positions - j).abs()
                out[rows, h, g] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ values
    return out.view(s.rows, heads * dim)


def _exact_values(raw, case, which):
    page, dim = case["page"], case["dim"]
    raw = raw.contiguous()
    if case["cache"] == "f16":
        return raw.view(torch.float16).double().view(-1, dim)
    codes = page * dim // (1 if case["cache"] == "q8" else 2)
    d = raw[:, codes:].contiguous().view(torch.float16).double().view(-1, dim // BLOCK, page).transpose(1, 2)
    d = d.repeat_interleave(BLOCK, -1)
    n = raw[:, :codes].contiguous()
    if case["cache"] == "q8":
        return (n.view(torch.int8).double().view(-1, page, dim) * d).half().double().reshape(-1, dim)
    token, element = torch.arange(page, device="cuda")[:, None], torch.arange(dim, device="cuda")
    at = token // 4 * (2 * dim) + element // 4 * 8 + token % 4 * 2 + element % 4 // 2 if which else token * (dim // 2) + element // 2
    n = (n[:, at] >> (element % 2 * 4).to(torch.uint8) & 15).double() - 8
    return (n * d).half().double().reshape(-1, dim)


def _exact_logprobs(s, case):
    out = {"logprobs": [], "entropy": [], "top_logprobs": []}
    for rows in torch.arange(case["rows"], device="cuda").split(64):
        x = s.logits[rows].double()
        if case["cap"]:
            x = torch.tanh(x / case["cap"]) * case["cap"]
        logp = torch.log_softmax(x * case["scale"], -1)
        out["logprobs"].append(torch.take_along_dim(logp, s.tokens[rows].long(), 1))
        out["entropy"].append(-torch.special.xlogy(logp.exp(), logp.exp()).sum(-1))
        best = logp.topk(s.top_tokens.shape[1], -1).values
        out["top_logprobs"].append(best)
    return {"logprobs": torch.cat(out["logprobs"]), "entropy": torch.cat(out["entropy"]), "top": None, "top_logprobs": torch.cat(out["top_logprobs"])}


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": 4 * rows * (vocab + 2 * case["tokens"] + 1 + 2 * min(case["top"], vocab)), "flops": rows * vocab * (5 if not case["cap"] else 9)}
    heads, kv, dim = (case[k] for k in ("heads", "kv", "dim"))
    token = 2 * kv * _head_page_bytes(case) // case["page"]                          # bytes of a token's keys and values
    if case["op"] == "append":
        rows = case["rows"]
        return {"bytes": rows * (4 * (heads + 2 * kv) * dim + 4 * heads * dim + 2 * token + 4 * kv * dim + 8),
                "flops": rows * (heads + kv) * 3 * case["rotated"]}
    seen = cached = rows = 0
    for past, fresh in _requests(case):
        first, end = _ranges(case, past, fresh)
        seen += int((end - first).sum())
        cached += int(end.max() - first.min())
        rows += fresh
    return {"bytes": cached * token + rows * heads * dim * (4 + (2 if case["half"] else 4)) + 4 * (cached // case["page"] + 2 * rows),
            "flops": 4 * heads * dim * seen}
